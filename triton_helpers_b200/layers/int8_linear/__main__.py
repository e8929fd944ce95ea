r"""``python -m triton_helpers_b200.layers.int8_linear benchmark|profile ...``: the 8-bit linear layer, its input in 16 bits, against
``F.linear`` over the number of tokens ``L`` (``D`` inputs, ``N`` outputs)."""
from dataclasses import dataclass
from typing import Any, Dict

import torch
import torch.nn.functional as F
from torch import Tensor

from ...benchmark import CLI, KernelExecutor
from .kernel import Int8Rows, int8_linear, quantize_rows


@dataclass
class Baseline(KernelExecutor):

    def prepare_inputs(self, L, D, N, dtype=torch.float16, device="cuda", requires_grad=False, **_) -> Dict[str, Any]:
        torch.random.manual_seed(0)
        return {"x": torch.randn(L, D, device=device, dtype=dtype), "weight": torch.randn(N, D, device=device, dtype=dtype) * D**-0.5}

    def forward(self, x: Tensor, weight: Tensor) -> Tensor:
        return F.linear(x, weight)


@dataclass
class Int8(Baseline):

    def prepare_inputs(self, **kwargs) -> Dict[str, Any]:
        inputs = super().prepare_inputs(**kwargs)
        return {"x": inputs["x"], "weight": quantize_rows(inputs["weight"])}

    def forward(self, x: Tensor, weight: Int8Rows) -> Tensor:
        return int8_linear(x, weight)


if __name__ == "__main__":
    CLI.entrypoint(
        "Int8 Linear",
        [Baseline("baseline"), Int8("int8")],
        dims={"L": ((1, 16, 128, 1024, 8192), "values"), "D": (4096, "values"), "N": (4096, "values")},
    )
