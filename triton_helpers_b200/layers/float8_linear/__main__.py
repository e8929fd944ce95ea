r"""``python -m triton_helpers_b200.layers.float8_linear benchmark|profile ...``: the 8-bit floating-point layer for serving (its input in 16
bits) and the one for training against ``F.linear`` over the number of tokens ``L`` (``D`` inputs, ``N`` outputs)."""
from dataclasses import dataclass
from typing import Any, Dict

import torch
import torch.nn.functional as F
from torch import Tensor

from ...benchmark import CLI, KernelExecutor
from .kernel import Float8Blocks, float8_linear, float8_training_linear, quantize_float8_weight


@dataclass
class Baseline(KernelExecutor):

    def prepare_inputs(self, L, D, N, dtype=torch.float16, device="cuda", requires_grad=False, **_) -> Dict[str, Any]:
        torch.random.manual_seed(0)
        x = torch.randn(L, D, device=device, dtype=dtype, requires_grad=requires_grad)
        return {"x": x, "weight": (torch.randn(N, D, device=device, dtype=dtype) * D**-0.5).requires_grad_(requires_grad)}

    def forward(self, x: Tensor, weight: Tensor) -> Tensor:
        return F.linear(x, weight)


@dataclass
class Training(Baseline):

    def forward(self, x: Tensor, weight: Tensor) -> Tensor:
        return float8_training_linear(x, weight)


@dataclass
class Serving(Baseline):

    def prepare_inputs(self, **kwargs) -> Dict[str, Any]:
        inputs = super().prepare_inputs(**{**kwargs, "requires_grad": False})
        return {"x": inputs["x"], "weight": quantize_float8_weight(inputs["weight"])}

    def forward(self, x: Tensor, weight: Float8Blocks) -> Tensor:
        return float8_linear(x, weight)


if __name__ == "__main__":
    CLI.entrypoint(
        "Float8 Linear",
        [Baseline("baseline"), Training("training"), Serving("serving")],
        dims={"L": ((1, 16, 128, 1024, 8192), "values"), "D": (4096, "values"), "N": (4096, "values")},
    )
