r"""``python -m triton_helpers_b200.layers.checkpointed_linear benchmark|profile ...``: the linear layer that keeps its input in 8 bits
against ``F.linear`` over the number of rows ``L`` (``D`` inputs, ``N`` outputs)."""
from dataclasses import dataclass
from typing import Any, Dict

import torch
import torch.nn.functional as F
from torch import Tensor

from ...benchmark import CLI, KernelExecutor
from .kernel import checkpointed_linear


@dataclass
class Baseline(KernelExecutor):

    def prepare_inputs(self, L, D, N, dtype=torch.float16, device="cuda", requires_grad=False, **_) -> Dict[str, Any]:
        torch.random.manual_seed(0)
        x = torch.randn(L, D, device=device, dtype=dtype, requires_grad=requires_grad)
        weight = (torch.randn(N, D, device=device, dtype=dtype) * D**-0.5).requires_grad_(requires_grad)
        bias = torch.zeros(N, device=device, dtype=dtype, requires_grad=requires_grad)
        return {"x": x, "weight": weight, "bias": bias}

    def forward(self, x: Tensor, weight: Tensor, bias: Tensor) -> Tensor:
        return F.linear(x, weight, bias)


@dataclass
class Checkpointed(Baseline):

    def forward(self, x: Tensor, weight: Tensor, bias: Tensor) -> Tensor:
        return checkpointed_linear(x, weight, bias)


if __name__ == "__main__":
    CLI.entrypoint(
        "Checkpointed Linear",
        [Baseline("baseline"), Checkpointed("checkpointed")],
        dims={"L": ((300, 2048, 8192, 16384), "values"), "D": (4096, "values"), "N": (4096, "values")},
    )
