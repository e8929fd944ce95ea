r"""``python -m triton_helpers_b200.layers.expert_linear benchmark|profile ...``: layers of ``E`` experts with ``L / E`` rows each against a
batched product over the number of rows ``L`` (``D`` inputs, ``N`` outputs)."""
from dataclasses import dataclass
from typing import Any, Dict

import torch
from torch import Tensor

from ...benchmark import CLI, KernelExecutor
from .kernel import expert_linear


@dataclass
class Baseline(KernelExecutor):

    def prepare_inputs(self, L, E, D, N, dtype=torch.float16, device="cuda", requires_grad=False, **_) -> Dict[str, Any]:
        torch.random.manual_seed(0)
        rows = -(-L // E) * E
        x = torch.randn(rows, D, device=device, dtype=dtype, requires_grad=requires_grad)
        weight = (torch.randn(E, N, D, device=device, dtype=dtype) * D**-0.5).requires_grad_(requires_grad)
        ends = torch.arange(1, E + 1, device=device, dtype=torch.int32) * (rows // E)
        return {"x": x, "weight": weight, "ends": ends}

    def forward(self, x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
        return torch.bmm(x.view(weight.shape[0], -1, x.shape[1]), weight.transpose(1, 2)).view(x.shape[0], -1)


@dataclass
class Experts(Baseline):

    def forward(self, x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
        return expert_linear(x, weight, ends)


if __name__ == "__main__":
    CLI.entrypoint(
        "Expert Linear",
        [Baseline("baseline"), Experts("experts")],
        dims={"L": ((64, 1024, 16384), "values"), "E": (32, "values"), "D": (2048, "values"), "N": (2048, "values")},
    )
