r"""``python -m triton_helpers_b200.layers.rms_norm benchmark|profile ...``: the norm of ``x + residual`` against elementary torch
operations over the number of rows ``L`` (32 x L rows, width ``D``)."""
from dataclasses import dataclass
from typing import Any, Dict

import torch
from torch import Tensor

from ...benchmark import CLI, KernelExecutor
from .kernel import rms_norm


@dataclass
class Baseline(KernelExecutor):

    def prepare_inputs(self, L, D, dtype=torch.bfloat16, device="cuda", requires_grad=False, **_) -> Dict[str, Any]:
        torch.random.manual_seed(0)
        x, residual = (torch.randn(32, L, D, device=device, dtype=dtype, requires_grad=requires_grad) for _ in range(2))
        weight = torch.ones(D, device=device, dtype=dtype, requires_grad=requires_grad)
        return {"x": x, "weight": weight, "residual": residual}

    def forward(self, x: Tensor, weight: Tensor, residual: Tensor) -> Tensor:
        s = (x + residual).float()
        return (s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * weight.float()).to(x.dtype)


@dataclass
class Fused(Baseline):

    def forward(self, x: Tensor, weight: Tensor, residual: Tensor) -> Tensor:
        return rms_norm(x, weight, residual)[0]


if __name__ == "__main__":
    CLI.entrypoint("RMS Norm", [Baseline("baseline"), Fused("fused")], dims={"L": ((1, 16, 128, 512), "values"), "D": (4096, "values")})
