r"""``nn.Module`` around the layers of several experts; ``weight`` is ``(experts, out, in)``, each expert initialised as an ``nn.Linear``."""
import math

import torch
import torch.nn as nn
from torch import Tensor

from .kernel import MAX_EXPERTS, expert_linear


class ExpertLinear(nn.Module):

    def __init__(self, num_experts: int, in_features: int, out_features: int, device=None, dtype=None):
        super().__init__()
        assert 1 <= num_experts <= MAX_EXPERTS, f"1 to {MAX_EXPERTS} experts, got {num_experts}"
        self.weight = nn.Parameter(torch.empty((num_experts, out_features, in_features), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = 1 / math.sqrt(self.weight.shape[2])
        nn.init.uniform_(self.weight, -bound, bound)

    def forward(self, x: Tensor, ends: Tensor) -> Tensor:
        return expert_linear(x, self.weight, ends)
