r"""``nn.Module`` around the root-mean-square norm; the gain ``weight`` starts at one."""
from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch import Tensor

from ..int8_linear.kernel import Int8Rows
from .kernel import rms_norm, rms_norm_int8


class RMSNorm(nn.Module):

    def __init__(self, d_model: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d_model))
        self.eps = eps

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
        return rms_norm(x, self.weight, residual, self.eps)

    @torch.no_grad()
    def int8(self, x: Tensor, residual: Optional[Tensor] = None) -> Union[Int8Rows, Tuple[Int8Rows, Tensor]]:
        r"""The norm's output as 8-bit rows, for an ``Int8Linear`` that follows; no gradient."""
        return rms_norm_int8(x, self.weight, residual, self.eps)
