r"""``nn.Module`` around the 8-bit linear layer, for serving a trained ``nn.Linear``: the weights are turned into 8-bit rows once and
kept as buffers (``q``, ``scale``) next to the ``bias``."""
from typing import Optional, Union

import torch
import torch.nn as nn
from torch import Tensor

from .kernel import Int8Rows, int8_linear, int8_rows2d, quantize_rows


class Int8Linear(nn.Module):

    def __init__(self, weight: Int8Rows, bias: Optional[Tensor] = None):
        super().__init__()
        assert weight.q.dim() == 2, "the weight is a matrix of 8-bit rows"
        assert bias is None or bias.shape == (weight.q.shape[0],), "Bias shape mismatch"
        self.register_buffer("q", weight.q)
        self.register_buffer("scale", weight.scale)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        r"""The 8-bit form of a linear layer on a CUDA device; the bias keeps its type."""
        return cls(quantize_rows(linear.weight.detach()), None if linear.bias is None else linear.bias.detach().clone())

    def _apply(self, fn, recurse=True):
        # a conversion of the model (``half()``, ``to(dtype)``) reaches the bias; scales stay float32, and a copy to another device keeps
        # the layout of the rows
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = scale.to(self.scale.device)
        if self.q.is_cuda:
            self.q = int8_rows2d(Int8Rows(self.q, self.scale), "weight").q
        return self

    def forward(self, x: Union[Tensor, Int8Rows], dtype: Optional[torch.dtype] = None) -> Tensor:
        return int8_linear(x, Int8Rows(self.q, self.scale), self.bias, dtype)
