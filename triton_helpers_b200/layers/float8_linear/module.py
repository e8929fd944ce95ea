r"""``nn.Module``s around the 8-bit floating-point layers. ``Float8Linear`` serves a trained ``nn.Linear``: the weights are turned into 8-bit
blocks once and kept as buffers (``q``, ``scale``) next to the ``bias``. ``Float8TrainingLinear`` is an ``nn.Linear`` in training."""
from typing import Optional, Union

import torch
import torch.nn as nn
from torch import Tensor

from .kernel import Float8Blocks, _weight2d, float8_linear, float8_training_linear, quantize_float8_weight


class Float8Linear(nn.Module):

    def __init__(self, weight: Float8Blocks, bias: Optional[Tensor] = None):
        super().__init__()
        weight = _weight2d(weight, "weight")
        assert bias is None or bias.shape == (weight.q.shape[0],), "Bias shape mismatch"
        self.register_buffer("q", weight.q)
        self.register_buffer("scale", weight.scale)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Float8Linear":
        r"""The 8-bit form of a linear layer on a CUDA device; the bias keeps its type."""
        return cls(quantize_float8_weight(linear.weight.detach()), None if linear.bias is None else linear.bias.detach().clone())

    def _apply(self, fn, recurse=True):
        # a conversion of the model (``half()``, ``to(dtype)``) reaches the bias; values and scales keep their types, and a copy to another
        # device keeps the layout of the rows
        q, scale = self.q, self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = scale.to(self.scale.device)
        if self.q.dtype != torch.float8_e4m3fn:
            self.q = q.to(self.q.device)
        if self.q.is_cuda:
            self.q = _weight2d(Float8Blocks(self.q, self.scale), "weight").q
        return self

    def forward(self, x: Union[Tensor, Float8Blocks], dtype: Optional[torch.dtype] = None) -> Tensor:
        return float8_linear(x, Float8Blocks(self.q, self.scale), self.bias, dtype)


class Float8TrainingLinear(nn.Linear):

    def forward(self, x: Tensor) -> Tensor:
        return float8_training_linear(x, self.weight, self.bias)
