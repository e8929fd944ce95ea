r"""``nn.Linear`` that keeps its input as 8-bit rows for the backward pass: same parameters, initialisation and ``state_dict``."""
import torch.nn as nn
from torch import Tensor

from .kernel import checkpointed_linear


class CheckpointedLinear(nn.Linear):

    def forward(self, x: Tensor) -> Tensor:
        return checkpointed_linear(x, self.weight, self.bias)
