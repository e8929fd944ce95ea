from .kernel import checkpointed_linear
from .module import CheckpointedLinear


__all__ = ["checkpointed_linear", "CheckpointedLinear"]
