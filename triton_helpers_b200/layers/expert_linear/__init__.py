from .kernel import expert_linear
from .module import ExpertLinear


__all__ = ["expert_linear", "ExpertLinear"]
