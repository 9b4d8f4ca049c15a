from .distillation import distillation
from .log_probabilities import log_probabilities

__all__ = ["distillation", "log_probabilities"]
