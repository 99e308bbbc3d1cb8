"""What sits right behind the observation on the training side, and what a policy needs around its update:
categorical actions and gradient clipping."""
from .categorical import evaluate_categorical, evaluate_categorical_grad, sample_categorical
from .grad_clip import clip_grad_norm_, clip_grads, grad_norm
from .running_standard_scaler import RunningStandardScaler

__all__ = ["RunningStandardScaler", "clip_grad_norm_", "clip_grads", "evaluate_categorical", "evaluate_categorical_grad",
           "grad_norm", "sample_categorical"]
