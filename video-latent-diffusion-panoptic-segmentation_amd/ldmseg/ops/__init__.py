from . import native  # noqa: F401
from .label_probs import label_log_probs  # noqa: F401
from .native import clip_grads, grad_norm, label_log_probs_bwd, load_library  # noqa: F401
