from .clip import clip_grad_norm_, grad_norm  # noqa: F401
from .optimizer import OPTIMIZERS, FusedAdam, load_checkpoint, save_checkpoint  # noqa: F401
