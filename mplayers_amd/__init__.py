"""MI355X-native min-sum message-passing layers (TRWP, ISGMR) behind the reference's surface."""
from . import lib_seg, lib_stereo  # noqa: F401
from .distillation import best_labels, distill_costs  # noqa: F401
from .label_context import bucket_context, label_buckets  # noqa: F401
from .layout import labels_last_dropout, labels_last_norm  # noqa: F401
from .sampling import sample_labels, verify_labels  # noqa: F401
from .MP_module import ISGMRFunction, MPModule, TRWPFunction  # noqa: F401
