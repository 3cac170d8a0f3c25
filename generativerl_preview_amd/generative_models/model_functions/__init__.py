from .cross_entropy import linear_cross_entropy  # noqa: F401
from .losses import fused_loss, prepare_flow_matching, prepare_icfm, prepare_score_matching  # noqa: F401
