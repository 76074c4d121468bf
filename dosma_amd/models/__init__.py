"""Segmentation models (reference ``dosma/models/__init__.py``) and the operators on their answers."""
from dosma_amd.models.oaiunet2d import AnswerMaps, IWOAIOAIUnet2D, IWOAIOAIUnet2DNormalized, OAIUnet2D  # noqa: F401
from dosma_amd.models.stanford_qdess import StanfordQDessUNet2D  # noqa: F401
from dosma_amd.models.seg_model import SegModel, whiten_volume  # noqa: F401
from dosma_amd.models.util import SUPPORTED_MODELS, get_model, model_from_config  # noqa: F401
from dosma_amd.models.answers import (  # noqa: F401
    DistillLoss,
    LabelScores,
    distill_loss,
    distill_loss_grad,
    label_scores,
    label_scores_grad,
)
