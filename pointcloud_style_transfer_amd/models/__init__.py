"""Drop-in for the reference's `models/__init__.py:3-33` re-export surface."""
from .diffusion_model import (
    TimeEmbedding,
    StyleEncoder,
    NoisePredictor,
    HierarchicalProcessor,
    PointCloudDiffusionModel,
    DiffusionProcess,
)
from .blocks import (
    GatedBlock,
    GatedLinear,
    RMSNorm,
    gated_linear,
    gated_linear_quant,
    quant_rows,
    rms_norm,
    rms_norm_quant,
)
from .losses import DiffusionLoss
from .pointnet2_encoder import PointNet2Encoder

__all__ = [
    "TimeEmbedding",
    "StyleEncoder",
    "NoisePredictor",
    "HierarchicalProcessor",
    "PointCloudDiffusionModel",
    "DiffusionProcess",
    "DiffusionLoss",
    "PointNet2Encoder",
    "RMSNorm",
    "GatedLinear",
    "GatedBlock",
    "rms_norm",
    "rms_norm_quant",
    "quant_rows",
    "gated_linear",
    "gated_linear_quant",
]
