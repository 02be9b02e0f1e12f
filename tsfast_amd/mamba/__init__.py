"""Fused Mamba selective-SSM dispatch point and its HIP backend (``mamba_hip``), and a layer in service: packed
prompts and single tokens (``serving``, ``packed_hip``)."""

from .core import mamba_ssm  # noqa: F401
from .serving import mamba_conv_packed, mamba_ssm_packed, mamba_step  # noqa: F401
