"""B200-native (sm_100a) Gaussian-splat rasterizer with the ds-splat operator surface.

    from ds_splat_b200 import GaussianRasterizationSettings, GaussianRasterizer

mirrors ``from ds_splat import ...`` of the reference (ds_splat/__init__.py:1-4).  ``gated_recurrence`` (with its single-row
form) and ``dropout`` are additions.
"""
from .rasterizer import DsRasterizerFunction, GaussianRasterizationSettings, GaussianRasterizer
from .sequence import dropout, gated_recurrence, gated_recurrence_step

__all__ = ["GaussianRasterizationSettings", "GaussianRasterizer", "DsRasterizerFunction", "gated_recurrence",
           "gated_recurrence_step", "dropout"]
