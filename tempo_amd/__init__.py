"""tempo_amd: MI355X-native heatmap -> voxel unprojection for TEMPO.

Drop-in replacements for the reference's ``tempo/models/project_layer.py``
modules, running hand-written HIP kernels (gfx950) through a C ABI, and the
temporal head's operators that go in front of them.
"""
from .project_layer import (PackedHeatmaps, ProcessLayerNHWC, ProjectLayer,  # noqa: F401
                            ProjectLayerWithMask, RecurrentProcessLayerNHWC)
from .temporal import fused_linear, gated_recurrence  # noqa: F401

__all__ = ['ProjectLayer', 'ProjectLayerWithMask', 'ProcessLayerNHWC', 'PackedHeatmaps',
           'RecurrentProcessLayerNHWC', 'fused_linear', 'gated_recurrence']
