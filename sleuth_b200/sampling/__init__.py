"""Sampling: options, host-side state, and the GPU sampler."""

from .config import SamplingConfig
from .drafts import DraftPolicy, NgramDrafter
from .host import NgramBlocker, fresh_seed, recent_window, uniform, uniforms

__all__ = ["SamplingConfig", "DraftPolicy", "NgramDrafter", "NgramBlocker", "fresh_seed", "recent_window", "uniform", "uniforms"]
