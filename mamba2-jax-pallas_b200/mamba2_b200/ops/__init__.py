"""Ops around the SSD (B200 replacements of ``src/mamba2_jax/ops``)."""
from .causal_conv1d import causal_conv1d, causal_conv1d_update
from .cross_entropy import linear_cross_entropy, linear_cross_entropy_grad
from .embedding import embedding, embedding_grad
from .grad_clip import clip_grad_norm, grad_norm
from .rms_norm import rms_norm_gated
from .selective_state_update import selective_state_update

__all__ = ["selective_state_update", "causal_conv1d", "causal_conv1d_update", "rms_norm_gated",
           "embedding", "embedding_grad", "linear_cross_entropy", "linear_cross_entropy_grad",
           "grad_norm", "clip_grad_norm"]
