"""The reference TTT model's attention (``cloud_ttt_e2e/ttt_e2e``) on the HIP
kernels: ``GradGradAttentionFn`` with an additive mask and
``WindowedSelfAttention``, whose chunked window runs as one problem with a
structured mask, and the operators at the model's tail: layer norm and the
cross entropy of its head (``layer_norm``, ``linear_cross_entropy``), each
twice differentiable.  The model, its meta step and its data, the callers of this
attention, live outside the library package (top-level ``ttt_e2e``)."""
from .attention import GradGradAttentionFn, WindowedSelfAttention, gradgrad_attention, windowed_attention
from .loss import linear_cross_entropy
from .norm import LayerNorm, layer_norm
from .utils import local_window_mask, make_window_mask

__all__ = ["GradGradAttentionFn", "WindowedSelfAttention", "gradgrad_attention", "windowed_attention",
           "make_window_mask", "local_window_mask", "layer_norm", "LayerNorm", "linear_cross_entropy"]
