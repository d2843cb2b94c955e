"""``ttt_e2e.norm`` import path; see testtimeideas_amd.ttt_e2e.norm."""
from testtimeideas_amd.ttt_e2e.norm import LayerNorm, layer_norm  # noqa: F401
