"""``ttt_e2e.loss`` import path; see testtimeideas_amd.ttt_e2e.loss."""
from testtimeideas_amd.ttt_e2e.loss import linear_cross_entropy  # noqa: F401
