// ttt_ops.h — what the operators' sources (ttt_norm.hip, ttt_lce.hip) share
// with the attention's C entry points.
#pragma once

namespace ttt {

// Records a message for ttt_last_error() and returns `code` (ttt_capi.hip).
int ops_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace ttt
