// Error reporting of the C entry points: the message behind jq_last_error() is
// kept for each thread.
#pragma once

namespace jq {

// Record the message and return the code.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char *fmt, ...);
// JQ_OK, or JQ_E_HIP where the launch before it was refused.
__attribute__((visibility("hidden"))) int launch_check(const char *what);

}  // namespace jq
