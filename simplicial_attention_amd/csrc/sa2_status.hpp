// Failures of C entry points that live outside sa2_api.hip.
#pragma once

#include <cstdint>

namespace sa2 {

// a * b * c <= most, whatever the sizes (each at least 1)
inline bool product_within(int64_t a, int64_t b, int64_t c, int64_t most) { return a <= most && b <= most / a && c <= most / (a * b); }

// keeps the message for sa2_last_error on this thread, returns `code`
int fail_with(int code, const char *fmt, ...);
// SA2_OK, or SA2_ERR_LAUNCH with the message of the last launch
int launched(const char *what);

}  // namespace sa2
