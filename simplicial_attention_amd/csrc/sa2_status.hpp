// Failures of C entry points that live outside sa2_api.hip.
#pragma once

namespace sa2 {

// keeps the message for sa2_last_error on this thread, returns `code`
int fail_with(int code, const char *fmt, ...);
// SA2_OK, or SA2_ERR_LAUNCH with the message of the last launch
int launched(const char *what);

}  // namespace sa2
