// dd_common.h -- host-side pieces shared by the library's source files.
#pragma once

namespace dd {

// Record the reason that dd_last_error(NULL) returns and pass `code` on.
int global_fail(int code, const char* fmt, ...);

}  // namespace dd
