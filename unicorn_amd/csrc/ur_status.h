// Error reporting shared by the translation units of the library: the message behind ur_last_error() is one
// thread-local buffer, written through these functions (defined beside it, in ur_library.hip).
#pragma once
#include <stddef.h>

namespace ur {

// stores the message and returns `code` (a negative UR_ERR_* value)
__attribute__((visibility("hidden"), format(printf, 2, 3))) int set_error(int code, const char* fmt, ...);

// UR_OK, or UR_ERR_LAUNCH with the runtime's message when the launch just made was refused
__attribute__((visibility("hidden"))) int launch_status(const char* what);

// UR_OK, or UR_ERR_WORKSPACE: `need` bytes of 16-byte aligned workspace (nothing at all when need is 0)
__attribute__((visibility("hidden"))) int check_workspace(const void* workspace, size_t bytes, size_t need);

}  // namespace ur
