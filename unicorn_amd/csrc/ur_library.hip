// The renderer's translation unit (ur_render.hip as it stands) and, beside its thread-local error buffer, the
// functions through which the other translation units report errors.  -DUR_RENDER_SRC="..." builds the library around
// another renderer source (timing variants).
#ifndef UR_RENDER_SRC
#define UR_RENDER_SRC "ur_render.hip"
#endif
#include UR_RENDER_SRC
#include "ur_status.h"

namespace ur {

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int launch_status(const char* what) { return check_launch(what); }

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need == 0) return UR_OK;
  if (bytes < need || !workspace) return set_error(UR_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace ? bytes : 0, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(UR_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  return UR_OK;
}

}  // namespace ur
