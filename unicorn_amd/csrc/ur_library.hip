// The renderer's translation unit (ur_render.hip as it stands) and, beside its thread-local error buffer, the two
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

}  // namespace ur
