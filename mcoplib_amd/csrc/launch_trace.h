// launch_trace.h -- MCOP_DEBUG_TRACE lines of launches that the row kernels' geometry choice (abi.hip, which
// prints its own) does not make.
#pragma once

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>

namespace mcop {

inline bool launches_traced() {
  static const bool on = [] {
    const char* v = getenv("MCOP_DEBUG_TRACE");
    return v != nullptr && (strcmp(v, "1") == 0 || strcmp(v, "ON") == 0 || strcmp(v, "on") == 0);
  }();
  return on;
}

inline void trace_launch(const char* op, const char* fmt, ...) {
  if (!launches_traced()) return;
  char line[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(line, sizeof(line), fmt, ap);
  va_end(ap);
  fprintf(stdout, "[mcop] %s %s\n", op, line);
  fflush(stdout);
}

}  // namespace mcop
