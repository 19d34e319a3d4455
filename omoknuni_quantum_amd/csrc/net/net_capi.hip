// Error reporting of libomq_net_ops.so.  Declarations: include/omq_net_ops.h.
#include <cstdarg>
#include <cstdio>

#include "net_common.h"

namespace omq_net {

static thread_local char g_error[512] = "";

int net_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}

int net_status(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return OMQ_NET_OK;
  return net_fail(OMQ_NET_E_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace omq_net

extern "C" {

int omq_net_abi_version(void) { return OMQ_NET_ABI_VERSION; }

const char* omq_net_last_error(void) { return omq_net::g_error; }

}  // extern "C"
