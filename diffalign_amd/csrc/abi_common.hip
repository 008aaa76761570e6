#include "common.h"
#include <cstdarg>
#include <cstdio>

static thread_local char g_err[512] = "";

void da_set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

extern "C" {
const char* da_last_error(void) { return g_err; }
// 3: da_init added, the two-pass output stage (da_edge_out_g / da_edge_out_finish) removed; 2:
// da_y_film / da_y_update* take the y-chain weights k-major ((in, out)), da_edge_layer_stats resets its ticket word itself
int da_abi_version(void) { return 3; }
int da_stream_create(void** stream) {
  DA_CHECK_ARG(stream, "da_stream_create: null pointer");
  hipStream_t s = nullptr;
  const hipError_t e = hipStreamCreateWithFlags(&s, hipStreamNonBlocking);
  if (e != hipSuccess) { da_set_error("da_stream_create: %s", hipGetErrorString(e)); return DA_ERR_HIP; }
  *stream = (void*)s;
  return DA_OK;
}
}
