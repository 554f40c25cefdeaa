// Host-side runtime pieces of libpaged_hip: version, per-thread error messages, device queries.
#include <stdarg.h>
#include <string.h>

#include "pa_common.h"
#include "pa_internal.h"

namespace pa_host {

static thread_local char g_last_error[512] = {0};

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

void clear_error() { g_last_error[0] = '\0'; }

int device_cu_count() {
  constexpr int kMaxDevices = 64;
  static int cached[kMaxDevices] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 256;
  if (cached[dev] == 0) {
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
      cus = 256;
    cached[dev] = cus;
  }
  return cached[dev];
}

// (Workspaces of at least 1 MiB, as the wrappers make them, fall on mutexes of their own; others may share one,
// and then wait for each other's launches.)
std::mutex& workspace_mutex(const void* workspace) {
  static std::mutex all[64];
  return all[(reinterpret_cast<uintptr_t>(workspace) >> 20) % 64];
}

}  // namespace pa_host

extern "C" unsigned long long paged_internal_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusNone ? 0 : id;
}

extern "C" int paged_internal_device(void) {
  int dev = -1;
  return hipGetDevice(&dev) == hipSuccess ? dev : -1;
}

extern "C" int pa_version(void) { return 100; }  // 0.1.0

extern "C" const char* pa_last_error_message(void) { return pa_host::g_last_error; }
