// Stands in for the HIP runtime's launch: records which thread launches and dawdles, so that calls of two
// threads that may come between each other's launches do.
#include <hip/hip_runtime_api.h>
#include <unistd.h>

#include <mutex>
#include <vector>

static std::mutex m;
static std::vector<int> order;
static thread_local int me = -1;
static char symbol[64];

extern "C" {
void stub_thread(int id) { me = id; }
int stub_order(int* out, int room) {
  std::lock_guard<std::mutex> l(m);
  for (int i = 0; i < (int)order.size() && i < room; ++i) out[i] = order[i];
  const int n = (int)order.size();
  order.clear();
  return n;
}
// (without a device the runtime's own refuse, and a launch ends there)
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
  *grid = *block = dim3(1);
  *lds = 0;
  *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) {
  {
    std::lock_guard<std::mutex> l(m);
    order.push_back(me);
  }
  usleep(5000);
  return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) { return *p = symbol, hipSuccess; }
}
