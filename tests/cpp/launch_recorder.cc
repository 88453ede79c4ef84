// Stands in for the HIP runtime in a process without a GPU: two gfx950 devices, and a list of the kernels
// that the library launches, checked as the runtime checks them. Nothing runs. Loaded with RTLD_GLOBAL in
// front of libqvh.so (tests/launches.py).
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

struct Launch {
  std::string name;
  dim3 grid, block;
  size_t lds;
  int device;
  std::vector<char> argument;  // its first one, where recorder_keep asked for it
};

std::unordered_map<const void*, std::string>& names() {
  static std::unordered_map<const void*, std::string> n;
  return n;
}
std::vector<Launch> g_launches;
int g_device = 1;  // not the library's, which is 0
hipError_t g_error = hipSuccess;
std::string g_kept;
size_t g_kept_bytes = 0;
struct Config {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
} g_config;
void* g_module = nullptr;

}  // namespace

extern "C" {

void** __hipRegisterFatBinary(const void*) { return &g_module; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  names()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
  g_config = {grid, block, lds, stream};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
  *grid = g_config.grid;
  *block = g_config.block;
  *lds = g_config.lds;
  *stream = g_config.stream;
  return hipSuccess;
}

hipError_t hipGetDeviceCount(int* n) {
  *n = 2;
  return hipSuccess;
}
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_t* p, int) {
  std::memset(p, 0, sizeof(*p));
  std::strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipSetDevice(int device) {
  g_device = device;
  return hipSuccess;
}
hipError_t hipGetDevice(int* device) {
  *device = g_device;
  return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetLastError() {
  const hipError_t e = g_error;
  g_error = hipSuccess;
  return e;
}

/// Refuses what the runtime refuses: an empty grid, or 2^32 threads and more along an axis.
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t lds, hipStream_t) {
  const unsigned g[3] = {grid.x, grid.y, grid.z}, b[3] = {block.x, block.y, block.z};
  for (int i = 0; i < 3; ++i) {
    const unsigned long long threads = static_cast<unsigned long long>(g[i]) * b[i];
    if (threads == 0 || threads >= 1ull << 32) return g_error = hipErrorInvalidConfiguration;
  }
  g_launches.push_back({names()[f], grid, block, lds, g_device, {}});
  if (g_kept_bytes > 0 && names()[f].find(g_kept) != std::string::npos) {
    const char* p = static_cast<const char*>(args[0]);
    g_launches.back().argument.assign(p, p + g_kept_bytes);
  }
  return hipSuccess;
}

int recorder_count() { return static_cast<int>(g_launches.size()); }
const char* recorder_name(int i) { return g_launches[i].name.c_str(); }
void recorder_shape(int i, unsigned long long* out) {
  const Launch& l = g_launches[i];
  const unsigned long long v[7] = {l.grid.x, l.grid.y, l.block.x, l.grid.z, l.lds, static_cast<unsigned long long>(l.device), 0};
  std::memcpy(out, v, sizeof(v));
}
/// From now on, kernels whose name holds `part` leave the bytes of their first argument, of which there are so many.
void recorder_keep(const char* part, size_t bytes) {
  g_kept = part;
  g_kept_bytes = bytes;
}
/// They, or null.
const void* recorder_argument(int i) { return g_launches[i].argument.empty() ? nullptr : g_launches[i].argument.data(); }
void recorder_clear() { g_launches.clear(); }
/// The name of the i-th kernel that the library holds, null behind the last.
const char* recorder_kernel(int i) {
  static std::vector<const char*> all = [] {
    std::vector<const char*> v;
    for (const auto& n : names()) v.push_back(n.second.c_str());
    return v;
  }();
  return i < static_cast<int>(all.size()) ? all[i] : nullptr;
}
int recorder_device() { return g_device; }

}  // extern "C"
