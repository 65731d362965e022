// A CUDA runtime without devices, for tests of the library's host code: objects
// of the library linked with it launch nothing.  It keeps, for each of two
// pretended devices, what has been set there, refuses a launch that needs what
// has not been, and notes every launch.
#include <cuda_runtime_api.h>

#include <cstdint>
#include <cstring>
#include <map>
#include <string>
#include <utility>
#include <vector>

namespace {
struct Launch {
  int device;
  unsigned grid, cluster, smem;
};
int g_dev = 0, g_err_word[2];
int g_sms[2] = {148, 148}, g_cluster_ctas[2] = {148, 148};    // SMs; CTAs that run at once in clusters
bool g_wide[2] = {true, true};                                  // clusters of more than 8 allowed
std::map<std::pair<int, const void*>, int> g_smem, g_nonportable;
std::vector<Launch> g_launches;
cudaError_t g_last = cudaSuccess;
std::string g_message;

cudaError_t fail(cudaError_t e) { return g_last = e; }

unsigned cluster_of(const cudaLaunchConfig_t* c) {
  for (unsigned i = 0; i < c->numAttrs; ++i)
    if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) return c->attrs[i].val.clusterDim.x;
  return 1;
}
cudaError_t encode_ok(...) { return cudaSuccess; }
}  // namespace

namespace nnz {
void set_last_error(const std::string& s) { g_message = s; }
int op_device(int** err, int* num_sms) {
  *err = &g_err_word[g_dev];
  *num_sms = g_sms[g_dev];
  return 0;
}
}  // namespace nnz

extern "C" {
// ---- what the compiler's registration code asks for ----
void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }

// ---- the runtime ----
cudaError_t cudaGetDevice(int* d) { *d = g_dev; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int d) { *v = g_sms[d]; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { const cudaError_t e = g_last; g_last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t) { return "a fake error"; }
cudaError_t cudaMemcpyFromSymbol(void*, const void*, size_t, size_t, cudaMemcpyKind) { return cudaSuccess; }

cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int v) {
  if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) g_smem[{g_dev, f}] = v;
  else if (a == cudaFuncAttributeNonPortableClusterSizeAllowed) g_nonportable[{g_dev, f}] = v;
  return cudaSuccess;
}

static cudaError_t may_run(const cudaLaunchConfig_t* c, const void* f) {
  const unsigned cl = cluster_of(c);
  if (c->dynamicSmemBytes > 49152 && c->dynamicSmemBytes > (size_t)g_smem[{g_dev, f}]) return fail(cudaErrorInvalidValue);
  if (cl > 8 && (!g_wide[g_dev] || !g_nonportable[{g_dev, f}])) return fail(cudaErrorInvalidClusterSize);
  return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* f, const cudaLaunchConfig_t* c) {
  if (const cudaError_t e = may_run(c, f)) return e;
  *n = g_cluster_ctas[g_dev] / (int)cluster_of(c);
  return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
  if (const cudaError_t e = may_run(c, f)) return e;
  g_launches.push_back({g_dev, c->gridDim.x * c->gridDim.y * c->gridDim.z, cluster_of(c), (unsigned)c->dynamicSmemBytes});
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *p = reinterpret_cast<void*>(&encode_ok);
  if (q) *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}

// ---- what the tests set and read ----
void fake_use(int device) { g_dev = device; }
void fake_device(int device, int sms, int cluster_ctas, int wide) {
  g_sms[device] = sms;
  g_cluster_ctas[device] = cluster_ctas;
  g_wide[device] = wide != 0;
}
int fake_launches(void) { return (int)g_launches.size(); }
void fake_launch(int i, unsigned* out) { memcpy(out, &g_launches[i], sizeof(Launch)); }
const char* fake_message(void) { return g_message.c_str(); }
}
