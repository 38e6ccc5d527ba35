// A HIP runtime made of host memory, for CPU tests of the library's host code:
// loaded ahead of libmicksum.so (RTLD_GLOBAL), its functions take the place of
// the runtime's.  "Device" memory is malloc memory, copies run at once, kernels
// do not run.  It keeps what the tests ask about:
//   * the calling thread's last error, set by every call that fails (here or by
//     stub_fail) and returned and cleared by hipGetLastError, as HIP has it;
//   * per stream, the operations enqueued since its last synchronization;
//   * the live allocations, frees of memory that is not one of them, and copies
//     whose device side does not lie inside one.
// stub_fail(name, nth, err): the nth call of that function from now on fails
// (stub_fail_from: every call from the nth on).
#include <hip/hip_runtime_api.h>

#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>
#include <map>
#include <mutex>
#include <string>

namespace {
thread_local hipError_t t_last = hipSuccess;
std::mutex g_mu;
struct Fail {
  int nth = 0;
  hipError_t err = hipSuccess;
  bool all = false;  // every call from the nth on
};
std::map<std::string, Fail> g_fail;
std::map<std::string, int> g_calls;
std::map<void *, int> g_pending;  // stream -> operations in flight
std::map<void *, size_t> g_live;
std::map<void *, size_t> g_registered;
int g_bad_frees = 0, g_bad_copies = 0;
std::atomic<int> g_errors{0};

hipError_t ret(hipError_t e) {
  if (e != hipSuccess) t_last = e, ++g_errors;
  return e;
}
// Counts a call; its injected error, if this is the one.
hipError_t enter(const char *name) {
  std::lock_guard<std::mutex> lk(g_mu);
  ++g_calls[name];
  auto it = g_fail.find(name);
  if (it == g_fail.end() || --it->second.nth > 0) return hipSuccess;
  const hipError_t e = it->second.err;
  if (!it->second.all) g_fail.erase(it);
  return e;
}
#define ENTER(name)                          \
  do {                                       \
    const hipError_t e_ = enter(name);       \
    if (e_ != hipSuccess) return ret(e_);    \
  } while (0)
bool capturing();
void enqueue(void *s) {
  if (capturing()) return;
  std::lock_guard<std::mutex> lk(g_mu);
  ++g_pending[s];
}
// Does [p, p + n) lie inside a live allocation?  Counted if not.
bool on_device(const void *p, size_t n) {
  std::lock_guard<std::mutex> lk(g_mu);
  for (auto &a : g_live)
    if ((char *)p >= (char *)a.first && (char *)p + n <= (char *)a.first + a.second) return true;
  ++g_bad_copies;
  return false;
}
bool copy_ok(const void *d, const void *s, size_t n, hipMemcpyKind k) {
  return n == 0 || on_device(k == hipMemcpyHostToDevice ? d : s, n);
}
hipError_t alloc(void **p, size_t n) {
  *p = aligned_alloc(4096, (n + 8191) & ~(size_t)4095);
  memset(*p, 0, (n + 8191) & ~(size_t)4095);
  std::lock_guard<std::mutex> lk(g_mu);
  g_live[*p] = n;
  return hipSuccess;
}
hipError_t release(void *p) {
  if (!p) return hipSuccess;
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_live.erase(p)) {
    ++g_bad_frees;
    return ret(hipErrorInvalidValue);
  }
  free(p);
  return hipSuccess;
}
}  // namespace

extern "C" {
void stub_fail(const char *name, int nth, int err) {
  std::lock_guard<std::mutex> lk(g_mu);
  g_fail[name] = Fail{nth, (hipError_t)err};
}
void stub_fail_from(const char *name, int nth, int err) {
  std::lock_guard<std::mutex> lk(g_mu);
  g_fail[name] = Fail{nth, (hipError_t)err, true};
}
void stub_set_last(int err) { t_last = (hipError_t)err; }
int stub_last(void) { return (int)t_last; }
// Every function called since the last stub_reset, as "name count" lines.
const char *stub_counts(void) {
  static thread_local std::string out;
  std::lock_guard<std::mutex> lk(g_mu);
  out.clear();
  for (auto &c : g_calls) out += c.first + " " + std::to_string(c.second) + "\n";
  return out.c_str();
}
// No counts, no injected failures, no last error.
void stub_reset(void) {
  std::lock_guard<std::mutex> lk(g_mu);
  g_calls.clear();
  g_fail.clear();
  t_last = hipSuccess;
}
int stub_calls(const char *name) {
  std::lock_guard<std::mutex> lk(g_mu);
  return g_calls[name];
}
// In flight on the streams the library made (own) / on the default stream.
int stub_pending(int own) {
  std::lock_guard<std::mutex> lk(g_mu);
  int n = 0;
  for (auto &p : g_pending)
    if ((p.first != nullptr) == (own != 0)) n += p.second;
  return n;
}
int stub_live(void) {
  std::lock_guard<std::mutex> lk(g_mu);
  return (int)g_live.size();
}
int stub_registered(void) {
  std::lock_guard<std::mutex> lk(g_mu);
  return (int)g_registered.size();
}
int stub_errors(void) { return g_errors; }
int stub_bad_frees(void) { return g_bad_frees; }
int stub_bad_copies(void) { return g_bad_copies; }

hipError_t hipGetLastError(void) {
  const hipError_t e = t_last;
  t_last = hipSuccess;
  return e;
}
hipError_t hipPeekAtLastError(void) { return t_last; }
const char *hipGetErrorString(hipError_t e) {
  static thread_local char b[32];
  snprintf(b, sizeof b, "stub error %d", (int)e);
  return b;
}

hipError_t hipGetDeviceCount(int *n) {
  ENTER("hipGetDeviceCount");
  *n = 1;
  return hipSuccess;
}
hipError_t hipGetDevice(int *d) {
  ENTER("hipGetDevice");
  *d = 0;
  return hipSuccess;
}
hipError_t hipSetDevice(int) {
  ENTER("hipSetDevice");
  return hipSuccess;
}
hipError_t hipSetDeviceFlags(unsigned) {
  ENTER("hipSetDeviceFlags");
  return hipSuccess;
}
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
  ENTER("hipGetDeviceProperties");
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) {
  ENTER("hipDeviceGetAttribute");
  *v = 256;
  return hipSuccess;
}
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) {
  ENTER("hipOccupancyMaxActiveBlocksPerMultiprocessor");
  *n = 5;
  return hipSuccess;
}
// (no HSA agent behind this runtime: the library's own queues stay closed)
hipError_t hipFuncGetAttributes(hipFuncAttributes *, const void *) {
  (void)enter("hipFuncGetAttributes");
  return ret(hipErrorInvalidDeviceFunction);
}

hipError_t hipMalloc(void **p, size_t n) {
  ENTER("hipMalloc");
  return alloc(p, n);
}
hipError_t hipHostMalloc(void **p, size_t n, unsigned) {
  ENTER("hipHostMalloc");
  return alloc(p, n);
}
hipError_t hipFree(void *p) {
  ENTER("hipFree");
  return release(p);
}
hipError_t hipHostFree(void *p) {
  ENTER("hipHostFree");
  return release(p);
}
hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned) {
  ENTER("hipHostGetDevicePointer");
  *d = h;
  return hipSuccess;
}
hipError_t hipHostRegister(void *p, size_t n, unsigned) {
  ENTER("hipHostRegister");
  std::lock_guard<std::mutex> lk(g_mu);
  g_registered[p] = n;
  return hipSuccess;
}
hipError_t hipHostUnregister(void *p) {
  ENTER("hipHostUnregister");
  std::lock_guard<std::mutex> lk(g_mu);
  return g_registered.erase(p) ? hipSuccess : ret(hipErrorHostMemoryNotRegistered);
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *base, size_t *size, hipDeviceptr_t p) {
  ENTER("hipMemGetAddressRange");
  std::lock_guard<std::mutex> lk(g_mu);
  for (auto &a : g_live)
    if ((char *)p >= (char *)a.first && (char *)p < (char *)a.first + a.second) {
      *base = a.first;
      *size = a.second;
      return hipSuccess;
    }
  return ret(hipErrorInvalidValue);
}

hipError_t hipMemset(void *p, int v, size_t n) {
  ENTER("hipMemset");
  memset(p, v, n);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void *p, int v, size_t n, hipStream_t s) {
  ENTER("hipMemsetAsync");
  memset(p, v, n);
  enqueue(s);
  return hipSuccess;
}
hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind k) {
  ENTER("hipMemcpy");
  if (!copy_ok(d, s, n, k)) return ret(hipErrorInvalidValue);
  memcpy(d, s, n);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind k, hipStream_t st) {
  ENTER("hipMemcpyAsync");
  if (!copy_ok(d, s, n, k)) return ret(hipErrorInvalidValue);
  memcpy(d, s, n);
  enqueue(st);
  return hipSuccess;
}
hipError_t hipMemcpy2DAsync(void *d, size_t dp, const void *s, size_t sp, size_t w, size_t h, hipMemcpyKind k,
                            hipStream_t st) {
  ENTER("hipMemcpy2DAsync");
  if (h && !copy_ok(d, s, (h - 1) * (k == hipMemcpyHostToDevice ? dp : sp) + w, k)) return ret(hipErrorInvalidValue);
  for (size_t r = 0; r < h; ++r) memcpy((char *)d + r * dp, (const char *)s + r * sp, w);
  enqueue(st);
  return hipSuccess;
}

int stub_capturing(void);
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) {
  ENTER("hipStreamCreateWithFlags");
  *s = (hipStream_t)malloc(16);
  return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t s) {
  ENTER("hipStreamDestroy");
  free(s);
  return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t s) {
  ENTER("hipStreamSynchronize");
  if (stub_capturing()) return ret(hipErrorStreamCaptureUnsupported);
  std::lock_guard<std::mutex> lk(g_mu);
  g_pending[s] = 0;
  return hipSuccess;
}
hipError_t hipStreamQuery(hipStream_t s) { return hipStreamSynchronize(s); }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t e, unsigned) {
  ENTER("hipStreamWaitEvent");
  if (!e) return ret(hipErrorInvalidHandle);
  return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t *e) {
  ENTER("hipEventCreate");
  *e = (hipEvent_t)malloc(16);
  return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t e) {
  ENTER("hipEventDestroy");
  free(e);
  return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t e, hipStream_t) {
  ENTER("hipEventRecord");
  if (!e) return ret(hipErrorInvalidHandle);
  return hipSuccess;
}
hipError_t hipEventQuery(hipEvent_t) {
  ENTER("hipEventQuery");
  return hipSuccess;
}
hipError_t hipEventSynchronize(hipEvent_t) {
  ENTER("hipEventSynchronize");
  return hipSuccess;
}
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) {
  ENTER("hipEventElapsedTime");
  *ms = 1.f;
  return hipSuccess;
}

// Stream capture: one at a time; while it lasts, launches are recorded (not in
// flight) and its stream cannot be synchronized.
static hipStream_t g_capturing = nullptr;
static int g_graphs = 0;  // graphs and executables not destroyed
int stub_capturing(void) { return g_capturing != nullptr; }
int stub_graphs(void) { return g_graphs; }
hipError_t hipStreamBeginCapture(hipStream_t s, hipStreamCaptureMode) {
  ENTER("hipStreamBeginCapture");
  if (g_capturing) return ret(hipErrorIllegalState);
  g_capturing = s;
  return hipSuccess;
}
hipError_t hipStreamEndCapture(hipStream_t s, hipGraph_t *g) {
  const hipError_t e = enter("hipStreamEndCapture");  // (a failed one ends the capture too)
  *g = nullptr;
  if (g_capturing != s) return ret(hipErrorIllegalState);
  g_capturing = nullptr;
  if (e != hipSuccess) return ret(e);
  *g = (hipGraph_t)malloc(16);
  ++g_graphs;
  return hipSuccess;
}
hipError_t hipGraphDestroy(hipGraph_t g) {
  ENTER("hipGraphDestroy");
  free(g);
  --g_graphs;
  return hipSuccess;
}
hipError_t hipGraphInstantiate(hipGraphExec_t *x, hipGraph_t, hipGraphNode_t *, char *, size_t) {
  ENTER("hipGraphInstantiate");
  *x = (hipGraphExec_t)malloc(16);
  ++g_graphs;
  return hipSuccess;
}
hipError_t hipGraphExecDestroy(hipGraphExec_t x) {
  ENTER("hipGraphExecDestroy");
  free(x);
  --g_graphs;
  return hipSuccess;
}
hipError_t hipGraphUpload(hipGraphExec_t, hipStream_t) {
  ENTER("hipGraphUpload");
  return hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t s) {
  ENTER("hipGraphLaunch");
  enqueue(s);
  return hipSuccess;
}

// kernel<<<>>>: the configuration pushed here is popped by the kernel's host
// stub, which then calls hipLaunchKernel.
struct LaunchConfig {
  dim3 grid, block;
  size_t shm;
  hipStream_t s;
};
static thread_local LaunchConfig t_config;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shm, hipStream_t s) {
  t_config = LaunchConfig{grid, block, shm, s};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *shm, hipStream_t *s) {
  *grid = t_config.grid;
  *block = t_config.block;
  *shm = t_config.shm;
  *s = t_config.s;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t s) {
  ENTER("hipLaunchKernel");
  enqueue(s);
  return hipSuccess;
}
hipError_t hipExtLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t s, hipEvent_t, hipEvent_t, int) {
  ENTER("hipExtLaunchKernel");
  enqueue(s);
  return hipSuccess;
}
}

namespace {
bool capturing() { return g_capturing != nullptr; }
}  // namespace
