// A HIP runtime of host memory for tests of the library's host code: loaded
// globally before libmimoe.so, its calls take the place of the real ones.
// Allocations can be made to fail, kernels are counted and never run.
#include <cstdlib>
#include <cstring>
#include <map>

namespace {
struct Block { size_t bytes; bool cleared; };
std::map<void*, Block> live;
long fail_at = -1, mallocs = 0, launches = 0, syncs = 0;
int last_error = 0;     // kept until hipGetLastError takes it
int unordered = 0;      // launches while a clear on the default stream may still run
bool clearing = false;
struct Dim3 { unsigned x, y, z; };
struct Config { Dim3 g, b; size_t shared; void* stream; } config;
constexpr int kOutOfMemory = 2;
}  // namespace

extern "C" {
// ---------------------------------------------------------------- for the tests
int fake_last_error() { return last_error; }
void fake_fail_at(long n) { fail_at = n; mallocs = 0; }   // the n-th allocation from now on fails (-1: none)
long fake_mallocs() { return mallocs; }
long fake_launches() { return launches; }
long fake_syncs() { return syncs; }
int fake_unordered() { return unordered; }
long fake_live(size_t* sizes, int* cleared, long max) {
  long i = 0;
  for (const auto& b : live) {
    if (i < max) { sizes[i] = b.second.bytes; cleared[i] = b.second.cleared; }
    ++i;
  }
  return i;
}

// ---------------------------------------------------------------- the runtime
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int, int) { *v = 65536; return 0; }
int hipMalloc(void** p, size_t bytes) {
  *p = nullptr;
  if (mallocs++ == fail_at) return last_error = kOutOfMemory;
  *p = std::malloc(bytes);
  live[*p] = Block{bytes, false};
  return 0;
}
int hipFree(void* p) {
  live.erase(p);
  std::free(p);
  return 0;
}
int hipHostMalloc(void** p, size_t bytes, unsigned) {
  const int e = hipMalloc(p, bytes);
  if (!e) std::memset(*p, 0, bytes);
  return e;
}
int hipHostFree(void* p) { return hipFree(p); }
int hipMemset(void* p, int v, size_t bytes) {
  std::memset(p, v, bytes);
  const auto it = live.find(p);
  if (it != live.end() && it->second.bytes == bytes) it->second.cleared = true;
  clearing = true;
  return 0;
}
int hipMemcpyAsync(void* d, const void* s, size_t bytes, int, void*) { std::memcpy(d, s, bytes); return 0; }
int hipMemcpy(void* d, const void* s, size_t bytes, int) { std::memcpy(d, s, bytes); return 0; }
int hipStreamCreateWithFlags(void** s, unsigned) { *s = std::malloc(1); return 0; }
int hipStreamDestroy(void* s) { std::free(s); return 0; }
int hipStreamWaitEvent(void*, void*, unsigned) { return 0; }
int hipLaunchHostFunc(void*, void (*fn)(void*), void* data) { fn(data); return 0; }
int hipStreamSynchronize(void* s) { ++syncs; if (!s) clearing = false; return 0; }
int hipDeviceSynchronize() { clearing = false; return 0; }
int hipStreamIsCapturing(void*, int* s) { *s = 0; return 0; }
int hipEventCreate(void** e) { *e = std::malloc(1); return 0; }
int hipEventCreateWithFlags(void** e, unsigned) { return hipEventCreate(e); }
int hipEventDestroy(void* e) { std::free(e); return 0; }
int hipEventRecord(void*, void*) { return 0; }
int hipEventSynchronize(void*) { return 0; }
int hipEventElapsedTime(float* ms, void*, void*) { *ms = 1.0f; return 0; }
int hipGetSymbolAddress(void** p, const void*) {
  static void* scratch = std::malloc((size_t)64 << 20);
  *p = scratch;
  return 0;
}
int hipFuncSetAttribute(const void*, int, int) { return 0; }
int hipGetLastError() {
  const int e = last_error;
  last_error = 0;
  return e;
}
const char* hipGetErrorString(int e) { return e ? "out of memory" : "no error"; }
int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t shared, void* stream) {
  config = Config{g, b, shared, stream};
  return 0;
}
int __hipPopCallConfiguration(Dim3* g, Dim3* b, size_t* shared, void** stream) {
  *g = config.g;
  *b = config.b;
  *shared = config.shared;
  *stream = config.stream;
  return 0;
}
int hipLaunchKernel(const void*, Dim3, Dim3, void**, size_t, void*) {
  ++launches;
  unordered += clearing;
  return 0;
}
}
