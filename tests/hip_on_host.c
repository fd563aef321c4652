/* The HIP runtime calls of libnemo.so on host memory, for tests of what the
 * library does around its kernels: device memory is the host's, a launch is
 * recorded and computes nothing. Loaded before the library, with its symbols
 * global, in a process of its own. */
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

typedef struct { uint32_t x, y, z; } dim3_t;

/* Launches so far, and the largest number of threads of one of them. */
uint64_t host_launches, host_most_threads;
/* The last address that was handed out, and the last that was taken back. */
void *host_last_malloc, *host_last_free;
/* Called for each launch, if set: its grid and block, and the first argument. */
void (*host_on_launch)(uint32_t grid, uint32_t block, void* first);

static struct { dim3_t grid, block; size_t lds; void* stream; } pushed;

int __hipPushCallConfiguration(dim3_t grid, dim3_t block, size_t lds, void* stream) {
  pushed.grid = grid, pushed.block = block, pushed.lds = lds, pushed.stream = stream;
  return 0;
}
int __hipPopCallConfiguration(dim3_t* grid, dim3_t* block, size_t* lds, void** stream) {
  *grid = pushed.grid, *block = pushed.block, *lds = pushed.lds, *stream = pushed.stream;
  return 0;
}
int hipLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t lds, void* stream) {
  const uint64_t threads = (uint64_t)grid.x * block.x;
  (void)f, (void)lds, (void)stream;
  ++host_launches;
  if (threads > host_most_threads) host_most_threads = threads;
  if (host_on_launch) host_on_launch(grid.x, block.x, args[0]);
  return 0;
}

int hipMalloc(void** p, size_t n) { return (host_last_malloc = *p = calloc(1, n)) ? 0 : 2; }
int hipFree(void* p) { return free(host_last_free = p), 0; }
int hipHostMalloc(void** p, size_t n, unsigned flags) { return (void)flags, hipMalloc(p, n); }
int hipHostFree(void* p) { return free(p), 0; }
int hipMemcpy(void* to, const void* from, size_t n, int kind) { return (void)kind, memcpy(to, from, n), 0; }
int hipMemcpyAsync(void* to, const void* from, size_t n, int kind, void* s) {
  return (void)s, hipMemcpy(to, from, n, kind);
}
int hipMemcpy2D(void* to, size_t tp, const void* from, size_t fp, size_t w, size_t h, int kind) {
  (void)kind;
  for (size_t i = 0; i < h; ++i) memcpy((char*)to + i * tp, (const char*)from + i * fp, w);
  return 0;
}
int hipMemcpy2DAsync(void* to, size_t tp, const void* from, size_t fp, size_t w, size_t h, int kind, void* s) {
  return (void)s, hipMemcpy2D(to, tp, from, fp, w, h, kind);
}
int hipGetSymbolAddress(void** p, const void* symbol) { return (void)symbol, hipMalloc(p, 64 << 20); }
int hipGetDeviceCount(int* n) { return *n = 1, 0; }
int hipGetDevice(int* d) { return *d = 0, 0; }
int hipSetDevice(int d) { return (void)d, 0; }
int hipDeviceSynchronize(void) { return 0; }
int hipGetLastError(void) { return 0; }
const char* hipGetErrorString(int e) { return (void)e, "error on the host"; }
int hipFuncSetAttribute(const void* f, int a, int v) { return (void)f, (void)a, (void)v, 0; }
int hipStreamCreateWithFlags(void** s, unsigned flags) { return (void)flags, hipMalloc(s, 8); }
int hipStreamDestroy(void* s) { return free(s), 0; }
int hipStreamSynchronize(void* s) { return (void)s, 0; }
int hipStreamWaitEvent(void* s, void* e, unsigned flags) { return (void)s, (void)e, (void)flags, 0; }
int hipEventCreate(void** e) { return hipMalloc(e, 8); }
int hipEventCreateWithFlags(void** e, unsigned flags) { return (void)flags, hipMalloc(e, 8); }
int hipEventDestroy(void* e) { return free(e), 0; }
int hipEventRecord(void* e, void* s) { return (void)e, (void)s, 0; }
int hipEventSynchronize(void* e) { return (void)e, 0; }
int hipEventElapsedTime(float* ms, void* a, void* b) { return (void)a, (void)b, *ms = 0, 0; }
