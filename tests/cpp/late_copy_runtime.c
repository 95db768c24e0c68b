/* A CUDA runtime for one host test (tests/test_gradient_set_table.py, by LD_PRELOAD):
 * device memory is host memory, and a copy to it arrives as late as the runtime allows,
 * when its stream is waited for.  cudaMemcpy from pageable memory too returns before. */
#include <stdlib.h>
#include <string.h>

static struct { void* dst; void* staged; size_t n; } pending[64];
static int count;

static int late(void* dst, const void* src, size_t n) {
  pending[count].dst = dst;
  pending[count].staged = malloc(n);
  pending[count].n = n;
  memcpy(pending[count++].staged, src, n);
  return 0;
}
int late_copies(void) { return count; }

int cudaGetDeviceCount(int* n) { *n = 1; return 0; }
int cudaGetDevice(int* d) { *d = 0; return 0; }
int cudaSetDevice(int d) { return d != 0; }
int cudaGetLastError(void) { return 0; }
int cudaMalloc(void** p, size_t n) { *p = calloc(1, n); return *p ? 0 : 2; }
int cudaFree(void* p) { free(p); return 0; }
int cudaMemcpy(void* dst, const void* src, size_t n, int kind) { return kind == 1 ? late(dst, src, n) : (memcpy(dst, src, n), 0); }
int cudaMemcpyAsync(void* dst, const void* src, size_t n, int kind, void* stream) { (void)stream; return cudaMemcpy(dst, src, n, kind); }
int cudaStreamSynchronize(void* stream) {
  (void)stream;
  while (count) {
    --count;
    memcpy(pending[count].dst, pending[count].staged, pending[count].n);
    free(pending[count].staged);
  }
  return 0;
}
int cudaDeviceSynchronize(void) { return cudaStreamSynchronize(0); }
