/* A stand-in for the parts of the CUDA runtime that the serving operators call, preloaded before the real one: two devices
 * of 148 SMs, every call recorded with the device that is current, nothing launched. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

typedef struct { unsigned x, y, z; } dim;
typedef struct { dim grid, block; size_t smem; void* stream; void* attrs; unsigned n; } launch_config;

static int device = 0;
static int sets = 0, fail_set = 0;
static char text[1 << 16];
static size_t used = 0;

static void note(const char* what, unsigned grid, const void* stream) {
  if (used < sizeof text - 128)
    used += snprintf(text + used, sizeof text - used, "%s %d %u %llu\n", what, device, grid, (unsigned long long)(uintptr_t)stream);
}

const char* fake_log(void) { return text; }
void fake_clear(void) { used = 0; text[0] = 0; sets = 0; }
int fake_sets(void) { return sets; }
void fake_fail_set(int on) { fail_set = on; }

int cudaGetDeviceCount(int* n) { *n = 2; return 0; }
int cudaGetDevice(int* d) { *d = device; return 0; }
int cudaSetDevice(int d) { ++sets; if (fail_set) return 101; device = d; return 0; }
int cudaDeviceGetAttribute(int* v, int attr, int d) {
  (void)d;
  *v = attr == 75 ? 10 : attr == 76 ? 0 : attr == 16 ? 148 : attr == 97 ? 232448 : 1;
  return 0;
}
int cudaGetLastError(void) { return 0; }
int cudaStreamCreateWithFlags(void** s, unsigned f) { (void)f; *s = (void*)(uintptr_t)(0x5000 + device); return 0; }
int cudaStreamDestroy(void* s) { (void)s; return 0; }
int cudaMalloc(void** p, size_t n) { *p = calloc(1, n); return 0; }
int cudaFree(void* p) { free(p); return 0; }
int cudaMemset(void* p, int v, size_t n) { memset(p, v, n); return 0; }
int cudaMemcpy(void* d, const void* s, size_t n, int k) { (void)k; memcpy(d, s, n); return 0; }
int cudaDeviceGetDefaultMemPool(void** p, int d) { (void)p; (void)d; return 801; }
int cudaFuncSetAttribute(const void* f, int a, int v) { (void)f; (void)a; (void)v; note("attribute", 0, 0); return 0; }
int cudaFuncGetAttributes(void* a, const void* f) { (void)f; memset(a, 0, 64); return 0; }
int cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void* f, int b, size_t s, unsigned g) {
  (void)f; (void)b; (void)s; (void)g; *n = 1; return 0;
}
static int nothing(void) { return 0; }
int cudaGetDriverEntryPoint(const char* name, void** f, unsigned long long flags, int* q) {
  (void)name; (void)flags; (void)q;
  *f = (void*)nothing;
  return 0;
}
/* clusters of x CTAs on 148 SMs, with as many CTAs an SM as 227 KB hold */
int cudaOccupancyMaxActiveClusters(int* n, const void* f, const launch_config* c) {
  (void)f;
  unsigned x = c->grid.x ? c->grid.x : 1;
  *n = (int)(148 * (232448 / (c->smem + 1024 ? c->smem + 1024 : 1)) / x);
  note("occupancy", x, 0);
  return 0;
}
int cudaLaunchKernelExC(const launch_config* c, const void* f, void** args) {
  (void)f; (void)args;
  note("launch", c->grid.x, c->stream);
  return 0;
}
