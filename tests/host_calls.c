/* Entry points of the library over a CUDA runtime that only takes notes: this program
 * defines the runtime's functions itself, so nothing here needs or reaches a GPU.
 *
 *   host_calls LIBRARY FAIL CALL...
 *
 * For each CALL it prints "call NAME STATUS", before that "attribute KERNEL",
 * "occupancy KERNEL" and "launch KERNEL" (mangled names) as they were asked for.
 * Attributes and occupancies of kernels whose name contains FAIL are refused. */
#include <dlfcn.h>
#include <stdio.h>
#include <string.h>

#include "moe_b200.h"

static struct { const void* host; const char* name; } kernels[1024];
static int n_kernels;
static const char* fail;

static const char* name_of(const void* host) {
  for (int i = 0; i < n_kernels; ++i)
    if (kernels[i].host == host) return kernels[i].name;
  return "?";
}
static int note(const char* what, const void* host) {
  const char* name = name_of(host);
  printf("%s %s\n", what, name);
  return *fail && strstr(name, fail) ? 999 : 0;
}

typedef struct { unsigned x, y, z; } dim;
static dim grid, block;
static size_t shared;
static void* stream;

void** __cudaRegisterFatBinary(void* b) { static void* h; (void)b; return &h; }
void __cudaRegisterFatBinaryEnd(void** h) { (void)h; }
void __cudaUnregisterFatBinary(void** h) { (void)h; }
void __cudaRegisterVar(void** h, char* a, char* b, const char* c, int d, size_t e, int f, int g) {
  (void)h; (void)a; (void)b; (void)c; (void)d; (void)e; (void)f; (void)g;
}
void __cudaRegisterFunction(void** h, const char* host, char* f, const char* name, int limit, void* a, void* b,
                            void* c, void* d, int* e) {
  (void)h; (void)f; (void)limit; (void)a; (void)b; (void)c; (void)d; (void)e;
  if (n_kernels < 1024) {
    kernels[n_kernels].host = host;
    kernels[n_kernels++].name = name;
  }
}
unsigned __cudaPushCallConfiguration(dim g, dim b, size_t m, void* s) {
  grid = g; block = b; shared = m; stream = s;
  return 0;
}
int __cudaPopCallConfiguration(dim* g, dim* b, size_t* m, void** s) {
  *g = grid; *b = block; *m = shared; *s = stream;
  return 0;
}
int cudaGetDevice(int* d) { *d = 0; return 0; }
int cudaDeviceGetAttribute(int* v, int attr, int d) {
  (void)d;
  *v = attr == 16 ? 148 : attr == 75 ? 10 : 0;   /* multiprocessors, major version */
  return 0;
}
int cudaGetLastError(void) { return 0; }
int cudaFuncSetAttribute(const void* f, int attr, int v) { (void)attr; (void)v; return note("attribute", f); }
int cudaOccupancyMaxActiveClusters(int* n, const void* f, const void* cfg) { (void)cfg; *n = 10; return note("occupancy", f); }
int cudaLaunchKernel(const void* f, dim g, dim b, void** args, size_t m, void* s) {
  (void)g; (void)b; (void)args; (void)m; (void)s;
  note("launch", f);
  return 0;
}
int cudaLaunchKernelExC(const void* cfg, const void* f, void** args) {
  (void)cfg; (void)args;
  note("launch", f);
  return 0;
}
int cudaMemsetAsync(void* p, int v, size_t n, void* s) { (void)p; (void)v; (void)n; (void)s; return 0; }
int cudaStreamSynchronize(void* s) { (void)s; return 0; }
static int encode_tiled(void) { return 0; }
int cudaGetDriverEntryPoint(const char* name, void** fn, unsigned long long flags, int* q) {
  (void)name; (void)flags;
  *fn = (void*)encode_tiled;
  *q = 0;
  return 0;
}

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  void* lib = dlopen(argv[1], RTLD_NOW);
  if (!lib) {
    fprintf(stderr, "%s\n", dlerror());
    return 2;
  }
  fail = argv[2];
  static char memory[64];
  void* p = (void*)((size_t)1 << 30);   /* an address that only the kernels would read */
  for (int i = 3; i < argc; ++i) {
    const char* c = argv[i];
    int st = 999;
    if (!strcmp(c, "norm")) {
      st = ((__typeof__(&moe_rms_norm_1x128))dlsym(lib, "moe_rms_norm_1x128"))(
          p, MOE_BF16, 512, NULL, MOE_BF16, 512, p, MOE_BF16, 1e-6f, 4, 512, NULL, 512, NULL, 512, p, p, NULL);
    } else if (!strcmp(c, "route")) {
      st = ((__typeof__(&moe_route_topk))dlsym(lib, "moe_route_topk"))(
          p, MOE_F32, 64, NULL, MOE_F32, 4, 64, 8, MOE_SCORE_SOFTMAX, 1, 1, MOE_GROUP_MAX, 1, 1.f, p, p, NULL);
    } else if (!strcmp(c, "quantize")) {
      st = ((__typeof__(&moe_fp4_quantize))dlsym(lib, "moe_fp4_quantize"))(p, MOE_BF16, 64, 4, 64, MOE_NVFP4, NULL, p, p,
                                                                           NULL);
    } else if (!strcmp(c, "linear")) {
      st = ((__typeof__(&moe_fp4_linear))dlsym(lib, "moe_fp4_linear"))(p, MOE_BF16, 512, NULL, p, 256, p, NULL, MOE_NVFP4, 4,
                                                                       128, 512, (char*)p + 65536, MOE_BF16, 128, NULL, 0,
                                                                       NULL);
    } else if (!strcmp(c, "matmul")) {
      st = ((__typeof__(&moe_fp4_matmul))dlsym(lib, "moe_fp4_matmul"))(p, 256, p, NULL, p, 256, p, NULL, MOE_NVFP4, 600, 512,
                                                                       512, p, MOE_BF16, 512, NULL);
    } else if (!strcmp(c, "forward")) {
      MoeFwdArgs a;
      memset(&a, 0, sizeof(a));
      a.T = 64, a.H = 512, a.I = 256, a.E_global = a.E_local = 16, a.n_group = 4, a.topk_group = 2, a.top_k = 4;
      a.routed_scaling_factor = 1.f;
      a.routing_logits = a.hidden_states_scale = a.gemm1_weights_scale = a.gemm2_weights_scale = p;
      a.routing_bias = a.hidden_states = a.gemm1_weights = a.gemm2_weights = p;
      a.output = a.workspace = p;
      a.workspace_bytes = (size_t)1 << 30;
      st = ((__typeof__(&moe_fp8_forward))dlsym(lib, "moe_fp8_forward"))(&a, memory);
    }
    printf("call %s %d\n", c, st);
  }
  return 0;
}
