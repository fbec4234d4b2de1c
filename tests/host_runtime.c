/* A stand-in for the CUDA runtime on host memory, for tests of the library's host code without a
 * GPU: allocations and copies are the host's, kernels are recorded and not run, and the n-th
 * allocation from now can be made to fail.  Linked with the library's object files in place of the
 * runtime. */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

enum { kOk = 0, kInvalidValue = 1, kNoMemory = 2, kKernels = 256, kLaunches = 4096 };

typedef struct {
    const void *host;
    char name[256];
    int smem;                /* its largest dynamic shared memory, as last set */
} Kernel;
static Kernel g_kernels[kKernels];
static int g_n_kernels;
static int g_launches[kLaunches];   /* places in g_kernels */
static int g_n_launches, g_fail_at, g_live, g_device;

/* ---- what the tests use */
void fake_fail_alloc(int n) { g_fail_at = n; }   /* 1: the next one; 0: none */
int fake_live_allocs(void) { return g_live; }
int fake_launches(void) { return g_n_launches; }
void fake_forget(void) { g_n_launches = 0; }
const char *fake_launched(int i) { return g_kernels[g_launches[i]].name; }
/* the smallest or largest limit among the kernels whose names hold `part`, -1 without one */
int fake_smem_limit(const char *part, int largest)
{
    int v = -1;
    for (int i = 0; i < g_n_kernels; i++)
        if (strstr(g_kernels[i].name, part) && (v < 0 || (largest ? g_kernels[i].smem > v : g_kernels[i].smem < v)))
            v = g_kernels[i].smem;
    return v;
}

/* ---- registration */
void **__cudaRegisterFatBinary(void *bin) { return (void **)bin; }
void __cudaRegisterFatBinaryEnd(void **h) { (void)h; }
void __cudaUnregisterFatBinary(void **h) { (void)h; }
void __cudaRegisterVar(void **h, char *a, char *b, const char *c, int d, size_t e, int f, int g)
{
    (void)h, (void)a, (void)b, (void)c, (void)d, (void)e, (void)f, (void)g;
}
void __cudaRegisterFunction(void **h, const char *host, char *dev, const char *name, int limit, void *a, void *b,
                            void *c, void *d, int *e)
{
    (void)h, (void)dev, (void)limit, (void)a, (void)b, (void)c, (void)d, (void)e;
    if (g_n_kernels == kKernels) abort();
    Kernel *k = &g_kernels[g_n_kernels++];
    k->host = host;
    k->smem = 48 * 1024;
    strncpy(k->name, name, sizeof(k->name) - 1);
}
static Kernel *find(const void *host)
{
    for (int i = 0; i < g_n_kernels; i++)
        if (g_kernels[i].host == host) return &g_kernels[i];
    abort();
}

/* ---- launches */
typedef struct {
    unsigned x, y, z;
} Dim3;
typedef struct {
    Dim3 grid, block;
    size_t smem;
    void *stream, *attrs;
    unsigned n_attrs;
} Config;
static _Thread_local Config g_pushed;

static int launch(const void *host, size_t smem)
{
    Kernel *k = find(host);
    if ((long long)smem > k->smem) return kInvalidValue;
    if (g_n_launches < kLaunches) g_launches[g_n_launches++] = (int)(k - g_kernels);
    return kOk;
}
unsigned __cudaPushCallConfiguration(Dim3 grid, Dim3 block, size_t smem, void *stream)
{
    g_pushed.grid = grid, g_pushed.block = block, g_pushed.smem = smem, g_pushed.stream = stream;
    return 0;
}
int __cudaPopCallConfiguration(Dim3 *grid, Dim3 *block, size_t *smem, void *stream)
{
    *grid = g_pushed.grid, *block = g_pushed.block, *smem = g_pushed.smem, *(void **)stream = g_pushed.stream;
    return kOk;
}
int cudaLaunchKernel(const void *f, Dim3 grid, Dim3 block, void **args, size_t smem, void *stream)
{
    (void)grid, (void)block, (void)args, (void)stream;
    return launch(f, smem);
}
int cudaLaunchKernelExC(const Config *c, const void *f, void **args)
{
    (void)args;
    if (c->grid.y > 65535u || c->grid.z > 65535u || c->grid.x > 2147483647u) return kInvalidValue;
    return launch(f, c->smem);
}
int cudaFuncSetAttribute(const void *f, int attr, int value)
{
    if (attr == 8) find(f)->smem = value;   /* cudaFuncAttributeMaxDynamicSharedMemorySize */
    return kOk;
}
int cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int *n, const void *f, int t, size_t s, unsigned flags)
{
    (void)f, (void)t, (void)s, (void)flags;
    *n = 1;
    return kOk;
}
int cudaOccupancyMaxActiveClusters(int *n, const void *f, const void *c)
{
    (void)f, (void)c;
    *n = 74;
    return kOk;
}

/* ---- memory */
int cudaMalloc(void **p, size_t n)
{
    *p = NULL;
    if (g_fail_at > 0 && --g_fail_at == 0) return kNoMemory;
    *p = calloc(n ? n : 1, 1);
    g_live++;
    return *p ? kOk : kNoMemory;
}
int cudaFree(void *p)
{
    if (p) g_live--;
    free(p);
    return kOk;
}
int cudaHostAlloc(void **p, size_t n, unsigned flags)
{
    (void)flags;
    *p = calloc(n ? n : 1, 1);
    return *p ? kOk : kNoMemory;
}
int cudaFreeHost(void *p)
{
    free(p);
    return kOk;
}
int cudaHostGetDevicePointer(void **d, void *h, unsigned flags)
{
    (void)flags;
    *d = h;
    return kOk;
}
int cudaMemcpy(void *d, const void *s, size_t n, int kind)
{
    (void)kind;
    memmove(d, s, n);
    return kOk;
}
int cudaMemcpyAsync(void *d, const void *s, size_t n, int kind, void *stream)
{
    (void)kind, (void)stream;
    memmove(d, s, n);
    return kOk;
}
int cudaMemcpy2DAsync(void *d, size_t dp, const void *s, size_t sp, size_t w, size_t h, int kind, void *stream)
{
    (void)kind, (void)stream;
    for (size_t i = 0; i < h; i++) memmove((char *)d + i * dp, (const char *)s + i * sp, w);
    return kOk;
}
int cudaMemsetAsync(void *d, int v, size_t n, void *stream)
{
    (void)stream;
    memset(d, v, n);
    return kOk;
}
int cudaMemcpyFromSymbol(void *d, const void *s, size_t n, size_t off, int kind)
{
    (void)s, (void)off, (void)kind;
    memset(d, 0, n);
    return kOk;
}
int cudaMemcpyToSymbol(const void *d, const void *s, size_t n, size_t off, int kind)
{
    (void)d, (void)s, (void)n, (void)off, (void)kind;
    return kOk;
}
int cudaGetSymbolAddress(void **p, const void *s)
{
    *p = (void *)(uintptr_t)s;
    return kOk;
}
int cudaIpcGetMemHandle(void *h, void *p) { return (void)h, (void)p, kInvalidValue; }
int cudaIpcOpenMemHandle(void **p, ...) { return (void)p, kInvalidValue; }
int cudaIpcCloseMemHandle(void *p) { return (void)p, kInvalidValue; }

/* ---- devices, streams, errors */
int cudaGetDeviceCount(int *n)
{
    *n = 1;
    return kOk;
}
int cudaGetDevice(int *d)
{
    *d = g_device;
    return kOk;
}
int cudaSetDevice(int d)
{
    g_device = d;
    return kOk;
}
int cudaDeviceGetAttribute(int *v, int attr, int dev)
{
    (void)dev;
    *v = attr == 16 ? 148 : 1;   /* cudaDevAttrMultiProcessorCount */
    return kOk;
}
int cudaDeviceSynchronize(void) { return kOk; }
int cudaStreamCreateWithFlags(void **s, unsigned flags)
{
    (void)flags;
    *s = malloc(1);
    return kOk;
}
int cudaStreamDestroy(void *s)
{
    free(s);
    return kOk;
}
int cudaStreamSynchronize(void *s) { return (void)s, kOk; }
int cudaStreamIsCapturing(void *s, int *status)
{
    (void)s;
    *status = 0;
    return kOk;
}
int cudaGetLastError(void) { return kOk; }
const char *cudaGetErrorString(int e) { return e == kNoMemory ? "out of memory" : "error"; }
static int encode_tiled(void) { return 0; }
int cudaGetDriverEntryPoint(const char *name, void **p, unsigned long long flags, int *status)
{
    (void)flags;
    *p = strcmp(name, "cuTensorMapEncodeTiled") ? NULL : (void *)encode_tiled;
    *status = *p ? 0 : 1;
    return kOk;
}
