/* A stand-in for the CUDA driver and NVRTC, for tests of what the host enqueues
 * and in which order: device memory is host memory, copies happen at once,
 * kernels do nothing, and every call that orders or enqueues work is a line of
 * the file named by FAKE_CUDA_LOG:
 *   <thread> launch <stream> <kernel> <grid> <threads> <dynamic shared memory>
 *   <thread> begin <stream> <kernel>     (before a launch that FAKE_CUDA_SLOW delays)
 *   <thread> record <stream> <event> | wait <stream> <event> | sync <stream>
 *   <thread> copy <stream> | create <stream> | load
 *   <thread> compile <seconds>           (1 where the source has the text FAKE_CUDA_SLOW_COMPILE, else 0)
 * As the driver, it refuses a launch of over 48 KB of shared memory that was not
 * asked for; of the static kind it takes every kernel to have a quarter KB.
 * Built and loaded by fake_driver.py. No GPU is involved. */
#define _GNU_SOURCE
#include <cuda.h>
#include <nvrtc.h>
#include <pthread.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
static FILE* out;
static unsigned long handles = 0x1000;

static void say(const char* format, ...) {
    va_list args;
    va_start(args, format);
    pthread_mutex_lock(&lock);
    if (out == NULL) out = fopen(getenv("FAKE_CUDA_LOG"), "w");
    fprintf(out, "%d ", gettid());
    vfprintf(out, format, args);
    fputc('\n', out);
    fflush(out);
    pthread_mutex_unlock(&lock);
    va_end(args);
}
static void* handle(void) {
    pthread_mutex_lock(&lock);
    void* h = (void*)(handles += 0x10);
    pthread_mutex_unlock(&lock);
    return h;
}

CUresult cuInit(unsigned int flags) { return CUDA_SUCCESS; }
CUresult cuDriverGetVersion(int* v) { *v = 12090; return CUDA_SUCCESS; }
CUresult cuDeviceGetCount(int* n) { *n = 1; return CUDA_SUCCESS; }
CUresult cuDeviceGet(CUdevice* d, int ordinal) { *d = ordinal; return CUDA_SUCCESS; }
CUresult cuDeviceGetAttribute(int* v, CUdevice_attribute a, CUdevice d) {
    *v = a == CU_DEVICE_ATTRIBUTE_MULTIPROCESSOR_COUNT ? 148
       : a == CU_DEVICE_ATTRIBUTE_COMPUTE_CAPABILITY_MAJOR ? 10 : 0;
    return CUDA_SUCCESS;
}
CUresult cuDeviceGetName(char* name, int n, CUdevice d) { snprintf(name, n, "none"); return CUDA_SUCCESS; }
CUresult cuDevicePrimaryCtxRetain(CUcontext* c, CUdevice d) { *c = handle(); return CUDA_SUCCESS; }
CUresult cuCtxSetCurrent(CUcontext c) { return CUDA_SUCCESS; }
CUresult cuStreamCreate(CUstream* s, unsigned int flags) { *s = handle(); say("create %p", *s); return CUDA_SUCCESS; }
CUresult cuStreamDestroy_v2(CUstream s) { return CUDA_SUCCESS; }
CUresult cuStreamSynchronize(CUstream s) { say("sync %p", s); return CUDA_SUCCESS; }
CUresult cuStreamWaitEvent(CUstream s, CUevent e, unsigned int flags) { say("wait %p %p", s, e); return CUDA_SUCCESS; }
CUresult cuEventCreate(CUevent* e, unsigned int flags) { *e = handle(); return CUDA_SUCCESS; }
CUresult cuEventDestroy_v2(CUevent e) { return CUDA_SUCCESS; }
CUresult cuEventRecord(CUevent e, CUstream s) {
    const char* slow = getenv("FAKE_CUDA_SLOW");
    if (slow != NULL && strcmp(slow, "cuEventRecord") == 0) usleep(400000);
    say("record %p %p", s, e);
    return CUDA_SUCCESS;
}
CUresult cuEventSynchronize(CUevent e) { return CUDA_SUCCESS; }
CUresult cuEventQuery(CUevent e) { return CUDA_SUCCESS; }
CUresult cuEventElapsedTime(float* ms, CUevent a, CUevent b) { *ms = 0; return CUDA_SUCCESS; }
CUresult cuMemAlloc_v2(CUdeviceptr* p, size_t n) {
    void* x = NULL;
    if (posix_memalign(&x, 512, n) != 0) return CUDA_ERROR_OUT_OF_MEMORY;
    *p = (CUdeviceptr)x;
    return CUDA_SUCCESS;
}
CUresult cuMemAllocAsync(CUdeviceptr* p, size_t n, CUstream s) { return cuMemAlloc_v2(p, n); }
CUresult cuMemFree_v2(CUdeviceptr p) { free((void*)p); return CUDA_SUCCESS; }
CUresult cuMemFreeAsync(CUdeviceptr p, CUstream s) { return cuMemFree_v2(p); }
CUresult cuDeviceGetDefaultMemPool(CUmemoryPool* p, CUdevice d) { *p = handle(); return CUDA_SUCCESS; }
CUresult cuMemPoolSetAttribute(CUmemoryPool p, CUmemPool_attribute a, void* v) { return CUDA_SUCCESS; }
CUresult cuMemHostAlloc(void** p, size_t n, unsigned int flags) { *p = malloc(n); return CUDA_SUCCESS; }
CUresult cuMemFreeHost(void* p) { free(p); return CUDA_SUCCESS; }
CUresult cuMemcpyHtoDAsync_v2(CUdeviceptr d, const void* h, size_t n, CUstream s) {
    say("copy %p", s);
    memcpy((void*)d, h, n);
    return CUDA_SUCCESS;
}
CUresult cuMemcpyDtoHAsync_v2(void* h, CUdeviceptr d, size_t n, CUstream s) {
    say("copy %p", s);
    memcpy(h, (void*)d, n);
    return CUDA_SUCCESS;
}
CUresult cuMemcpyDtoDAsync_v2(CUdeviceptr a, CUdeviceptr b, size_t n, CUstream s) {
    say("copy %p", s);
    memcpy((void*)a, (void*)b, n);
    return CUDA_SUCCESS;
}
CUresult cuMemcpyPeerAsync(CUdeviceptr a, CUcontext ca, CUdeviceptr b, CUcontext cb, size_t n, CUstream s) {
    return cuMemcpyDtoDAsync_v2(a, b, n, s);
}
CUresult cuMemsetD32Async(CUdeviceptr p, unsigned int v, size_t n, CUstream s) {
    for (size_t i = 0; i < n; ++i) ((unsigned int*)p)[i] = v;
    return CUDA_SUCCESS;
}
CUresult cuDeviceCanAccessPeer(int* can, CUdevice a, CUdevice b) { *can = 0; return CUDA_SUCCESS; }
CUresult cuCtxEnablePeerAccess(CUcontext c, unsigned int flags) { return CUDA_SUCCESS; }
CUresult cuModuleLoadData(CUmodule* m, const void* image) { *m = handle(); say("load"); return CUDA_SUCCESS; }
struct function { char name[64]; unsigned dynamic; };
CUresult cuModuleGetFunction(CUfunction* f, CUmodule m, const char* name) {
    struct function* x = calloc(1, sizeof *x);
    strncpy(x->name, name, sizeof x->name - 1);
    *f = (CUfunction)x;
    return CUDA_SUCCESS;
}
CUresult cuFuncSetAttribute(CUfunction f, CUfunction_attribute a, int v) {
    if (a == CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES) ((struct function*)f)->dynamic = v;
    return CUDA_SUCCESS;
}
CUresult cuFuncGetAttribute(int* v, CUfunction_attribute a, CUfunction f) { *v = 0; return CUDA_SUCCESS; }
CUresult cuOccupancyMaxActiveBlocksPerMultiprocessor(int* n, CUfunction f, int threads, size_t smem) {
    *n = 1;
    return CUDA_SUCCESS;
}
CUresult cuOccupancyMaxActiveClusters(int* n, CUfunction f, const CUlaunchConfig* c) { *n = 1; return CUDA_SUCCESS; }
CUresult cuLaunchKernelEx(const CUlaunchConfig* c, CUfunction f, void** params, void** extra) {
    const char *name = ((struct function*)f)->name, *slow = getenv("FAKE_CUDA_SLOW");
    const unsigned dynamic = c->sharedMemBytes, asked = ((struct function*)f)->dynamic;
    if (dynamic > asked && dynamic + 256 > 48 * 1024) return CUDA_ERROR_INVALID_VALUE;
    if (slow != NULL && strcmp(slow, name) == 0) {
        say("begin %p %s", c->hStream, name);
        usleep(400000);
    }
    say("launch %p %s %u %u %u", c->hStream, name, c->gridDimX, c->blockDimX, c->sharedMemBytes);
    return CUDA_SUCCESS;
}
CUresult cuTensorMapEncodeTiled(CUtensorMap* m, CUtensorMapDataType type, cuuint32_t rank, void* p,
                                const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                                const cuuint32_t* steps, CUtensorMapInterleave i, CUtensorMapSwizzle s,
                                CUtensorMapL2promotion l, CUtensorMapFloatOOBfill fill) {
    memset(m, 0, sizeof *m);
    return CUDA_SUCCESS;
}
CUresult cuGetErrorName(CUresult r, const char** name) { *name = "error"; return CUDA_SUCCESS; }
CUresult cuGetErrorString(CUresult r, const char** text) { *text = "error"; return CUDA_SUCCESS; }

nvrtcResult nvrtcVersion(int* major, int* minor) { *major = 12; *minor = 9; return NVRTC_SUCCESS; }
nvrtcResult nvrtcCreateProgram(nvrtcProgram* p, const char* source, const char* name, int n, const char* const* headers,
                               const char* const* names) {
    *p = (nvrtcProgram)strdup(source);
    return NVRTC_SUCCESS;
}
nvrtcResult nvrtcCompileProgram(nvrtcProgram p, int n, const char* const* options) {
    const char* slow = getenv("FAKE_CUDA_SLOW_COMPILE");
    const int wait = slow != NULL && strstr((const char*)p, slow) != NULL;
    say("compile %d", wait);
    if (wait) sleep(1);
    return NVRTC_SUCCESS;
}
nvrtcResult nvrtcGetCUBINSize(nvrtcProgram p, size_t* n) { *n = 8; return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetCUBIN(nvrtcProgram p, char* image) { memset(image, 0, 8); return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetPTXSize(nvrtcProgram p, size_t* n) { *n = 8; return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetPTX(nvrtcProgram p, char* image) { memset(image, 0, 8); return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetProgramLogSize(nvrtcProgram p, size_t* n) { *n = 0; return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetProgramLog(nvrtcProgram p, char* log) { return NVRTC_SUCCESS; }
nvrtcResult nvrtcDestroyProgram(nvrtcProgram* p) { free(*p); *p = NULL; return NVRTC_SUCCESS; }
const char* nvrtcGetErrorString(nvrtcResult r) { return "error"; }
