// A stand-in for the CUDA runtime, for tests of the library's host code without a GPU: device memory is
// host memory, copies and memsets happen at once, kernels do nothing. It is preloaded into a process of its own
// (tests/fake_cuda.py). A test can make a call fail and read what was called.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

namespace {

struct State {
    std::vector<std::string> calls;
    std::map<const void*, std::string> kernels;
    std::map<const char*, size_t> memory;  // device allocations
    std::string fail_name;
    int fail_at = -1;    // calls of fail_name before the one that fails
    int in_flight = 0;   // copies from pageable memory and memsets of the legacy stream, not yet waited for
    int raced = 0;       // work for another stream while there are some
    cudaError_t last = cudaSuccess;
};
State& st() {
    static State* s = new State;  // (outlives the library's destructors)
    return *s;
}

cudaError_t call(const std::string& name) {
    State& s = st();
    s.calls.push_back(name);
    if (s.fail_at >= 0 && name == s.fail_name && s.fail_at-- == 0) return s.last = cudaErrorUnknown;
    return cudaSuccess;
}

void work_on(cudaStream_t s) {
    if (s && s != cudaStreamLegacy && st().in_flight) st().raced++;
}

bool on_device(const void* p) {
    auto it = st().memory.upper_bound((const char*)p);
    if (it == st().memory.begin()) return false;
    --it;
    return (const char*)p < it->first + it->second;
}

CUresult fake_encode(...) { return CUDA_SUCCESS; }
char symbol[1 << 16];
dim3 push_grid, push_block;
size_t push_smem;
cudaStream_t push_stream;

}  // namespace

extern "C" {

// ---- the test's side ----
void fake_fail(const char* name, int at) {
    st().fail_name = name;
    st().fail_at = at;
}
void fake_clear() {
    st().calls.clear();
    st().fail_at = -1;
}
int fake_in_flight() { return st().in_flight; }
int fake_raced() { return st().raced; }
size_t fake_calls(char* out, size_t cap) {
    std::string all;
    for (const std::string& c : st().calls) all += c + "\n";
    const size_t n = all.size() < cap ? all.size() : cap;
    memcpy(out, all.data(), n);
    return all.size();
}

// ---- registration and launches ----
void** __cudaRegisterFatBinary(void*) {
    static void* handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host, char*, const char* name, int, uint3*, uint3*, dim3*, dim3*, int*) {
    st().kernels[host] = name;
}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t smem, cudaStream_t stream) {
    push_grid = grid;
    push_block = block;
    push_smem = smem;
    push_stream = stream;
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* smem, void* stream) {
    *grid = push_grid;
    *block = push_block;
    *smem = push_smem;
    *(cudaStream_t*)stream = push_stream;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t, cudaStream_t s) {
    work_on(s);
    return call("launch " + st().kernels[f]);
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
    work_on(c->stream);
    return call("launch " + st().kernels[f]);
}
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) {
    *n = 16;
    return cudaSuccess;
}
cudaError_t cudaGetSymbolAddress(void** p, const void*) {
    *p = symbol;
    return cudaSuccess;
}

// ---- the device ----
cudaError_t cudaGetDeviceCount(int* n) {
    *n = 1;
    return cudaSuccess;
}
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->name, "no GPU");
    p->major = 10;
    p->multiProcessorCount = 148;
    return cudaSuccess;
}
cudaError_t cudaGetDevice(int* d) {
    *d = 0;
    return cudaSuccess;
}
cudaError_t cudaSetDevice(int) { return call("cudaSetDevice"); }
cudaError_t cudaDeviceSynchronize() {
    st().in_flight = 0;
    return call("cudaDeviceSynchronize");
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    *fn = (void*)fake_encode;
    if (q) *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
const char* cudaGetErrorString(cudaError_t e) { return e == cudaSuccess ? "no error" : "an error by request"; }
cudaError_t cudaGetLastError() {
    const cudaError_t e = st().last;
    st().last = cudaSuccess;
    return e;
}

// ---- memory ----
cudaError_t cudaMalloc(void** p, size_t n) {
    if (cudaError_t e = call("cudaMalloc")) return e;
    *p = aligned_alloc(256, (n + 255) / 256 * 256);
    memset(*p, 0x5A, n);
    st().memory[(const char*)*p] = n;
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    st().memory.erase((const char*)p);
    free(p);
    return cudaSuccess;
}
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) {
    *p = calloc(1, n);
    return cudaSuccess;
}
cudaError_t cudaFreeHost(void* p) {
    free(p);
    return cudaSuccess;
}
cudaError_t cudaMemGetInfo(size_t* f, size_t* t) {
    *f = *t = 1ull << 37;
    return cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void* p) {
    memset(a, 0, sizeof *a);
    a->type = on_device(p) ? cudaMemoryTypeDevice : cudaMemoryTypeUnregistered;
    return cudaSuccess;
}
cudaError_t cudaMemcpy(void* to, const void* of, size_t n, cudaMemcpyKind kind) {
    if (cudaError_t e = call("cudaMemcpy")) return e;
    memcpy(to, of, n);
    // A copy from pageable memory returns once its source is staged; one to the host waits for the stream.
    if (kind == cudaMemcpyHostToDevice) st().in_flight++;
    else st().in_flight = 0;
    return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void* to, const void* of, size_t n, cudaMemcpyKind, cudaStream_t s) {
    work_on(s);
    if (cudaError_t e = call("cudaMemcpyAsync")) return e;
    memcpy(to, of, n);
    return cudaSuccess;
}
cudaError_t cudaMemcpy2DAsync(void* to, size_t tp, const void* of, size_t fp, size_t w, size_t h, cudaMemcpyKind, cudaStream_t) {
    if (cudaError_t e = call("cudaMemcpy2DAsync")) return e;
    for (size_t i = 0; i < h; i++) memcpy((char*)to + i * tp, (const char*)of + i * fp, w);
    return cudaSuccess;
}
cudaError_t cudaMemset(void* p, int v, size_t n) {
    if (cudaError_t e = call("cudaMemset")) return e;
    memset(p, v, n);
    st().in_flight++;
    return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t s) {
    work_on(s);
    if (cudaError_t e = call("cudaMemsetAsync")) return e;
    memset(p, v, n);
    return cudaSuccess;
}

// ---- streams and events ----
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) {
    *s = (cudaStream_t)malloc(16);
    return cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t s) {
    free(s);
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t s) {
    if (!s || s == cudaStreamLegacy) st().in_flight = 0;
    return call("cudaStreamSynchronize");
}
cudaError_t cudaStreamGetDevice(cudaStream_t, int* d) {
    *d = 0;
    return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) {
    *c = cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaEventCreate(cudaEvent_t* e) {
    *e = (cudaEvent_t)malloc(16);
    return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return cudaEventCreate(e); }
cudaError_t cudaEventDestroy(cudaEvent_t e) {
    free(e);
    return cudaSuccess;
}
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return call("cudaEventRecord"); }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return call("cudaEventSynchronize"); }
cudaError_t cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) {
    *ms = 0;
    return cudaSuccess;
}

}  // extern "C"
