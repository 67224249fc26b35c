// The HIP runtime calls that the libraries make, answered on the host: memory is host memory, a launch is written down and runs
// nothing.  Loaded in front of the real runtime, for tests of what the libraries check, allocate and launch, from which thread and in
// which order.
#include <unistd.h>

#include <atomic>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

#include <hip/hip_runtime_api.h>

namespace {

struct Launch {
    std::string name;  // "graph" for a recording
    size_t thread;
    unsigned grid, block, lds;
};

std::mutex guard;
// made when first used and never taken down: the libraries register their kernels before this file's own objects would exist
std::map<const void*, std::string>& kernels() { static auto* m = new std::map<const void*, std::string>(); return *m; }
std::vector<Launch>& launches() { static auto* v = new std::vector<Launch>(); return *v; }
std::map<void*, size_t>& memory() { static auto* m = new std::map<void*, size_t>(); return *m; }
std::atomic<long> streams{1};
thread_local hipStream_t capturing;
int pause_us;

void write_down(const std::string& name, unsigned grid, unsigned block, unsigned lds)
{
    {
        std::lock_guard<std::mutex> g(guard);
        launches().push_back({name, std::hash<std::thread::id>()(std::this_thread::get_id()), grid, block, lds});
    }
    if (pause_us) usleep(pause_us);  // the other thread's turn, if it may have one
}

hipError_t take(void** p, size_t bytes)
{
    *p = std::aligned_alloc(256, (bytes + 255) & ~(size_t)255);
    if (!*p) return hipErrorOutOfMemory;
    std::lock_guard<std::mutex> g(guard);
    memory()[*p] = bytes;
    return hipSuccess;
}

hipError_t give(void* p)
{
    std::lock_guard<std::mutex> g(guard);
    if (p && !memory().erase(p)) return hipErrorInvalidValue;
    std::free(p);
    return hipSuccess;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------- for the tests
void host_pause(int us) { pause_us = us; }
int host_launches() { std::lock_guard<std::mutex> g(guard); return (int)launches().size(); }
size_t host_launch(int i, char* name, int size, unsigned* shape)
{
    std::lock_guard<std::mutex> g(guard);
    const Launch& l = launches()[i];
    strncpy(name, l.name.c_str(), size - 1);
    shape[0] = l.grid, shape[1] = l.block, shape[2] = l.lds;
    return l.thread;
}
size_t host_memory() { std::lock_guard<std::mutex> g(guard); size_t n = 0; for (auto& m : memory()) n += m.second; return n; }

// ---------------------------------------------------------------- the runtime
void** __hipRegisterFatBinary(const void*) { static void* handle; return &handle; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, dim3*, dim3*, int*)
{
    std::lock_guard<std::mutex> g(guard);
    kernels()[host] = name;
}

hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int)
{
    memset(p, 0, sizeof *p);
    strcpy(p->name, "host");
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256, p->warpSize = 64, p->maxThreadsPerBlock = 1024, p->sharedMemPerBlock = 160 << 10;
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error of the host's runtime"; }

hipError_t hipMalloc(void** p, size_t bytes) { return take(p, bytes); }
hipError_t hipFree(void* p) { return give(p); }
hipError_t hipHostMalloc(void** p, size_t bytes, unsigned) { return take(p, bytes); }
hipError_t hipHostFree(void* p) { return give(p); }
hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind) { memcpy(to, from, n); return hipSuccess; }
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind, hipStream_t) { memcpy(to, from, n); return hipSuccess; }
hipError_t hipMemset(void* p, int v, size_t n) { memset(p, v, n); return hipSuccess; }
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { memset(p, v, n); return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) { static char memory[256]; *p = memory; return hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = (hipStream_t)(streams.fetch_add(1) * 16); return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamQuery(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWriteValue64(hipStream_t, void* p, uint64_t v, unsigned) { *(uint64_t*)p = v; return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* c)
{
    *c = s && s == capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipStreamBeginCapture(hipStream_t s, hipStreamCaptureMode) { capturing = s; return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { capturing = nullptr; *g = (hipGraph_t)16; return hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t, hipGraphNode_t*, char*, size_t) { *e = (hipGraphExec_t)16; return hipSuccess; }
hipError_t hipGraphUpload(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { write_down("graph", 0, 0, 0); return hipSuccess; }

hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void**, size_t lds, hipStream_t s)
{
    if (s == capturing && s) return hipSuccess;
    std::string name;
    {
        std::lock_guard<std::mutex> g(guard);
        name = kernels()[f];
    }
    write_down(name, grid.x * grid.y * grid.z, block.x * block.y * block.z, (unsigned)lds);
    return hipSuccess;
}
static thread_local struct { dim3 grid, block; size_t lds; hipStream_t stream; } configuration;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t s)
{
    configuration = {grid, block, lds, s};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* s)
{
    *grid = configuration.grid, *block = configuration.block, *lds = configuration.lds, *s = configuration.stream;
    return hipSuccess;
}

}  // extern "C"
