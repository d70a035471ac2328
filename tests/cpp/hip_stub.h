// hip_stub.h -- a HIP runtime for tests of the library's HOST logic where there is no GPU: a test program includes this once, links
// libfun_ofdm_amd.so, and the library's runtime calls arrive here instead (a program's own symbols come before a shared library's).
// Memory is host memory, copies are copies, kernels do nothing; what is queued, on which stream, behind which event, is written down in
// order.  An event that was destroyed and is used again is counted, which is what no real runtime reports.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <vector>

namespace stub {

struct Op {
    std::string what;          // "wait" "record" "launch" "copy" "fill" "sync"
    const void *stream, *event;
    std::string name;          // launch: the kernel's symbol
    const void *dst, *src;     // copy / fill
    size_t bytes;
};
struct Stream { unsigned flags; int priority; };
struct Event { bool alive; };

static std::mutex m;
static std::vector<Op> ops;
static std::vector<Stream *> streams;                  // every stream ever made, in order
static std::map<const void *, std::string> &kernels()  // host stub -> symbol (the library registers before this program's globals exist)
{
    static auto *k = new std::map<const void *, std::string>();
    return *k;
}
static int dead_event_uses = 0;
static bool fail_malloc = false, fail_set_device = false;

static void add(const char *what, const void *stream, const void *event = nullptr, const std::string &name = "", const void *dst = nullptr, const void *src = nullptr, size_t bytes = 0)
{
    std::lock_guard<std::mutex> lk(m);
    ops.push_back({ what, stream, event, name, dst, src, bytes });
}
static void use(hipEvent_t e) { if (!((Event *)e)->alive) { std::lock_guard<std::mutex> lk(m); dead_event_uses++; } }
static hipError_t make_stream(hipStream_t *s, unsigned flags, int priority)
{
    std::lock_guard<std::mutex> lk(m);
    streams.push_back(new Stream{ flags, priority });
    *s = (hipStream_t)streams.back();
    return hipSuccess;
}
static std::vector<Op> taken()                         // what was queued since the last look
{
    std::lock_guard<std::mutex> lk(m);
    std::vector<Op> r;
    r.swap(ops);
    return r;
}
struct Config { dim3 grid, block; size_t lds; hipStream_t stream; };
static thread_local Config config;

}  // namespace stub

extern "C" {

hipError_t hipGetDeviceCount(int *n) { *n = 1; return hipSuccess; }
hipError_t hipSetDevice(int) { return stub::fail_set_device ? hipErrorInvalidDevice : hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int)            // (the header renames it to the versioned symbol the library asks for)
{
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
hipError_t hipDeviceGetStreamPriorityRange(int *least, int *greatest) { *least = 1; *greatest = -1; return hipSuccess; }
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) { *n = 2; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "an error of the stub"; }

hipError_t hipMalloc(void **p, size_t n) { if (stub::fail_malloc) return hipErrorOutOfMemory; *p = calloc(1, n ? n : 1); return *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { free(p); return hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { *p = calloc(1, n ? n : 1); return *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipHostFree(void *p) { free(p); return hipSuccess; }
hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind) { memcpy(d, s, n); return hipSuccess; }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind, hipStream_t st) { memcpy(d, s, n); stub::add("copy", st, nullptr, "", d, s, n); return hipSuccess; }
hipError_t hipMemsetAsync(void *d, int v, size_t n, hipStream_t st) { memset(d, v, n); stub::add("fill", st, nullptr, "", d, nullptr, n); return hipSuccess; }
hipError_t hipMemcpyToSymbol(const void *, const void *, size_t, size_t, hipMemcpyKind) { return hipSuccess; }

hipError_t hipStreamCreate(hipStream_t *s) { return stub::make_stream(s, 0, 0); }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned flags) { return stub::make_stream(s, flags, 0); }
hipError_t hipStreamCreateWithPriority(hipStream_t *s, unsigned flags, int priority) { return stub::make_stream(s, flags, priority); }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) { stub::add("sync", s); return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t e, unsigned) { stub::use(e); stub::add("wait", s, e); return hipSuccess; }

hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { *e = (hipEvent_t) new stub::Event{ true }; return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t *e) { return hipEventCreateWithFlags(e, 0); }
hipError_t hipEventDestroy(hipEvent_t e) { ((stub::Event *)e)->alive = false; return hipSuccess; }          // (kept, so that a later use can be told)
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) { stub::use(e); stub::add("record", s, e); return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t e) { stub::use(e); return hipSuccess; }
hipError_t hipEventQuery(hipEvent_t e) { stub::use(e); return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { *ms = 0; return hipSuccess; }

void **__hipRegisterFatBinary(const void *) { static void *p; return &p; }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *, int *) { stub::kernels()[host] = name; }
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) { stub::config = { grid, block, lds, stream }; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream)
{
    *grid = stub::config.grid; *block = stub::config.block; *lds = stub::config.lds; *stream = stub::config.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **, size_t, hipStream_t s) { stub::add("launch", s, nullptr, stub::kernels()[f]); return hipSuccess; }

}  // extern "C"
