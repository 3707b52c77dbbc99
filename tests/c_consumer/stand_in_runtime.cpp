// A stand-in for the few HIP runtime calls that the library's launch paths make, for tests of its host code on a machine without a GPU: loaded with
// global symbols in front of the library, it answers for any device and runtime version and keeps a record of what is asked of it.
// Nothing is launched; addresses are never followed.
#include <cstddef>
#include <cstdint>
#include <map>
#include <set>
#include <utility>

struct Dim3 { uint32_t x, y, z; };

static int g_device = 0, g_version = 70000000, g_refuse_attribute = 0, g_last = 0;
static std::map<std::pair<int, const void*>, int> g_limit;          // (device, kernel) -> dynamic shared memory that it may ask for
static std::set<const void*> g_kernels;                              // launched since the last reset
static int64_t g_launches = 0, g_attributes = 0, g_threads = 0, g_workgroups = 0;
static thread_local struct { Dim3 grid, block; size_t shared; void* stream; } t_call;

extern "C" {
void stand_in_device(int d) { g_device = d; }
void stand_in_version(int v) { g_version = v; }
void stand_in_refuse_attribute(int on) { g_refuse_attribute = on; }
int64_t stand_in_kernels() { return (int64_t)g_kernels.size(); }
void stand_in_reset_kernels() { g_kernels.clear(); }
int64_t stand_in_launches() { return g_launches; }
int64_t stand_in_attributes() { return g_attributes; }
int64_t stand_in_workgroups() { return g_workgroups; }              // of all launches
int64_t stand_in_most_threads() { return g_threads; }               // threads of the largest launch along x

int hipGetDevice(int* d) { *d = g_device; return 0; }
int hipRuntimeGetVersion(int* v) { *v = g_version; return 0; }
int hipDeviceGetStreamPriorityRange(int* lo, int* hi) { *lo = 0; *hi = -1; return 0; }
int hipGetLastError() { const int e = g_last; g_last = 0; return e; }
int hipFuncSetAttribute(const void* f, int, int value) {
    ++g_attributes;
    if (g_refuse_attribute) return 1;
    g_limit[{g_device, f}] = value;
    return 0;
}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t shared, void* stream) { t_call = {grid, block, shared, stream}; return 0; }
int __hipPopCallConfiguration(Dim3* grid, Dim3* block, size_t* shared, void** stream) {
    *grid = t_call.grid; *block = t_call.block; *shared = t_call.shared; *stream = t_call.stream;
    return 0;
}
int hipLaunchKernel(const void* f, Dim3 grid, Dim3 block, void**, size_t shared, void*) {
    const auto it = g_limit.find({g_device, f});
    const int64_t threads = (int64_t)grid.x * block.x;
    if (threads > g_threads) g_threads = threads;
    if (shared > 65536 && (it == g_limit.end() || it->second < (int)shared)) return g_last = 1;      // the limit was not raised on this device
    if (threads >= (int64_t)1 << 32 || grid.y > 65535 || grid.z > 65535) return g_last = 9;         // no such configuration
    ++g_launches;
    g_kernels.insert(f);
    g_workgroups += (int64_t)grid.x * grid.y * grid.z;
    return 0;
}
}
