// A stand-in for the HIP runtime on the host: loaded ahead of libtiramisu_hip_wrappers.so it takes that library's calls, launches nothing and keeps a record.
// Kernels go by the names that the library registers them under; allocations are addresses that are no memory, out of as many bytes as are said.
#include <cstdint>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

struct dim3 { uint32_t x, y, z; };
enum { SUCCESS = 0, OUT_OF_MEMORY = 2, INVALID_CONFIGURATION = 9, INVALID_DEVICE = 101 };

namespace {

struct launch { std::string kernel; uint64_t blocks, threads; };
std::map<const void *, std::string> &names() { static std::map<const void *, std::string> n; return n; }
std::vector<launch> launches;
std::map<void *, uint64_t> blocks;
uint64_t memory = ~0ull, allocations = 0, next_address = 1ull << 40;
int last_error = SUCCESS, devices = 2, capturing = 0;
thread_local int device = 0;
std::string text;
struct configuration { dim3 grid, block; size_t shared; void *stream; };
thread_local configuration pushed;

int failed(int e) { return last_error = e; }

}  // namespace

extern "C" {

// ---- what a test says and asks
void recording_memory(uint64_t bytes) { memory = bytes; }
void recording_capture(int on) { capturing = on; }
uint64_t recording_held() { uint64_t n = 0; for (auto &b : blocks) n += b.second; return n; }
uint64_t recording_allocations() { return allocations; }
// the launches so far, a line of kernel, workgroups and threads each; they are forgotten then
const char *recording_launches() {
    text.clear();
    for (const launch &l : launches) text += l.kernel + " " + std::to_string(l.blocks) + " " + std::to_string(l.threads) + "\n";
    launches.clear();
    return text.c_str();
}
const char *recording_kernels() {
    text.clear();
    for (auto &n : names()) text += n.second + "\n";
    return text.c_str();
}

// ---- the runtime
void **__hipRegisterFatBinary(const void *) { static void *handle; return &handle; }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *function, char *, const char *name, unsigned, void *, void *, void *, void *, int *) { names()[function] = name; }
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, void *stream) { pushed = {grid, block, shared, stream}; return SUCCESS; }
int __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *shared, void **stream) {
    *grid = pushed.grid; *block = pushed.block; *shared = pushed.shared; *stream = pushed.stream;
    return SUCCESS;
}
int hipLaunchKernel(const void *function, dim3 grid, dim3 block, void **, size_t, void *) {
    // (threads along each dimension are counted in 32 bits)
    if ((uint64_t)grid.x * block.x > 0xffffffffull || grid.x == 0 || grid.y == 0 || block.x > 1024) return failed(INVALID_CONFIGURATION);
    launches.push_back({names()[function], (uint64_t)grid.x * grid.y, (uint64_t)grid.x * grid.y * block.x});
    return SUCCESS;
}
int hipMalloc(void **p, size_t bytes) {
    if (recording_held() + bytes > memory) return failed(OUT_OF_MEMORY);
    *p = (void *)next_address;
    next_address += (bytes + 4095) / 4096 * 4096;
    blocks[*p] = bytes;
    allocations++;
    return SUCCESS;
}
int hipFree(void *p) { blocks.erase(p); return SUCCESS; }
int hipGetDevice(int *d) { *d = device; return SUCCESS; }
int hipSetDevice(int d) { if (d < 0 || d >= devices) return failed(INVALID_DEVICE); device = d; return SUCCESS; }
int hipGetDeviceCount(int *n) { *n = devices; return SUCCESS; }
int hipGetLastError() { const int e = last_error; last_error = SUCCESS; return e; }
int hipPeekAtLastError() { return last_error; }
const char *hipGetErrorString(int e) { return e == OUT_OF_MEMORY ? "out of memory" : e == INVALID_CONFIGURATION ? "invalid configuration argument" : "error"; }
int hipFuncSetAttribute(const void *, int, int) { return SUCCESS; }
int hipStreamSynchronize(void *) { return SUCCESS; }
int hipDeviceSynchronize() { return SUCCESS; }
int hipStreamIsCapturing(void *, int *status) { *status = capturing; return SUCCESS; }
int hipThreadExchangeStreamCaptureMode(int *) { return SUCCESS; }

}  // extern "C"
