// Runs entry points of the library on a machine without a device: the runtime's calls that they make are answered here (a program's own definitions come before
// those of the libraries that it loads), launches are written down and launch nothing. What is printed is checked by test_language_launches.py.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "../include/dali_hip.h"

namespace {

std::map<const void*, std::string>& kernels() {
    static std::map<const void*, std::string> names;
    return names;
}

struct Launch {
    std::string kernel;
    unsigned long long blocks, threads;
};
std::mutex g_mutex;
std::vector<Launch> g_launches;
int g_fail_at = -1;                // number of the launch that fails
thread_local hipError_t t_error = hipSuccess;

struct Configuration {
    dim3 grid, block;
    size_t shared;
    hipStream_t stream;
};
thread_local Configuration t_configuration;

}  // namespace

extern "C" {

void** __hipRegisterFatBinary(const void*) {
    static void* handle = nullptr;
    return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) { kernels()[host] = name; }
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
    t_configuration = {grid, block, shared, stream};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
    *grid = t_configuration.grid, *block = t_configuration.block, *shared = t_configuration.shared, *stream = t_configuration.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3 block, void** arguments, size_t, hipStream_t) {
    const std::string name = kernels()[kernel];
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        const unsigned long long blocks = (unsigned long long)grid.x * grid.y * grid.z;
        // (what the runtime asks of a launch: fewer than 2^32 threads along each axis)
        const bool fits = (unsigned long long)grid.x * block.x < 1ull << 32 && (unsigned long long)grid.y * block.y < 1ull << 32;
        const bool fails = !fits || (int)g_launches.size() == g_fail_at;
        g_launches.push_back({name, blocks, (unsigned long long)grid.x * block.x});
        if (fails) return t_error = hipErrorInvalidConfiguration;
    }
    return hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = t_error;
    t_error = hipSuccess;
    return e;
}
const char* hipGetErrorString(hipError_t) { return "refused by the recorder"; }
hipError_t hipGetDeviceCount(int* count) {
    *count = 1;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_t* p, int) {
    std::memset((void*)p, 0, sizeof(*p));
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
    static int stream;
    *s = (hipStream_t)&stream;
    return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t bytes) {
    *p = std::malloc(bytes);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void* symbol) {
    *p = (void*)symbol;
    return hipSuccess;
}
}  // extern "C"

namespace {

// addresses that are never read: far apart, so that no operand meets another
void* at(int i) { return (void*)((uintptr_t)i << 44); }

void report(const char* what, int status) {
    unsigned long long most = 0, blocks = 0;
    for (const Launch& l : g_launches) most = l.threads > most ? l.threads : most, blocks += l.blocks;
    std::printf("%s %d %zu %llu %llu\n", what, status, g_launches.size(), blocks, most);
    g_launches.clear();
}

int log_probs(int dtype, long rows, int vocab, int k) {
    return dali_hip_token_log_probs(dtype, rows, vocab, at(1), 0, (const int32_t*)at(2), k, at(3), at(4), at(5), k ? at(6) : nullptr, k ? (int32_t*)at(7) : nullptr);
}
int log_probs_backward(int dtype, long rows, int vocab) {
    return dali_hip_token_log_probs_backward(dtype, rows, vocab, at(1), at(2), at(3), 0, (const int32_t*)at(4), at(5), at(6), at(7));
}
int norm(int dtype, long rows, int width) { return dali_hip_layer_norm(dtype, rows, width, at(1), 0, at(2), at(3), 1e-5, at(4), at(5), at(6)); }
int norm_backward(int dtype, long rows, int width) {
    return dali_hip_layer_norm_backward(dtype, rows, width, at(1), 0, at(2), 0, at(3), at(4), at(5), at(6), at(7), at(8));
}

}  // namespace

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "one") {  // operator dtype rows extent k
        const std::string op = argv[2];
        const int dtype = std::atoi(argv[3]), extent = std::atoi(argv[5]);
        const long rows = std::atol(argv[4]);
        if (argc > 7) g_fail_at = std::atoi(argv[7]);
        const int status = op == "log_probs" ? log_probs(dtype, rows, extent, std::atoi(argv[6])) : op == "log_probs_backward" ? log_probs_backward(dtype, rows, extent) :
                           op == "norm" ? norm(dtype, rows, extent) : norm_backward(dtype, rows, extent);
        report(op.c_str(), status);
    } else {
        return 2;
    }
    return 0;
}
