// Runs entry points of the library on a machine without a device: the runtime's calls that they make are answered here (a program's own definitions come before
// those of the libraries that it loads), launches are written down and launch nothing. What is printed is checked by test_language_launches.py.
#include <hip/hip_runtime_api.h>
#include <sys/resource.h>

#include <atomic>
#include <chrono>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <thread>
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
std::atomic<bool> g_paused{false};
const char* g_pause_at = nullptr;  // a launch of this kernel waits a while before it returns
std::vector<std::pair<char*, size_t>> g_blocks;
size_t g_scan = 0;                 // bytes of a launch's argument that are searched for addresses in the first block
std::vector<long> g_found;

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
    bool pause = false;
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        const unsigned long long blocks = (unsigned long long)grid.x * grid.y * grid.z;
        // (what the runtime asks of a launch: fewer than 2^32 threads along each axis)
        const bool fits = (unsigned long long)grid.x * block.x < 1ull << 32 && (unsigned long long)grid.y * block.y < 1ull << 32;
        const bool fails = !fits || (int)g_launches.size() == g_fail_at;
        g_launches.push_back({name, blocks, (unsigned long long)grid.x * block.x});
        if (g_scan)
            for (size_t at = 0; at + 8 <= g_scan; at += 8) {
                char* p;
                std::memcpy(&p, (const char*)arguments[0] + at, 8);
                if (p >= g_blocks[0].first + 65536 && p < g_blocks[0].first + g_blocks[0].second) g_found.push_back((long)(p - g_blocks[0].first));
            }
        if (fails) return t_error = hipErrorInvalidConfiguration;
        pause = g_pause_at && name.find(g_pause_at) != std::string::npos;
    }
    if (pause) {
        g_paused = true;
        std::this_thread::sleep_for(std::chrono::milliseconds(300));
    }
    return hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = t_error;
    t_error = hipSuccess;
    return e;
}
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) {
    const auto note = [](const char* what) {
        std::lock_guard<std::mutex> lock(g_mutex);
        g_launches.push_back({what, 1, 1});
    };
    note("graph_begins");
    g_paused = true;
    std::this_thread::sleep_for(std::chrono::milliseconds(300));
    note("graph_ends");
    return hipSuccess;
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
    g_blocks.push_back({(char*)*p, bytes});
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
int clip(int dtype, const std::vector<int64_t>& sizes) {
    std::vector<const void*> in;
    std::vector<void*> out;
    for (size_t i = 0; i < sizes.size(); ++i) in.push_back((char*)at(1) + (i << 36)), out.push_back((char*)at(40) + (i << 36));
    return dali_hip_clip_by_global_norm(dtype, (int)sizes.size(), in.data(), out.data(), sizes.data(), 1.0, at(100));
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
                           op == "clip" ? clip(dtype, std::vector<int64_t>(rows, extent)) : op == "norm" ? norm(dtype, rows, extent) : norm_backward(dtype, rows, extent);
        report(op.c_str(), status);
    } else if (what == "threads") {  // the kernel whose launch waits
        g_pause_at = argv[2];
        if (dali_hip_init(0)) return 1;
        int status[2] = {0, 0};
        const bool clip_first = std::strcmp(argv[2], "squares") == 0, graph_first = std::strcmp(argv[2], "graph") == 0;
        std::thread first([&] { status[0] = clip_first ? clip(0, {1 << 20, 77}) : graph_first ? dali_hip_graph_launch(at(1)) : norm_backward(0, 5000, 1024); });
        while (!g_paused) std::this_thread::yield();
        status[1] = clip_first ? norm_backward(0, 5000, 1024) : clip(0, {1 << 20, 77});
        first.join();
        if (status[0] || status[1]) return 1;
        for (const Launch& l : g_launches)
            for (const char* k : {"graph_begins", "graph_ends", "squares", "rescale", "norm_backward_team", "norm_weights", "norm_fold"})
                if (l.kernel.find(k) != std::string::npos) std::printf("%s\n", k);
    } else if (what == "memory") {  // many arrays, and then no memory for what the call notes about them
        if (dali_hip_init(0)) return 1;
        const size_t count = 1 << 23;
        std::vector<const void*> in(count, at(1));
        std::vector<void*> out(count, at(2));
        const std::vector<int64_t> sizes(count, 0);
        rlimit limit;
        getrlimit(RLIMIT_AS, &limit);
        limit.rlim_cur = 64 << 20;  // (less than is in use: nothing more is given)
        if (setrlimit(RLIMIT_AS, &limit)) return 1;
        const int status = dali_hip_clip_by_global_norm(0, (int)count, in.data(), out.data(), sizes.data(), 1.0, at(3));
        std::printf("%d %s\n", status, dali_hip_last_error());
    } else if (what == "places") {
        if (dali_hip_init(0)) return 1;
        // (searched: what the launches' arguments hold at least)
        auto run = [&](const char* name, size_t scan, auto&& call) {
            g_scan = scan;
            std::printf("%s %d", name, call());
            for (long f : g_found) std::printf(" %ld", f);
            std::printf("\n");
            g_found.clear();
        };
        run("one", 104, [&] { return log_probs(0, 1, 50257, 5); });
        run("two", 88, [&] { return norm_backward(0, 5000, 1024); });
        run("two", 88, [&] { return norm_backward(1, 500, 20000); });
        run("two", 480, [&] { return clip(0, {1 << 20, 77}); });
        run("two", 480, [&] { return clip(1, {1 << 20, 77}); });
    } else {
        return 2;
    }
    return 0;
}
