// What the host side of the product and of the log probabilities asks of the runtime: the launches of
// each call and the memory it takes. The runtime's calls that they make are answered here, without a
// device (this program's definitions come before the runtime library's), and memory ends where the
// test says. Compiled and run by tests/test_dense_host_cpu.py.
//
// Commands, one an argument:
//   product:TOKENS,ROWS,COLS     logprobs:ROWS,VOCAB,DTYPE,TOP     memory:BYTES     capture:0|1
// Prints a line for each call: its status, then grid x, grid y and threads of each launch; at the end the
// sizes of the allocations.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "host_common.hpp"

namespace {
struct Launch {
    dim3 grid, block;
};
std::vector<Launch> launches;
std::vector<size_t> regions;
size_t room = ~size_t(0), next_address = size_t(1) << 40;
bool capturing = false;
hipError_t last = hipSuccess;
dim3 pushed_grid, pushed_block;
}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
hipError_t hipMalloc(void** p, size_t n) {
    if (n > room) return last = hipErrorOutOfMemory;
    room -= n;
    regions.push_back(n);
    *p = reinterpret_cast<void*>(next_address);
    next_address += (n + 4095) / 4096 * 4096;
    return hipSuccess;
}
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    return *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) {
    return pushed_grid = grid, pushed_block = block, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* s) {
    return *grid = pushed_grid, *block = pushed_block, *shared = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
    return launches.push_back(Launch{grid, block}), hipSuccess;
}
}

int main(int argc, char** argv) {
    objeta_hip_context ctx;
    int stream = 0;
    auto at = [](uint64_t i) { return reinterpret_cast<void*>(i << 44); };  // never read
    for (int i = 1; i < argc; ++i) {
        const char* values = std::strchr(argv[i], ':');
        if (!values) return 2;
        unsigned long long v[4] = {};
        std::sscanf(values, ":%llu,%llu,%llu,%llu", &v[0], &v[1], &v[2], &v[3]);
        launches.clear();
        int32_t rc = 0;
        if (!std::strncmp(argv[i], "memory:", 7)) {
            room = v[0];
            continue;
        } else if (!std::strncmp(argv[i], "capture:", 8)) {
            capturing = v[0] != 0;
            continue;
        } else if (!std::strncmp(argv[i], "product:", 8)) {
            rc = objeta_hip_i8_product_device(&ctx, &stream, v[0], v[1], v[2], static_cast<int8_t*>(at(1)), v[2],
                                              static_cast<float*>(at(2)), static_cast<int8_t*>(at(3)), v[2],
                                              static_cast<float*>(at(4)), nullptr, 2, at(5), v[1]);
        } else if (!std::strncmp(argv[i], "logprobs:", 9)) {
            rc = objeta_hip_log_probs_device(&ctx, &stream, v[0], v[1], static_cast<int32_t>(v[2]), at(1), v[1], 1.0f, nullptr, 0,
                                             nullptr, static_cast<float*>(at(2)), nullptr, v[3],
                                             v[3] ? static_cast<int32_t*>(at(3)) : nullptr, nullptr);
        } else {
            return 2;
        }
        std::printf("%d", rc);
        for (const Launch& l : launches) std::printf(" %u,%u,%u", l.grid.x, l.grid.y, l.block.x);
        std::printf("\n");
    }
    std::printf("regions");
    for (size_t n : regions) std::printf(" %zu", n);
    std::printf("\n");
    return 0;
}
