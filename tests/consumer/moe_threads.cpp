// Two host threads in the experts' down product for the first time, on a CUDA
// runtime of this file's own that runs nothing: it keeps each kernel's limit of
// dynamic shared memory and refuses launches above it, as the real one does.
//
// The first thread's limit is set and its call held there until the second
// thread, with fewer tokens, has gone through; both calls and a third one have
// to be launched. Linked against lib/libpopcorn.a without the CUDA runtime.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <condition_variable>
#include <map>
#include <mutex>
#include <thread>

#include <cuda_runtime.h>

#include "popcorn_serve.h"

namespace {

std::mutex lock;
std::condition_variable changed;
std::map<const void*, int> limits;
bool held = false, let_go = false;
int launches = 0, refused = 0;
thread_local int hold_from = 0;  // hold this thread in the first limit of at least so many bytes

cudaError_t launch(const void* kernel, size_t shared) {
    std::lock_guard<std::mutex> g(lock);
    ++launches;
    const auto at = limits.find(kernel);
    if (shared <= 48 * 1024 || (at != limits.end() && shared <= static_cast<size_t>(at->second))) return cudaSuccess;
    ++refused;
    return cudaErrorInvalidValue;
}

}  // namespace

extern "C" {

cudaError_t cudaFuncSetAttribute(const void* kernel, cudaFuncAttribute, int value) {
    std::unique_lock<std::mutex> g(lock);
    limits[kernel] = value;
    if (hold_from > 0 && value >= hold_from && !held) {
        held = true;
        changed.notify_all();
        changed.wait(g, [] { return let_go; });
    }
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* kernel, void**) { return launch(kernel, c->dynamicSmemBytes); }
cudaError_t cudaGetDevice(int* device) { return *device = 0, cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* value, cudaDeviceAttr, int) { return *value = 148, cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
void** __cudaRegisterFatBinary(void*) {
    static void* handle = nullptr;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
}

int main(int argc, char** argv) {
    if (argc != 6) return 2;
    const int64_t K = std::atol(argv[1]), F = 64, E = 2, top = 2;
    const int64_t many = std::atol(argv[2]), few = std::atol(argv[3]);
    const int from = std::atoi(argv[4]), kernels = std::atoi(argv[5]);
    char* const p = reinterpret_cast<char*>(0x10000);  // never dereferenced
    const auto call = [&](int64_t M) {
        float* const f = reinterpret_cast<float*>(p);
        const int8_t* const q = reinterpret_cast<const int8_t*>(p);
        return popcornMoe_i8f32(f, nullptr, nullptr, f, f, q, f, q, f, q, f, M, K, F, E, top, 1, p,
                                popcornMoeWorkspace(M, K, F, E, top), nullptr);
    };
    popcornStatus_t first = POPCORN_ERROR_CUDA, second = POPCORN_ERROR_CUDA;
    std::thread a([&] {
        hold_from = from;
        first = call(many);
    });
    {
        std::unique_lock<std::mutex> g(lock);
        if (!changed.wait_for(g, std::chrono::seconds(30), [] { return held; })) {
            std::printf("the first thread set no limit of %d bytes\n", from);
            std::_Exit(2);
        }
    }
    std::thread b([&] { second = call(few); });
    b.join();
    {
        std::lock_guard<std::mutex> g(lock);
        let_go = true;
    }
    changed.notify_all();
    a.join();
    const popcornStatus_t third = call(many);
    std::printf("status %d %d %d, %d launches, %d refused, %zu kernels with a limit\n", first, second, third, launches, refused,
                limits.size());
    return first || second || third || refused || launches != 9 || limits.size() != static_cast<size_t>(kernels);
}
