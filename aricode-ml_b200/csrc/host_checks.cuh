// host_checks.cuh — what entry points refuse with and check arguments by: messages for
// b2_last_error, alignment, rows that share memory.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>

#include "../../include/b2dec.h"

void b2_internal_set_error(const std::string& msg);   // runtime.cu

namespace b2 {

inline int refuse(const char* fn, const std::string& why) {
    b2_internal_set_error(std::string(fn) + ": " + why);
    return B2_E_INVALID;
}

inline int status(const char* fn, cudaError_t e) {
    if (e == cudaSuccess) return B2_OK;
    b2_internal_set_error(std::string(fn) + ": " + cudaGetErrorString(e));
    return B2_E_CUDA;
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool al4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// f32 rows of `width` elements, `ld` apart, read and written 16 bytes at a time
inline bool rows_ok(const float* p, int64_t ld, int64_t width) { return p && al16(p) && ld >= width && ld % 4 == 0; }

// f32 rows as they lie in memory
struct Span {
    const float* p;
    int64_t ld, width;
};

// whether n rows each of a and b may share an element: side by side in one buffer (the
// slices of a fused projection) they do not, and rows that interleave with other strides
// count as sharing
inline bool overlap(const Span& a, const Span& b, int64_t n) {
    if (!a.p || !b.p || n <= 0) return false;
    const int64_t off = ((int64_t)reinterpret_cast<intptr_t>(b.p) - (int64_t)reinterpret_cast<intptr_t>(a.p)) / 4;
    if (off >= (n - 1) * a.ld + a.width || -off >= (n - 1) * b.ld + b.width) return false;
    if (a.ld != b.ld) return true;
    const int64_t at = ((off % a.ld) + a.ld) % a.ld;               // b's column, seen from a's first one
    return at < a.width || at + b.width > a.ld;
}

// memory from the first to the last byte of something, and whether two such share a byte
struct Bytes {
    const void* p;
    int64_t n;
};

inline bool touch(const Bytes& a, const Bytes& b) {
    if (!a.p || !b.p || a.n <= 0 || b.n <= 0) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x < y ? y - x < (uint64_t)a.n : x - y < (uint64_t)b.n;
}

template <int N>
inline bool touch(const Bytes& a, const Bytes (&others)[N]) {
    for (const Bytes& b : others)
        if (touch(a, b)) return true;
    return false;
}

// n rows of `width` elements of `size` bytes, ld apart
inline Bytes rows_bytes(const void* p, int64_t ld, int64_t width, int64_t n, int64_t size) { return {p, ((n - 1) * ld + width) * size}; }

inline bool same(const Span& a, const Span& b) { return a.p == b.p && a.ld == b.ld; }

// the current device's SMs, looked up once a device
inline int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) return n;
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// dynamic shared memory of up to `bytes` for kernel k on the current device, asked for where no
// call there has asked for as much (the question costs as much as a quarter of a launch). A kernel's calls all ask
// for the same, so that one thread never takes back what another has asked for.
template <auto k>
inline cudaError_t allow_smem(int bytes) {
    static std::atomic<int> allowed[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && allowed[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) allowed[dev].store(bytes, std::memory_order_relaxed);
    return e;
}

}  // namespace b2
