// entry.cuh -- what the C entry points of the plaintext operators
// (decode_ops.cu, train_ops.cu) share: errors, the device, overlap of what a
// call reads and writes.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/tsgpu.h"

namespace tsg_host {
int noalloc_fail(int code, const char* msg);  // tsgpu.cu: sets the thread's last error
}

namespace {

inline int bad(const char* msg) { return tsg_host::noalloc_fail(TS_ERR_ARG, msg); }

// Makes `device` current for a scope.
struct OnDevice {
    int before = -1;
    cudaError_t status;
    explicit OnDevice(int device) {
        status = cudaGetDevice(&before);
        if (status != cudaSuccess) return;
        if (before == device)
            before = -1;
        else
            status = cudaSetDevice(device);
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

inline int cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return TS_OK;
    const int code = e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver ? TS_ERR_NODEVICE : TS_ERR_CUDA;
    cudaGetLastError();
    return tsg_host::noalloc_fail(code, cudaGetErrorString(e));
}

// A matrix of `rows` rows of `row` bytes, `stride` bytes apart.
struct Region {
    uintptr_t p;
    uint64_t rows, row, stride;
    uint64_t bytes() const { return rows && p ? (rows - 1) * stride + row : 0; }
};

inline Region region(const void* p, uint64_t rows, uint64_t cols, int64_t stride, size_t size) {
    return {reinterpret_cast<uintptr_t>(p), rows, cols * size, (uint64_t)stride * size};
}

inline bool overlap(const Region& a, const Region& b) {
    if (!a.bytes() || !b.bytes() || a.p + a.bytes() <= b.p || b.p + b.bytes() <= a.p) return false;
    if (a.stride != b.stride || !a.stride) return true;
    // column ranges of one wider matrix
    const uint64_t off = a.p <= b.p ? (b.p - a.p) % a.stride : (a.stride - (a.p - b.p) % a.stride) % a.stride;
    return !(off >= a.row && off + b.row <= a.stride);
}

inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr uint64_t kMaxStride = 1ull << 40;

inline bool stride_ok(int64_t s) { return s >= 0 && (uint64_t)s <= kMaxStride; }

inline uint64_t up(uint64_t b) { return (b + 255) & ~255ull; }

// No exception leaves a C entry point (the launch bookkeeping may fail to
// allocate on the host).
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (...) {
        return TS_ERR_OOM;
    }
}

}  // namespace
