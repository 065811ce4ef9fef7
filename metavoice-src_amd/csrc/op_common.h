// Helpers of the stand-alone operators (mxfp4.hip, logits.hip): error reporting, the device a call works on, grids, buffers that overlap, a fast division.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/metavoice_hip.h"

int mv_fail(int code, const char* fmt, ...);

// Kernels are launched on the device that owns the stream; the null stream names no device, so there the device of `p` (a buffer of the call)
// decides.  The calling thread's current device is restored.  With one device in the process nothing is asked.
class OpDevice {
  public:
    OpDevice(hipStream_t s, const void* p) {
        static const int count = [] {
            int n = 0;
            return hipGetDeviceCount(&n) == hipSuccess ? n : 0;
        }();
        if (count <= 1) return;
        int want = -1, cur = -1;
        if ((status_ = hipGetDevice(&cur)) != hipSuccess) return;
        if (s == nullptr || s == hipStreamLegacy || s == hipStreamPerThread) {
            hipPointerAttribute_t attr;
            if ((status_ = hipPointerGetAttributes(&attr, p)) != hipSuccess) return;
            want = attr.device;
        } else {
            hipDevice_t d = -1;
            if ((status_ = hipStreamGetDevice(s, &d)) != hipSuccess) return;
            want = d;
        }
        if (want != cur && want >= 0) {
            status_ = hipSetDevice(want);
            if (status_ == hipSuccess) prev_ = cur;
        }
    }
    ~OpDevice() {
        if (prev_ >= 0) (void)hipSetDevice(prev_);
    }
    OpDevice(const OpDevice&) = delete;
    OpDevice& operator=(const OpDevice&) = delete;
    hipError_t status() const { return status_; }

  private:
    int prev_ = -1;
    hipError_t status_ = hipSuccess;
};

// n workgroups of up to 512 threads.  A grid's dimension is below 2^32 threads: beyond 2^22 workgroups a second one counts on, and the last workgroups
// find nothing to do.
constexpr int OP_GRID_BITS = 22;
inline dim3 op_grid(uint64_t n) {
    if (n <= 1u << OP_GRID_BITS) return dim3((uint32_t)n);
    return dim3(1u << OP_GRID_BITS, (uint32_t)((n + (1u << OP_GRID_BITS) - 1) >> OP_GRID_BITS));
}
__device__ __forceinline__ uint32_t op_workgroup() { return blockIdx.y << OP_GRID_BITS | blockIdx.x; }

inline bool op_aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// A buffer of a call: `rows` rows of `width` bytes, `stride` >= width apart.  Null: none.
struct OpRows {
    const void* p;
    int64_t rows, stride, width;
};
constexpr int64_t OP_FAR = 1ll << 60;  // a stride beyond it (a single row may have any) is this one here
inline OpRows op_bytes(const void* p, int64_t rows, int64_t width) { return {p, rows, width, width}; }

// Do two buffers share a byte?  Exact where one of them has no gaps or both have the same stride (a row of one may lie in a gap of the other); two
// different strides with gaps are taken to interleave as their owner means them to.
inline bool op_overlap(const OpRows& a, const OpRows& b) {
    typedef __int128 wide;  // sizes that no memory holds do not wrap around
    if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
    const auto solid = [](const OpRows& r) { return r.rows == 1 || r.stride <= r.width; };
    // rows lo .. hi of a grid that begins at byte `at`, against bytes 0 .. n - 1: does the first row that ends behind byte 0 begin before byte n?
    const auto meets = [](wide at, wide lo, wide hi, wide stride, wide width, wide n) {
        stride = std::max(stride, width);
        const wide past = -at - width;
        const wide i = std::max(lo, (past >= 0 ? past / stride : -((stride - 1 - past) / stride)) + 1);
        return i <= hi && at + i * stride < n;
    };
    const wide at = (wide)(uintptr_t)b.p - (wide)(uintptr_t)a.p;
    const wide span_a = (wide)(a.rows - 1) * a.stride + a.width, span_b = (wide)(b.rows - 1) * b.stride + b.width;
    if (at >= span_a || -at >= span_b) return false;
    if (solid(a)) return meets(at, 0, b.rows - 1, b.stride, b.width, span_a);
    if (solid(b)) return meets(-at, 0, a.rows - 1, a.stride, a.width, span_b);
    if (a.stride == b.stride) return meets(at, -(wide)(a.rows - 1), b.rows - 1, b.stride, b.width, a.width);
    return false;
}

// n / d for 0 <= n < 2^31 by a multiply and a shift: the division by an invariant of Granlund and Montgomery (1994), mul = 2^32 (2^shift - d) / d + 1
struct FastDiv {
    uint32_t mul = 0, shift = 0, d = 1;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << shift) < div) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};
