// Microscaled 4-bit floating point (MXFP4): quantiser and products.
//
// A row of K values is cut into blocks of 32 columns (the last one may be short).  A block is 32 codes of 4 bits (sign, 2 exponent bits, 1 mantissa
// bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times one power of two, stored as a byte s for 2^(s - 127); s = 255 makes every value of the block NaN.
//   codes  [rows][16 * nb] bytes, nb = ceil(K / 32): column 2j in the low, 2j + 1 in the high nibble of byte j; zero past K
//   scales [rows][nb] bytes
// 4.25 bits per weight.  gfx950 converts codes to bf16 with the scale applied (v_cvt_scalef32_pk_bf16_fp4: two values per instruction; the scale operand
// counts by its exponent bits alone, so s << 23 stands for every byte, 0 = 2^-127 and 255 = NaN among them) and multiplies them directly
// (v_mfma_scale_f32_16x16x128_f8f6f4: a lane brings 32 consecutive codes and their scale byte).  Both exact: a code times a power of two is a bf16
// number, products accumulate in fp32.
#include "common.h"
#include "op_common.h"

#include <algorithm>

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at the alignment of a bf16 element

#define MX_TRY(expr)                                                                                                               \
    do {                                                                                                                           \
        hipError_t _e = (expr);                                                                                                    \
        if (_e != hipSuccess) return mv_fail(MV_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(_e), __FILE__, __LINE__); \
    } while (0)

namespace {

// ---- quantiser --------------------------------------------------------------------------------------------------------------------------
// One thread: 8 columns; the 4 threads of a quad share a block and its largest magnitude.  Memory bound.
struct QuantArgs {
    const void* w;
    unsigned char* codes;
    unsigned char* scales;
    bf16_t* deq;
    int64_t ldw;
    uint32_t chunks;  // 8-column chunks of this launch: rows * nb * 4
    int32_t K, nb;
    FastDiv per_row;  // chunks per row
    int32_t vec_in, vec_out;
};

template <bool F32>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const QuantArgs a) {
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.chunks) return;  // whole quads leave: chunks is a multiple of 4
    const uint32_t row = a.per_row.div(id), c8 = id - row * a.per_row.d;
    const int col = (int)c8 * 8;
    const int left = a.K - col;  // columns from here to the end of the row
    float v[8];
    if (F32) {
        const float* p = (const float*)a.w + (int64_t)row * a.ldw + col;
        if (a.vec_in && left >= 8) {
            const f32x4_t lo = __builtin_nontemporal_load((const f32x4_t*)p), hi = __builtin_nontemporal_load((const f32x4_t*)p + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
        }
    } else {
        const bf16_t* p = (const bf16_t*)a.w + (int64_t)row * a.ldw + col;
        if (a.vec_in && left >= 8) {
            const u32x4 q = __builtin_nontemporal_load((const u32x4*)p);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(q[i]); v[2 * i + 1] = bf_hi(q[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? bf2f(p[i]) : 0.f;
        }
    }
    // magnitudes order like their bits, infinities and NaN on top
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
    const int e = (int)(top >> 23);                                // floor(log2) + 127, 0 below the smallest normal number
    const uint32_t s = e == 255 ? 255u : (uint32_t)max(e - 2, 0);  // 6 = 1.5 * 2^2 is the largest code
    const float scale = __uint_as_float(s << 23);
    uint32_t q = 0;  // ties to the even code, above 6 to 6: the conversion's own rounding
    if (s != 255u) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
    }
    *(uint32_t*)(a.codes + ((int64_t)row * a.nb * 16 + (int64_t)c8 * 4)) = q;
    if ((c8 & 3) == 0) a.scales[(int64_t)row * a.nb + (c8 >> 2)] = (unsigned char)s;
    if (a.deq != nullptr && left > 0) {
        u32x4 d;
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3));
        bf16_t* o = a.deq + (int64_t)row * a.K + col;
        if (a.vec_out && left >= 8) {
            *(u32x4*)o = d;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) o[i] = (bf16_t)(d[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// ---- products ---------------------------------------------------------------------------------------------------------------------------
struct MxArgs {
    const void* x;            // bf16 [M][ldx], or codes [M][16 nb]
    const unsigned char* xs;  // scales of x's codes [M][nb]
    const unsigned char *w, *ws, *w2, *ws2;
    const bf16_t *bias, *bias2;
    const void* res;  // [M][N], the output's type
    void* out;
    int64_t ldx;
    int32_t M, N, K, nb, out_f32;
    uint32_t tiles_n;
};

// y = x . w + bias (gated: silu(y) * (x . w2 + bias2)) + residual, in fp32, rounded once
__device__ __forceinline__ void mx_store(const MxArgs& a, int m, int n, float v, float v2) {
    if (a.bias) v += bf2f(a.bias[n]);
    if (a.w2) {
        if (a.bias2) v2 += bf2f(a.bias2[n]);
        v = v / (1.0f + __expf(-v)) * v2;
    }
    const int64_t at = (int64_t)m * a.N + n;
    if (a.out_f32) {
        if (a.res) v += ((const float*)a.res)[at];
        ((float*)a.out)[at] = v;
    } else {
        if (a.res) v += bf2f(((const bf16_t*)a.res)[at]);
        ((bf16_t*)a.out)[at] = f2bf(v);
    }
}

// 8 bf16 of a row from column c on, zero from column K on
__device__ __forceinline__ u32x4 mx_load_x8(const bf16_t* row, int c, int K) {
    if (c + 8 <= K) return *(const u32x4_any*)(row + c);
    u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < K) r[i >> 1] |= (uint32_t)row[c + i] << (16 * (i & 1));
    return r;
}

__device__ __forceinline__ bf16x8_t mx_widen(uint32_t q, float scale) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3));
    return __builtin_bit_cast(bf16x8_t, r);
}

#define MX_WAVES 8

// One workgroup: 16 weight rows against 16 rows of x; the waves take the 128-column steps of K in turn and their sums meet in LDS, in wave order.
// Lane (r = lane & 15, g = lane >> 4) holds block 4 step + g of weight row r and of x row r.  The weights are the first operand of the matrix
// instruction, so a lane ends with 4 consecutive output columns of one row.
template <bool X4, bool GATED>
__global__ void __launch_bounds__(64 * MX_WAVES) mx_rows_kernel(const MxArgs a) {
    __shared__ f32x4_t part[GATED ? 2 : 1][MX_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const uint32_t tm = blockIdx.x / a.tiles_n, tn = blockIdx.x - tm * a.tiles_n;
    const int m = (int)tm * 16 + r, n = (int)tn * 16 + r;
    const bool has_m = m < a.M, has_n = n < a.N;
    f32x4_t acc[GATED ? 2 : 1];
    acc[0] = f32x4_t{0, 0, 0, 0};
    if (GATED) acc[GATED ? 1 : 0] = f32x4_t{0, 0, 0, 0};
    for (int b0 = wave * 4; b0 < a.nb; b0 += MX_WAVES * 4) {
        const int b = b0 + g;
        const bool in_k = b < a.nb;
        u32x4 wq[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
        uint32_t wsc[2] = {127u, 127u};
        if (in_k && has_n) {
            const int64_t at = (int64_t)n * a.nb + b;
            wq[0] = *(const u32x4*)(a.w + at * 16);
            wsc[0] = a.ws[at];
            if (GATED) {
                wq[1] = *(const u32x4*)(a.w2 + at * 16);
                wsc[1] = a.ws2[at];
            }
        }
        if (X4) {
            u32x4 xq = {0u, 0u, 0u, 0u};
            uint32_t xsc = 127u;
            if (in_k && has_m) {
                const int64_t at = (int64_t)m * a.nb + b;
                xq = *(const u32x4*)((const unsigned char*)a.x + at * 16);
                xsc = a.xs[at];
            }
            const i32x8_t xv = {(int)xq[0], (int)xq[1], (int)xq[2], (int)xq[3], 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < (GATED ? 2 : 1); ++i) {
                const i32x8_t wv = {(int)wq[i][0], (int)wq[i][1], (int)wq[i][2], (int)wq[i][3], 0, 0, 0, 0};
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[i], 4, 4, 0, (int)wsc[i], 0, (int)xsc);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 xv = {0u, 0u, 0u, 0u};
                if (in_k && has_m) xv = mx_load_x8((const bf16_t*)a.x + (int64_t)m * a.ldx, b * 32 + j * 8, a.K);
#pragma unroll
                for (int i = 0; i < (GATED ? 2 : 1); ++i)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_widen(wq[i][j], __uint_as_float(wsc[i] << 23)), __builtin_bit_cast(bf16x8_t, xv), acc[i], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < (GATED ? 2 : 1); ++i) part[i][wave][lane] = acc[i];
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int ln = threadIdx.x >> 2, c = threadIdx.x & 3;  // lane and register of the output element
    float v = 0.f, v2 = 0.f;
#pragma unroll
    for (int w = 0; w < MX_WAVES; ++w) {
        v += part[0][w][ln][c];
        if (GATED) v2 += part[GATED ? 1 : 0][w][ln][c];
    }
    const int om = (int)tm * 16 + (ln & 15), on = (int)tn * 16 + (ln >> 4) * 4 + c;
    if (om < a.M && on < a.N) mx_store(a, om, on, v, v2);
}

hipError_t launch_products(hipStream_t s, MxArgs a, bool x4) {
    a.tiles_n = (uint32_t)((a.N + 15) / 16);
    const int64_t rows_per_launch = std::max<int64_t>(1, 0x7FFFFFFF / (int64_t)a.tiles_n / 16) * 16;  // a grid is below 2^31 workgroups
    const int M = a.M;
    const int64_t x_row = x4 ? (int64_t)a.nb * 16 : a.ldx * 2, y_row = (int64_t)a.N * (a.out_f32 ? 4 : 2);
    for (int64_t m0 = 0; m0 < M; m0 += rows_per_launch) {
        MxArgs b = a;
        b.M = (int)std::min<int64_t>(M - m0, rows_per_launch);
        b.x = (const char*)a.x + m0 * x_row;
        if (x4) b.xs = a.xs + m0 * a.nb;
        if (a.res) b.res = (const char*)a.res + m0 * y_row;
        b.out = (char*)a.out + m0 * y_row;
        const dim3 grid(a.tiles_n * (uint32_t)((b.M + 15) / 16)), block(64 * MX_WAVES);
        if (x4 && a.w2) hipLaunchKernelGGL((mx_rows_kernel<true, true>), grid, block, 0, s, b);
        else if (x4) hipLaunchKernelGGL((mx_rows_kernel<true, false>), grid, block, 0, s, b);
        else if (a.w2) hipLaunchKernelGGL((mx_rows_kernel<false, true>), grid, block, 0, s, b);
        else hipLaunchKernelGGL((mx_rows_kernel<false, false>), grid, block, 0, s, b);
    }
    return hipGetLastError();
}

// the checks that both products share; null: fine
const char* product_fault(int32_t M, int32_t N, int32_t K, const void* codes, const void* scales, const void* codes2, const void* scales2, const void* bias,
                          const void* bias2, const void* residual, int32_t out_dtype, const void* out) {
    if (M < 0 || N < 0 || K < 1) return "M and N must not be negative, K must be positive";
    if (K > 0x7FFFFFFF - 4096) return "K is too large";
    if (out_dtype != MV_BF16 && out_dtype != MV_F32) return "out_dtype must be MV_BF16 or MV_F32";
    if (M == 0 || N == 0) return nullptr;
    if (!codes || !scales || !out) return "null argument";
    if (!codes2 != !scales2) return "codes2 and scales2 go together";
    if (bias2 && !codes2) return "bias2 without codes2";
    if (!op_aligned(codes, 16) || !op_aligned(codes2, 16)) return "codes must be aligned to 16 bytes";
    const size_t esz = out_dtype == MV_F32 ? 4 : 2;
    if (!op_aligned(out, esz) || !op_aligned(residual, esz) || !op_aligned(bias, 2) || !op_aligned(bias2, 2)) return "a buffer is not aligned to its element";
    return nullptr;
}

}  // namespace

extern "C" {

int mv_op_quantize_mxfp4(void* stream, int32_t N, int32_t K, int32_t dtype, const void* w, int64_t ldw, void* codes, void* scales, void* dequantised) {
    if (N < 0 || K < 1 || K > 0x7FFFFFFF - 4096) return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: bad shape N=%d K=%d", N, K);
    if (dtype != MV_BF16 && dtype != MV_F32) return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: dtype %d (MV_BF16 or MV_F32)", dtype);
    if (ldw < K) return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: ldw %lld below K %d", (long long)ldw, K);
    if (N == 0) return MV_OK;
    if (!w || !codes || !scales) return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: null argument");
    const size_t esz = dtype == MV_F32 ? 4 : 2;
    if (!op_aligned(w, esz) || !op_aligned(codes, 16) || !op_aligned(dequantised, 2))
        return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: codes must be aligned to 16 bytes, the other buffers to their element");
    OpDevice dev((hipStream_t)stream, codes);
    MX_TRY(dev.status());
    QuantArgs a;
    a.K = K;
    a.nb = (K + 31) / 32;
    a.per_row = FastDiv((uint32_t)a.nb * 4);
    a.ldw = ldw;
    a.vec_in = op_aligned(w, 16) && (size_t)ldw * esz % 16 == 0;
    a.vec_out = op_aligned(dequantised, 16) && K % 8 == 0;
    const int64_t slice = std::max<int64_t>(1, 0x7FFFFFFF / ((int64_t)a.nb * 4));  // chunk numbers stay below 2^31
    for (int64_t n0 = 0; n0 < N; n0 += slice) {
        const int64_t rows = std::min<int64_t>(N - n0, slice);
        a.w = (const char*)w + n0 * ldw * (int64_t)esz;
        a.codes = (unsigned char*)codes + n0 * a.nb * 16;
        a.scales = (unsigned char*)scales + n0 * a.nb;
        a.deq = dequantised ? (bf16_t*)dequantised + n0 * K : nullptr;
        a.chunks = (uint32_t)(rows * a.nb * 4);
        const dim3 grid((a.chunks + 255) / 256);
        if (dtype == MV_F32) hipLaunchKernelGGL(mx_quantize_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(mx_quantize_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    }
    MX_TRY(hipGetLastError());
    return MV_OK;
}

int mv_op_linear_mxfp4(void* stream, int32_t M, int32_t N, int32_t K, const void* x, int64_t ldx, const void* codes, const void* scales, const void* codes2,
                       const void* scales2, const void* bias, const void* bias2, const void* residual, int32_t out_dtype, void* out) {
    const char* fault = product_fault(M, N, K, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out);
    if (!fault && ldx < K) fault = "ldx below K";
    if (!fault && M > 0 && N > 0 && (!x || !op_aligned(x, 2))) fault = "x is null or not aligned to its element";
    if (fault) return mv_fail(MV_ERR_INVALID, "linear_mxfp4: %s (M=%d N=%d K=%d)", fault, M, N, K);
    if (M == 0 || N == 0) return MV_OK;
    OpDevice dev((hipStream_t)stream, out);
    MX_TRY(dev.status());
    MxArgs a{x, nullptr, (const unsigned char*)codes, (const unsigned char*)scales, (const unsigned char*)codes2, (const unsigned char*)scales2,
             (const bf16_t*)bias, (const bf16_t*)bias2, residual, out, ldx, M, N, K, (K + 31) / 32, out_dtype == MV_F32, 0};
    MX_TRY(launch_products((hipStream_t)stream, a, false));
    return MV_OK;
}

int mv_op_gemm_mxfp4(void* stream, int32_t M, int32_t N, int32_t K, const void* x_codes, const void* x_scales, const void* codes, const void* scales,
                     const void* codes2, const void* scales2, const void* bias, const void* bias2, const void* residual, int32_t out_dtype, void* out) {
    const char* fault = product_fault(M, N, K, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out);
    if (!fault && M > 0 && N > 0 && (!x_codes || !x_scales || !op_aligned(x_codes, 16))) fault = "x_codes must be aligned to 16 bytes, x_scales not null";
    if (fault) return mv_fail(MV_ERR_INVALID, "gemm_mxfp4: %s (M=%d N=%d K=%d)", fault, M, N, K);
    if (M == 0 || N == 0) return MV_OK;
    OpDevice dev((hipStream_t)stream, out);
    MX_TRY(dev.status());
    MxArgs a{x_codes, (const unsigned char*)x_scales, (const unsigned char*)codes, (const unsigned char*)scales, (const unsigned char*)codes2,
             (const unsigned char*)scales2, (const bf16_t*)bias, (const bf16_t*)bias2, residual, out, 0, M, N, K, (K + 31) / 32, out_dtype == MV_F32, 0};
    MX_TRY(launch_products((hipStream_t)stream, a, true));
    return MV_OK;
}

}  // extern "C"
