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
#include <atomic>
#include <cmath>
#include <type_traits>

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));    // 16 bytes at the alignment of a bf16 element
typedef f32x4_t f32x4_any __attribute__((aligned(4)));  // and of a float
typedef uint64_t u64_byte __attribute__((aligned(1)));

#define MX_TRY(expr)                                                                                                               \
    do {                                                                                                                           \
        hipError_t _e = (expr);                                                                                                    \
        if (_e != hipSuccess) return mv_fail(MV_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(_e), __FILE__, __LINE__); \
    } while (0)

namespace {

// ---- quantiser --------------------------------------------------------------------------------------------------------------------------
// One thread: 8 columns; the 4 threads of a quad share a block and its largest magnitude by two lane moves: no LDS, no second pass.  Memory bound: 28672 x
// 8192 fp32 in 268 us, 5.7 TB/s (a large copy: 5.1); 2562 x 2048 bf16 with the dequantised copy in 6.3 us, where a launch's latency shows; 2 .. 256 rows of
// activations 2 - 3 us, 2048 x 5632 5.3 us.
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
    int32_t x_direct, s_direct;  // rows of x and of scales are aligned to 4 bytes
};

// silu(v) = v / (1 + exp(-v)).  The fast exponential rounds its argument times log2(e), an error of up to |v| 2^-24 of the result: nothing beside half a step
// of bf16 (2^-8), but tens of steps of fp32.  So fp32 outputs take the accurate one (256 x 5632 x 2048 in codes 10.6 -> 11.4 us; bf16 outputs would lose 3 - 6 %
// to it, and as much to a choice per element: the choice stands around whole runs of columns).
__device__ __forceinline__ float mx_silu_bf16(float v) { return v / (1.0f + __expf(-v)); }
__device__ __forceinline__ float mx_silu_f32(float v) { return v / (1.0f + expf(-v)); }

// y = x . w + bias (gated: silu(y) * (x . w2 + bias2)) + residual, in fp32, rounded once
template <bool GATED>
__device__ __forceinline__ void mx_store(const MxArgs& a, int m, int n, float v, float v2) {
    if (a.bias) v += bf2f(a.bias[n]);
    if (GATED && a.bias2) v2 += bf2f(a.bias2[n]);
    const int64_t at = (int64_t)m * a.N + n;
    if (a.out_f32) {
        if (GATED) v = mx_silu_f32(v) * v2;
        if (a.res) v += ((const float*)a.res)[at];
        ((float*)a.out)[at] = v;
    } else {
        if (GATED) v = mx_silu_bf16(v) * v2;
        if (a.res) v += bf2f(((const bf16_t*)a.res)[at]);
        ((bf16_t*)a.out)[at] = f2bf(v);
    }
}

// mx_store for 8 consecutive columns
template <bool GATED>
__device__ __forceinline__ void mx_store8(const MxArgs& a, int m, int n, float (&v)[8], float (&v2)[8]) {
    if (n + 8 > a.N) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < a.N) mx_store<GATED>(a, m, n + e, v[e], v2[e]);
        return;
    }
    if (a.bias) {
        const u32x4 b = *(const u32x4_any*)(a.bias + n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += e & 1 ? bf_hi(b[e >> 1]) : bf_lo(b[e >> 1]);
    }
    if (GATED && a.bias2) {
        const u32x4 b = *(const u32x4_any*)(a.bias2 + n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v2[e] += e & 1 ? bf_hi(b[e >> 1]) : bf_lo(b[e >> 1]);
    }
    if (GATED && !a.out_f32) {  // here and not beside the stores of bf16, where it costs 512 x 11008 x 4096 4 %
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mx_silu_bf16(v[e]) * v2[e];
    }
    const int64_t at = (int64_t)m * a.N + n;
    if (a.out_f32) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (GATED) v[e] = mx_silu_f32(v[e]) * v2[e];
        if (a.res) {
            const f32x4_any lo = *(const f32x4_any*)((const float*)a.res + at), hi = *(const f32x4_any*)((const float*)a.res + at + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] += lo[e]; v[4 + e] += hi[e]; }
        }
        *(f32x4_any*)((float*)a.out + at) = f32x4_t{v[0], v[1], v[2], v[3]};
        *(f32x4_any*)((float*)a.out + at + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
        if (a.res) {
            const u32x4 q = *(const u32x4_any*)((const bf16_t*)a.res + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += e & 1 ? bf_hi(q[e >> 1]) : bf_lo(q[e >> 1]);
        }
        *(u32x4_any*)((bf16_t*)a.out + at) = u32x4{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
    }
}

// 8 bf16 of a row from column c on, zero from column K on
__device__ __forceinline__ u32x4 mx_load_x8(const bf16_t* row, int c, int K) {
    if (c + 8 <= K) return *(const u32x4_any*)(row + c);
    u32x4 r = {0u, 0u, 0u, 0u};
    if (c >= K) return r;
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

#define MX_INLINE __attribute__((always_inline))
#define MX_WAVES 8

// Few rows: one workgroup computes 16 MT rows of x against 16 NT weight rows; its waves take steps of K in turn, each straight from memory to registers,
// and their sums meet in LDS, in wave order.  The weights are the first operand of the matrix instruction, so a lane ends with 4 consecutive output
// columns of one row.  Bound by the cache lines that a CU reads, or by latency when the matrix is small: bf16 rows 2 x 2562 x 2048 4.1 us, 16 x 5632 x 2048
// gated 9.2 us (1.36 TB/s), codes 16 x 2048 x 5632 5.8 us.
// LINES, where all rows begin on a 128-byte line: a step is 256 columns and a load of a wave covers 8 rows x 128 bytes.  Lane (r = lane & 15, g =
// lane >> 4) reads row r & 7 (a second load: 8 + (r & 7)), piece g + 4 (r >> 3) of 16 bytes; mx_pair turns two such loads into the two halves of the
// 128 bytes in operand order: row r, pieces g and 4 + g.
// Without it a step is 128 columns and the lane reads block g of row r, which is its operand already.  On whole lines the first is 5 - 8 % faster with
// bf16 rows (16 x 16384 x 8192: 25.3 -> 23.2 us) and 10 - 25 % with codes; on rows that straddle lines it loses 10 - 25 % (16 x 4096 x 4064: 5.8 -> 6.3 us,
// codes 4.4 -> 5.0 us).
__device__ __forceinline__ void mx_pair(u32x4& a, u32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // rotated by 8 within 16 lanes; lanes 8 .. 15 of the first, 0 .. 7 of the second half
        const uint32_t p = a[i], q = b[i];
        a[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)p, (int)q, 0x128, 0xF, 0xC, false);
        b[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)q, (int)p, 0x128, 0xF, 0x3, false);
    }
}
// lane group g holds the four words of block g -> word j of the result holds word g of block j
__device__ __forceinline__ u32x4 mx_across(const u32x4& w) {
    const auto p = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false), q = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
    const auto e = __builtin_amdgcn_permlane32_swap(p[0], q[0], false, false), o = __builtin_amdgcn_permlane32_swap(p[1], q[1], false, false);
    return u32x4{(uint32_t)e[0], (uint32_t)o[0], (uint32_t)e[1], (uint32_t)o[1]};
}
// the scales of a step: 8 of a row, or one; past the row's end anything but 255 will do, the codes there are zeros
template <bool LINES>
__device__ __forceinline__ uint64_t mx_row_scales(const unsigned char* row, int b0, int g, int nb) {
    if constexpr (LINES) return *(const u64_byte*)(row + b0);  // 8 at a time: nb is a multiple of 8
    else return b0 + g < nb ? row[b0 + g] : 127u;
}

template <bool X4, bool GATED, bool LINES, int MT, int NT>
__global__ void __launch_bounds__(64 * MX_WAVES, 2) mx_rows_kernel(const MxArgs a) {
    constexpr int MATS = GATED ? 2 : 1, XQ = X4 ? 1 : 4, E = LINES ? 2 : 1, STEP = 4 * E;  // blocks per step
    extern __shared__ __attribute__((aligned(16))) f32x4_t part[];  // [wave][matrix, weight tile, x tile][lane]
    constexpr int TILES = MATS * NT * MT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, piece = LINES ? g + 4 * (r >> 3) : g;
    const uint32_t id = op_workgroup(), tm = id / a.tiles_n, tn = id - tm * a.tiles_n;
    if (tm * (16 * MT) >= (uint32_t)a.M) return;
    const int m0 = (int)tm * 16 * MT, n0 = (int)tn * 16 * NT;
    f32x4_t acc[MATS][NT][MT];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[i][n][m] = f32x4_t{0, 0, 0, 0};
    for (int b0 = wave * STEP; b0 < a.nb; b0 += MX_WAVES * STEP) {
        u32x4 w[MATS][NT][E], x[MT][XQ][E];
        uint64_t ws[MATS][NT], xs[MT];  // LINES: the step's 8 scales of row r; else block g's own
        const bool in_k = b0 + piece < a.nb;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int row = n0 + n * 16 + (LINES ? e * 8 + (r & 7) : r);
                const int64_t at = ((int64_t)row * a.nb + b0 + piece) * 16;
#pragma unroll
                for (int i = 0; i < MATS; ++i) w[i][n][e] = u32x4{0u, 0u, 0u, 0u};
                if (in_k && row < a.N)
#pragma unroll
                    for (int i = 0; i < MATS; ++i) w[i][n][e] = *(const u32x4*)((i ? a.w2 : a.w) + at);
            }
            const int64_t row = (int64_t)min(n0 + n * 16 + r, a.N - 1) * a.nb;
#pragma unroll
            for (int i = 0; i < MATS; ++i) ws[i][n] = mx_row_scales<LINES>((i ? a.ws2 : a.ws) + row, b0, g, a.nb);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int row = m0 + m * 16 + (LINES ? e * 8 + (r & 7) : r);
#pragma unroll
                for (int q = 0; q < XQ; ++q) x[m][q][e] = u32x4{0u, 0u, 0u, 0u};
                if (row < a.M) {
                    if (X4) {
                        if (in_k) x[m][0][e] = *(const u32x4*)((const unsigned char*)a.x + ((int64_t)row * a.nb + b0 + piece) * 16);
                    } else {
                        const bf16_t* p = (const bf16_t*)a.x + (int64_t)row * a.ldx;
                        const int c = b0 * 32 + piece * (LINES ? 8 : 32);  // the pieces of 8 columns: 64 apart, or a block's four
                        if (LINES ? (b0 + STEP) * 32 <= a.K : c + 32 <= a.K) {
#pragma unroll
                            for (int q = 0; q < XQ; ++q) x[m][q][e] = *(const u32x4_any*)(p + c + q * (LINES ? 64 : 8));
                        } else if (LINES || in_k) {
#pragma unroll
                            for (int q = 0; q < XQ; ++q) x[m][q][e] = mx_load_x8(p, c + q * (LINES ? 64 : 8), a.K);
                        }
                    }
                }
            }
            if (X4) xs[m] = mx_row_scales<LINES>(a.xs + (int64_t)min(m0 + m * 16 + r, a.M - 1) * a.nb, b0, g, a.nb);
        }
        if constexpr (LINES) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < XQ; ++q) mx_pair(x[m][q][0], x[m][q][E - 1]);
#pragma unroll
            for (int i = 0; i < MATS; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) mx_pair(w[i][n][0], w[i][n][E - 1]);
        }
#pragma unroll
        for (int i = 0; i < MATS; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < E; ++e) {  // blocks b0 + 4 e + ..
                    const uint32_t sw = (uint32_t)(ws[i][n] >> (32 * e));
                    if (X4) {
                        const u32x4 v = w[i][n][e];
                        const i32x8_t wv = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const u32x4 u = x[m][0][e];
                            const i32x8_t xv = {(int)u[0], (int)u[1], (int)u[2], (int)u[3], 0, 0, 0, 0};
                            const uint32_t sx = (uint32_t)(xs[m] >> (32 * e));
                            acc[i][n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[i][n][m], 4, 4, 0, (int)(LINES ? sw >> (8 * g) : sw), 0,
                                                                                           (int)(LINES ? sx >> (8 * g) : sx));
                        }
                    } else {  // LINES: x piece 8 q + 4 e' + g is part g of block 2 q + e'; else lane group g has part j of its block at turn j
                        const u32x4 v = LINES ? mx_across(w[i][n][e]) : w[i][n][e];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t s = LINES ? sw >> (8 * j) & 255u : sw;
                            const bf16x8_t wv = mx_widen(v[j], __uint_as_float(s << 23));
#pragma unroll
                            for (int m = 0; m < MT; ++m)
                                acc[i][n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    wv, __builtin_bit_cast(bf16x8_t, LINES ? x[m][(4 * e + j) >> 1 & (XQ - 1)][j & (E - 1)] : x[m][j & (XQ - 1)][0]), acc[i][n][m], 0, 0, 0);
                        }
                    }
                }
    }
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) part[(wave * TILES + (i * NT + n) * MT + m) * 64 + lane] = acc[i][n][m];
    __syncthreads();
    // one output per thread and turn: neighbouring threads take neighbouring columns of a row
    const float* sums = (const float*)part;
    for (int o = threadIdx.x; o < MT * NT * 256; o += 64 * MX_WAVES) {
        const int c = o % (16 * NT), row = o / (16 * NT);  // column and row in the workgroup's tile
        const int at = (((c >> 4) * MT + (row >> 4)) * 64 + (((c & 15) >> 2) << 4) + (row & 15)) * 4 + (c & 3);
        float v = 0.f, v2 = 0.f;
#pragma unroll
        for (int w = 0; w < MX_WAVES; ++w) {
            v += sums[w * TILES * 256 + at];
            if (GATED) v2 += sums[w * TILES * 256 + NT * MT * 256 + at];
        }
        if (m0 + row < a.M && n0 + c < a.N) mx_store<GATED>(a, m0 + row, n0 + c, v, v2);
    }
}

// ---- large products -----------------------------------------------------------------------------------------------------------------------
// One workgroup computes BM rows of x against BN weight rows, a wave 32 TX x 32 TW of them on 32x32 matrix instructions with the weights as the first
// operand (a lane ends with 4 consecutive output columns of one row).  K advances in stages: 64 bf16 or 256 codes (128 bytes) of a row per team.
// Lane (r = lane & 31, h = lane >> 5) takes 16-byte chunk STEPS h + t of its row at step t.  With codes its steps are consecutive blocks: their scales
// lie side by side and byte t of one register serves step t.  With bf16 its 4 steps are one block of its weight row: one 16-byte read of codes that it
// widens 8 at a time.
// Stages go from memory to LDS without registers, NBUF of them in LDS: the transfers run NBUF - 1 stages ahead, since one from another XCD's share of
// memory takes longer than a stage.  The one barrier per stage stands before its last step, whose products cover its wait and the first reads of the
// next stage; the reads of step t + 1 are covered by the products of step t.
// Scales come 16 blocks of a row at a time, a group ahead, two groups in LDS (a few bytes per row and stage would touch as many cache lines as the
// codes do).
// LDS has 64 banks and serves 16 lanes of a 16-byte read at a time: chunk c of a row lies at c ^ (row / (rows per 256 bytes)), so 16 rows
// spread over all banks.  A transfer writes LDS in lane order: the permutation is applied to the lane's address in memory.  The scales are not spread: their
// reads (1 or 4 bytes of rows 16 bytes apart) are the bank conflicts that the counters show, 6 cycles each: 29 % of the LDS cycles with bf16 rows, 23 % with
// codes.
// Five tiles, the smaller ones for grids that would leave CUs idle: 256 x 256 (8 waves of 64 rows x 128 columns) and 128 x 256 (8 of 64 x 64); with the waves
// in teams that split a stage's columns 128 x 128 and 64 x 128 (two teams of 4 waves) and 64 x 64 (bf16 rows: four teams of 2, codes: two of 4).
// Measured: 64 x 16384 x 8192 by the last one bf16 rows 27 us (128 x 128: 57), codes 15 us (24), the weights at 4.7 TB/s; 384 x 16384 x 8192 by 128 x 256
// codes 41 us (128 x 128: 48), bf16 rows 115 us (121); by 256 x 256, medians, bf16 rows 4096 x 16384 x 8192 in 925 us, 1.19 PFLOP/s (fastest 850; a library
// product of two bf16 matrices: 713 us), codes 8192 x 16384 x 8192 in 608 us, 3.6 PFLOP/s (fastest 557).  The last two are bound by power: the matrix units are
// busy 68 % (bf16) and 57 % (codes) of the time at about 1.8 GHz, and a loop of the same matrix instructions alone, on operands of the same distribution in
// registers, takes 658 us and 2 x 198 us.
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* glb_ptr_t;
typedef u32x4 u32x4_byte __attribute__((aligned(1)));

template <bool X4, int KS, int WN, int WM, int TW, int TX>
struct Tile {
    static constexpr int TEAM = WN * WM, WAVES = KS * TEAM, THREADS = 64 * WAVES;
    static constexpr int BM = 32 * WM * TX, BN = 32 * WN * TW;       // rows of x and weight rows of a workgroup
    static constexpr int XROW = 128, WROW = X4 ? 128 : 32;           // bytes of a row in a team's share of a stage
    static constexpr int BLOCKS = X4 ? 8 : 2, STEPS = 4;             // blocks of 32 columns in it, and steps
    static constexpr int GROUP = 16 / (BLOCKS * KS);                 // stages per group of scales
    static constexpr int X = BM * XROW, W = BN * WROW, SHARE = X + W, STAGE = KS * SHARE;
    static constexpr int SROWS = X4 ? BM + BN : BN, S = SROWS * 16;
    // A group of scales has to be older than the transfers that a stage's wait leaves on their way: it is asked for AHEAD groups ahead, and lies in one
    // of AHEAD + 1 places in turn, a short one at the end of a row in a place of its own.
    static constexpr int fit(int bufs) { return bufs * STAGE + ((bufs + GROUP - 1) / GROUP + 2) * S; }
    static constexpr int NBUF = fit(4) <= 160 * 1024 ? 4 : fit(3) <= 160 * 1024 ? 3 : 2;
    static constexpr int AHEAD = (NBUF + GROUP - 1) / GROUP, RING = AHEAD + 1;
    static constexpr int EPI = TEAM * 32 * (32 * TW + 4) * 4;        // the epilogue's tiles: 32 rows of a wave's columns each
    static constexpr int JOIN = (KS - 1) * TEAM * TW * TX * 4096;    // the other teams' sums
    static constexpr int MAIN = fit(NBUF), TAIL = EPI + JOIN, LDS = MAIN > TAIL ? MAIN : TAIL;
    static constexpr int XI = X / 1024 / TEAM, WI = W / 1024 / TEAM;  // transfers of 1 KB per wave and stage
    static_assert(XI * TEAM * 1024 == X && WI * TEAM * 1024 == W && LDS <= 160 * 1024, "whole transfers per wave");
};

template <int ROWB>
__device__ __forceinline__ int mx_slot(int row, int c) { return c ^ ((row / (256 / ROWB)) & (ROWB / 16 - 1)); }

template <bool X4, int KS, int WN, int WM, int TW, int TX, bool GATED>
__global__ void __launch_bounds__(64 * KS * WN * WM, 2) mx_tile_kernel(const MxArgs a) {
    typedef Tile<X4, KS, WN, WM, TW, TX> T;
    constexpr int XCH = T::XROW / 16, WCH = T::WROW / 16, NBUF = T::NBUF;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave_of_all = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
    const int team = KS == 1 ? 0 : wave_of_all / T::TEAM, wave = KS == 1 ? wave_of_all : wave_of_all % T::TEAM;
    const int wm = wave % WM, wn = wave / WM;
    constexpr int NOUT = GATED ? T::BN / 2 : T::BN;  // output columns of a workgroup

    // workgroups go round the 8 XCDs: each XCD takes a contiguous range of tiles, ordered in bands of 4 row tiles so that the 32 tiles in flight on it
    // share rows of x and of the weights in its L2
    uint32_t id = blockIdx.x;
    {
        const uint32_t total = gridDim.x, q = total / 8, rem = total % 8, xcd = id % 8, k = id / 8;
        id = xcd * q + min(xcd, rem) + k;
    }
    const uint32_t tiles_m = (uint32_t)((a.M + T::BM - 1) / T::BM);
    const uint32_t band = id / (4 * a.tiles_n), in_band = id - band * 4 * a.tiles_n, rows_in = min(4u, tiles_m - band * 4);
    const int m0 = (int)(band * 4 + in_band % rows_in) * T::BM, n0 = (int)(in_band / rows_in) * NOUT;

    // row of the weights' LDS image -> matrix and weight row (gated: a wave's first half of columns from w, the second half the same columns of w2)
    auto w_row = [&](int row, int& second) MX_INLINE {
        if (!GATED) { second = 0; return min(n0 + row, a.N - 1); }
        second = (row / (16 * TW)) & 1;
        return min(n0 + (row / (32 * TW)) * (16 * TW) + row % (16 * TW), a.N - 1);
    };
    const int64_t code_row = (int64_t)a.nb * 16, x_row = X4 ? code_row : a.ldx * 2;

    // a lane's addresses in a stage: bytes from the workgroup's first row of x and first weight row
    const unsigned char* const xbase = (const unsigned char*)a.x + (int64_t)m0 * x_row;
    uint32_t gx[T::XI], gw[T::WI];
    const unsigned char* wbase[T::WI];
    static_assert(!GATED || (16 * TW) % (1024 / T::WROW) == 0, "a transfer reads one matrix");
#pragma unroll
    for (int i = 0; i < T::XI; ++i) {
        const int row = (wave * T::XI + i) * (64 / XCH) + lane / XCH;
        gx[i] = (uint32_t)min(row, a.M - 1 - m0) * (uint32_t)x_row + mx_slot<T::XROW>(row, lane % XCH) * 16;
    }
#pragma unroll
    for (int i = 0; i < T::WI; ++i) {
        const int row = (wave * T::WI + i) * (64 / WCH) + lane / WCH;
        int second;
        gw[i] = (uint32_t)(w_row(row, second) - n0) * (uint32_t)code_row + mx_slot<T::WROW>(row, lane % WCH) * 16;
        (void)w_row((wave * T::WI + i) * (64 / WCH), second);
        wbase[i] = (second ? a.w2 : a.w) + (int64_t)n0 * code_row;
    }
    const int stages = (a.nb + KS * T::BLOCKS - 1) / (KS * T::BLOCKS);
    const int whole = X4 ? a.nb / (KS * 8) : a.K / (KS * 64), direct = a.x_direct ? whole : 0;  // the stages that are not short; and aligned

    const int share = team * T::SHARE;
    auto transfer_x = [&](int st, int buf) MX_INLINE {
        const int v = st * KS + team;
#pragma unroll
        for (int i = 0; i < T::XI; ++i)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)(xbase + (int64_t)v * T::XROW + gx[i]), (lds_ptr_t)(lds + buf + share + (wave * T::XI + i) * 1024), 16, 0, 0);
    };
    auto transfer_w = [&](int st, int buf) MX_INLINE {
        const int v = st * KS + team;
#pragma unroll
        for (int i = 0; i < T::WI; ++i)
            __builtin_amdgcn_global_load_lds((glb_ptr_t)(wbase[i] + (int64_t)v * T::WROW + gw[i]), (lds_ptr_t)(lds + buf + share + T::X + (wave * T::WI + i) * 1024), 16, 0, 0);
    };
    // every second one of a stage's transfers
    auto transfer_half = [&](int st, int buf, int half) MX_INLINE {
        const int v = st * KS + team;
#pragma unroll
        for (int q = half; q < T::XI + T::WI; q += 2) {
            if (q < T::XI)
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(xbase + (int64_t)v * T::XROW + gx[q < T::XI ? q : 0]), (lds_ptr_t)(lds + buf + share + (wave * T::XI + q) * 1024), 16, 0, 0);
            else
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(wbase[q < T::XI ? 0 : q - T::XI] + (int64_t)v * T::WROW + gw[q < T::XI ? 0 : q - T::XI]),
                                                 (lds_ptr_t)(lds + buf + share + T::X + (wave * T::WI + q - T::XI) * 1024), 16, 0, 0);
        }
    };
    // What transfers cannot bring comes through registers, zeros past K: the short stage at the end of a row, and rows of bf16 that are not aligned to 4
    // bytes.  The latter are asked for at one stage and put into LDS at the next (by the tiles of teams; the largest has no registers for that).
    auto carry_w = [&](int st, int buf) MX_INLINE {
        const int v = st * KS + team;
#pragma unroll 1
        for (int i = tid % (64 * T::TEAM); i < T::W / 16; i += 64 * T::TEAM) {
            const int row = i / WCH, c = mx_slot<T::WROW>(row, i % WCH);
            int second;
            const int n = w_row(row, second);
            u32x4 q = {0u, 0u, 0u, 0u};
            if (v * T::BLOCKS + c < a.nb) q = *(const u32x4*)((second ? a.w2 : a.w) + n * code_row + (int64_t)(v * T::BLOCKS + c) * 16);
            *(u32x4*)(lds + buf + share + T::X + i * 16) = q;
        }
    };
    auto x_piece = [&](int st, int at) MX_INLINE {  // 16 bytes of a stage's x in the order of its LDS image
        const int v = st * KS + team, row = at / XCH, c = mx_slot<T::XROW>(row, at % XCH), m = min(m0 + row, a.M - 1);
        if (X4) return v * T::BLOCKS + c < a.nb ? *(const u32x4*)((const unsigned char*)a.x + m * x_row + (int64_t)(v * T::BLOCKS + c) * 16) : u32x4{0u, 0u, 0u, 0u};
        const bf16_t* p = (const bf16_t*)a.x + m * a.ldx;
        return (v + 1) * 64 <= a.K ? (u32x4) * (const u32x4_any*)(p + v * 64 + c * 8) : mx_load_x8(p, v * 64 + c * 8, a.K);
    };
    auto carry_x = [&](int st, int buf) MX_INLINE {
#pragma unroll 1
        for (int i = tid % (64 * T::TEAM); i < T::X / 16; i += 64 * T::TEAM) *(u32x4*)(lds + buf + share + i * 16) = x_piece(st, i);
    };
    constexpr bool LATER = KS > 1;
    constexpr int XC = LATER ? T::X / 1024 / T::TEAM : 0;  // 16-byte pieces of x per thread and stage
    u32x4 xreg[XC + 1];
    auto x_in = [&](int st) MX_INLINE {
#pragma unroll
        for (int i = 0; i < XC; ++i) xreg[i] = x_piece(st, tid % (64 * T::TEAM) + i * 64 * T::TEAM);
    };
    auto x_out = [&](int buf) MX_INLINE {
#pragma unroll
        for (int i = 0; i < XC; ++i) *(u32x4*)(lds + buf + share + (tid % (64 * T::TEAM) + i * 64 * T::TEAM) * 16) = xreg[i];
    };

    // scales of a group: 16 bytes of row t (with 4-bit x the rows of x come first) by transfer t / 64, wave after wave
    constexpr int SBASE = NBUF * T::STAGE, SN = T::SROWS / 64, SI = (SN + T::WAVES - 1) / T::WAVES;
    auto scale_row = [&](int row) MX_INLINE {
        if (X4 && row < T::BM) return a.xs + (int64_t)min(m0 + row, a.M - 1) * a.nb;
        int second;
        const int n = w_row(X4 ? row - T::BM : row, second);
        return (second ? a.ws2 : a.ws) + (int64_t)n * a.nb;
    };
    const unsigned char* gs[SI];
#pragma unroll
    for (int i = 0; i < SI; ++i) gs[i] = scale_row(min(wave_of_all + i * T::WAVES, SN - 1) * 64 + lane);
    const int whole_groups = a.nb / 16;
    auto scale_at = [&](int group) MX_INLINE { return SBASE + (group >= whole_groups ? T::RING : group % T::RING) * T::S; };
    auto scales = [&](int group) MX_INLINE {  // a whole, aligned group
        const int to = scale_at(group);
#pragma unroll
        for (int i = 0; i < SI; ++i)
            if (SN % T::WAVES == 0 || wave_of_all + i * T::WAVES < SN)
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(gs[i] + group * 16), (lds_ptr_t)(lds + to + (wave_of_all + i * T::WAVES) * 1024), 16, 0, 0);
    };
    // whole groups of rows of scales that are not aligned to 4 bytes: through registers, asked for at one stage and put into LDS at the next
    u32x4 sreg = {0u, 0u, 0u, 0u};
    static_assert(T::SROWS <= T::THREADS, "a row of scales per thread");
    auto scales_in = [&](int group) MX_INLINE { sreg = *(const u32x4_byte*)(scale_row(min(tid, T::SROWS - 1)) + group * 16); };
    auto scales_out = [&](int group) MX_INLINE {
        if (tid < T::SROWS) *(u32x4*)(lds + scale_at(group) + tid * 16) = sreg;
    };
    auto carry_scales = [&](int group) MX_INLINE {  // at the start: a short group at the end of a row
        const int b = group * 16, to = scale_at(group);
#pragma unroll 1
        for (int i = tid; i < T::SROWS * 4; i += T::THREADS) {
            const unsigned char* p = scale_row(i >> 2);
            uint32_t q = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) q |= (uint32_t)(b + (i & 3) * 4 + k < a.nb ? p[b + (i & 3) * 4 + k] : 127u) << (8 * k);
            *(uint32_t*)(lds + to + i * 4) = q;
        }
    };

    f32x16_t acc[TW][TX];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TX; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    u32x4 fx[2][TX], fw[2][TW];     // fragments of two steps; of bf16 stages the weights' are the stage's codes
    uint32_t sx[2][TX], sw[2][TW];  // scales of a stage
    int xat[T::STEPS], wat[X4 ? T::STEPS : 1];
#pragma unroll
    for (int t = 0; t < T::STEPS; ++t) {
        xat[t] = share + (wm * 32 * TX + r) * T::XROW + mx_slot<T::XROW>(r, T::STEPS * h + t) * 16;
        if (X4 || t == 0) wat[X4 ? t : 0] = share + T::X + (wn * 32 * TW + r) * T::WROW + mx_slot<T::WROW>(r, X4 ? T::STEPS * h + t : h) * 16;
    }
    auto read_x = [&](int buf, int t, u32x4 (&f)[TX]) MX_INLINE {
#pragma unroll
        for (int j = 0; j < TX; ++j) f[j] = *(const u32x4*)(lds + buf + xat[t] + j * 32 * T::XROW);
    };
    auto read_w = [&](int buf, int t, u32x4 (&f)[TW]) MX_INLINE {
#pragma unroll
        for (int i = 0; i < TW; ++i) f[i] = *(const u32x4*)(lds + buf + wat[X4 ? t : 0] + i * 32 * T::WROW);
    };
    auto read_s = [&](int st, uint32_t (&fsx)[TX], uint32_t (&fsw)[TW]) MX_INLINE {
        const unsigned char* buf = lds + scale_at(st / T::GROUP) + (st % T::GROUP * KS + team) * T::BLOCKS + (X4 ? h * 4 : h) + r * 16;
        if (X4) {
#pragma unroll
            for (int j = 0; j < TX; ++j) fsx[j] = *(const uint32_t*)(buf + (wm * 32 * TX + j * 32) * 16);
#pragma unroll
            for (int i = 0; i < TW; ++i) fsw[i] = *(const uint32_t*)(buf + (T::BM + wn * 32 * TW + i * 32) * 16);
        } else {
#pragma unroll
            for (int i = 0; i < TW; ++i) fsw[i] = buf[(wn * 32 * TW + i * 32) * 16];
        }
    };
    // The products of a step.  They stay where they stand: left alone, the compiler carries them past the branches and reads of later steps, with all
    // the registers that takes.
    // The reads of the next step (`reads`) come behind the first products: the compiler waits for all reads on their way where it waits for one.
    auto multiply = [&](auto step, const u32x4 (&x)[TX], const u32x4 (&w)[TW], const uint32_t (&csx)[TX], const uint32_t (&csw)[TW], auto reads, auto asks) MX_INLINE {
        constexpr int t = decltype(step)::value;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            if constexpr (X4) {
                const i32x8_t wv = {(int)w[i][0], (int)w[i][1], (int)w[i][2], (int)w[i][3], 0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < TX; ++j) {
                    const i32x8_t xv = {(int)x[j][0], (int)x[j][1], (int)x[j][2], (int)x[j][3], 0, 0, 0, 0};
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, acc[i][j], 4, 4, t, (int)csw[i], t, (int)csx[j]);
                }
            } else {
                const bf16x8_t wv = mx_widen(w[i][t], __uint_as_float(csw[i] << 23));
#pragma unroll
                for (int j = 0; j < TX; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv, __builtin_bit_cast(bf16x8_t, x[j]), acc[i][j], 0, 0, 0);
            }
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < TX; ++j) asm volatile("" : "+v"(acc[i][j]));
                __builtin_amdgcn_sched_barrier(0);
                reads();
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == TW / 2) {
#pragma unroll
                for (int k = 1; k <= i; ++k)
#pragma unroll
                    for (int j = 0; j < TX; ++j) asm volatile("" : "+v"(acc[k][j]));
                __builtin_amdgcn_sched_barrier(0);
                asks();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 1; i < TW; ++i)
#pragma unroll
            for (int j = 0; j < TX; ++j) asm volatile("" : "+v"(acc[i][j]));
        __builtin_amdgcn_sched_barrier(0);
    };

#pragma unroll
    for (int i = 0; i < T::AHEAD; ++i)
        if (a.s_direct && i < whole_groups) scales(i);
#pragma unroll
    for (int i = 0; i < NBUF; ++i) {
        if (i >= stages) break;
        if (i < whole) transfer_w(i, i * T::STAGE);
        else carry_w(i, i * T::STAGE);
        if (i < direct) {
            transfer_x(i, i * T::STAGE);
        } else {
            carry_x(i, i * T::STAGE);
        }
    }
    if (a.nb % 16) carry_scales(whole_groups);
    if (!a.s_direct)
        for (int i = 0; i < min(T::AHEAD, whole_groups); ++i) {
            scales_in(i);
            scales_out(i);
        }
    // scales were asked for first, then the stages in order: the first one is enough to begin with (2 % at K = 2048 with bf16 rows, a loss of 3 % where
    // there are only two)
    if (NBUF > 2 && direct >= NBUF) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 1) * (T::XI + T::WI)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_s(0, sx[0], sw[0]);
    read_w(0, 0, fw[0]);
    read_x(0, 0, fx[0]);

    int cur = 0;  // byte offset of the stage's buffer
    const auto wait_and_ask = [&](auto kind, int st) MX_INLINE {
        constexpr bool DIRECT = decltype(kind)::value;
        if (!DIRECT && st > 0) {  // what stage st - 1 asked for: its buffer, and a place for scales
            if (LATER && st - 1 + NBUF >= direct && st - 1 + NBUF < stages) x_out(cur == 0 ? (NBUF - 1) * T::STAGE : cur - T::STAGE);
            if (!a.s_direct && (st - 1) % T::GROUP == 0 && (st - 1) / T::GROUP + T::AHEAD < whole_groups) scales_out((st - 1) / T::GROUP + T::AHEAD);
        }
        // stage st + 1 must have arrived, NBUF - 2 later ones may be on their way (a request for scales among them only makes the wait longer)
        if (st + NBUF - 1 < direct) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 2) * (T::XI + T::WI)) : "memory");
        else if (!DIRECT && st + NBUF - 1 < whole) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 2) * T::WI) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        // and every wave has read all of stage st: its buffer is free
        if (!DIRECT && st + NBUF < stages) {
            if (st + NBUF < direct) transfer_x(st + NBUF, cur);
            else if (LATER) x_in(st + NBUF);
            else carry_x(st + NBUF, cur);
            if (st + NBUF < whole) transfer_w(st + NBUF, cur);
            else carry_w(st + NBUF, cur);
        }
        if (st % T::GROUP == 0 && st / T::GROUP + T::AHEAD < whole_groups) {
            if (DIRECT || a.s_direct) scales(st / T::GROUP + T::AHEAD);
            else scales_in(st / T::GROUP + T::AHEAD);
        }
    };
    // A stage, P its parity.  DIRECT: all that it asks for comes without registers.  (In one loop with the other kind, the compiler would let every read
    // of LDS wait for all that are on their way.)
    auto stage = [&](auto parity, auto kind, int st) MX_INLINE {
        constexpr int P = decltype(parity)::value;
        constexpr bool DIRECT = decltype(kind)::value;
        const int next = cur + T::STAGE == NBUF * T::STAGE ? 0 : cur + T::STAGE;
        // Transfers into a buffer that a barrier has freed: half of them behind the first products after it, half in the next step (the buffer of stage
        // st - 1).  All at once, in front of the products, they hold them up: 297 -> 284 us at 4096 x 16384 x 8192 in 4 bits.
        const int last = cur == 0 ? (NBUF - 1) * T::STAGE : cur - T::STAGE;
        const auto nothing = [] {};
        const bool ask = DIRECT && st > 0 && st - 1 + NBUF < direct;
        multiply(std::integral_constant<int, 0>{}, fx[0], fw[X4 ? 0 : P], sx[P], sw[P], [&] {
            read_x(cur, 1, fx[1]);
            if (X4) read_w(cur, 1, fw[1]);
        }, [&] { if (ask) transfer_half(st - 1 + NBUF, last, 1); });
        multiply(std::integral_constant<int, 1>{}, fx[1], fw[X4 ? 1 : P], sx[P], sw[P], [&] {
            read_x(cur, 2, fx[0]);
            if (X4) read_w(cur, 2, fw[0]);
        }, nothing);
        multiply(std::integral_constant<int, 2>{}, fx[0], fw[X4 ? 0 : P], sx[P], sw[P], [&] {
            read_x(cur, 3, fx[1]);
            if (X4) read_w(cur, 3, fw[1]);
        }, nothing);
        if (st + 1 < stages) wait_and_ask(kind, st);
        multiply(std::integral_constant<int, 3>{}, fx[1], fw[X4 ? 1 : P], sx[P], sw[P], [&] {
            if (st + 1 < stages) {
                read_s(st + 1, sx[P ^ 1], sw[P ^ 1]);
                read_w(next, 0, fw[X4 ? 0 : P ^ 1]);
                read_x(next, 0, fx[0]);
            }
        }, [&] { if (DIRECT && st + NBUF < direct) transfer_half(st + NBUF, cur, 0); });
        cur = next;
    };
    const int easy = !a.s_direct ? 0 : direct == stages ? stages : max(0, direct - NBUF) & ~1;
    int st = 0;
#pragma unroll 1
    for (; st < easy; st += 2) {
        stage(std::integral_constant<int, 0>{}, std::true_type{}, st);
        if (st + 1 < easy) stage(std::integral_constant<int, 1>{}, std::true_type{}, st + 1);
    }
    if (easy > 0 && easy < stages && easy - 1 + NBUF < direct) {  // what the last of these stages left to its successor
        transfer_half(easy - 1 + NBUF, cur == 0 ? (NBUF - 1) * T::STAGE : cur - T::STAGE, 1);
    }
#pragma unroll 1
    for (; st < stages; st += 2) {
        stage(std::integral_constant<int, 0>{}, std::false_type{}, st);
        if (st + 1 < stages) stage(std::integral_constant<int, 1>{}, std::false_type{}, st + 1);
    }

    if constexpr (KS > 1) {  // the first team adds the others' sums, in their order
        __syncthreads();
        f32x4_t* const part = (f32x4_t*)lds;
#pragma unroll
        for (int k = 1; k < KS; ++k) {
            const int at = ((k - 1) * T::TEAM + wave) * TW * TX * 256;
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TX; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (team == k) part[at + ((i * TX + j) * 4 + q) * 64 + lane] = f32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
        __syncthreads();
        if (team != 0) return;
#pragma unroll
        for (int k = 1; k < KS; ++k) {
            const int at = ((k - 1) * T::TEAM + wave) * TW * TX * 256;
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TX; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4_t o = part[at + ((i * TX + j) * 4 + q) * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += o[e];
                    }
        }
    }

    // epilogue: a wave turns 32 rows of its columns at a time through LDS, so that rows are stored in runs
    if constexpr (KS == 1) __syncthreads();
    constexpr int COLS = 32 * TW, PITCH = COLS + 4, OUT = GATED ? COLS / 2 : COLS, LPR = OUT / 8;  // LPR lanes store a row, 8 columns each
    float* et = (float*)(lds + T::JOIN) + wave * 32 * PITCH;
    const int c8 = (lane % LPR) * 8, n = n0 + wn * OUT + c8;
#pragma unroll
    for (int j = 0; j < TX; ++j) {
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(f32x4_t*)(et + r * PITCH + i * 32 + q * 8 + h * 4) = f32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 2
        for (int row = lane / LPR; row < 32; row += 64 / LPR) {
            const int m = m0 + wm * 32 * TX + j * 32 + row;
            if (m >= a.M || n >= a.N) continue;
            float v[8], v2[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = et[row * PITCH + c8 + e];
                v2[e] = GATED ? et[row * PITCH + OUT + c8 + e] : 0.f;
            }
            mx_store8<GATED>(a, m, n, v, v2);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// more LDS per workgroup than the 64 KB that need no leave; the leave is the device's own copy of the kernel's
template <auto Kernel>
hipError_t allow_lds(int bytes) {
    static std::atomic<uint64_t> done[4];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || (dev < 256 && (done[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63) & 1))) return e;
    e = hipFuncSetAttribute((const void*)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && dev < 256) done[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    return e;
}

template <bool GATED, bool X4, int KS, int WN, int WM, int TW, int TX>
hipError_t launch_tiles(hipStream_t s, MxArgs a, Tile<X4, KS, WN, WM, TW, TX>) {
    typedef Tile<X4, KS, WN, WM, TW, TX> T;
    constexpr int NOUT = GATED ? T::BN / 2 : T::BN;
    const uint32_t tiles_m = (uint32_t)((a.M + T::BM - 1) / T::BM);
    a.tiles_n = (uint32_t)((a.N + NOUT - 1) / NOUT);
    constexpr auto kernel = mx_tile_kernel<X4, KS, WN, WM, TW, TX, GATED>;
    const hipError_t e = allow_lds<kernel>(T::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3(tiles_m * a.tiles_n), dim3(T::THREADS), T::LDS, s, a);
    return hipGetLastError();
}

template <bool X4, bool GATED, bool LINES, int MT, int NT>
hipError_t launch_rows(hipStream_t s, MxArgs a) {
    constexpr int LDS = MX_WAVES * (GATED ? 2 : 1) * MT * NT * 1024;
    constexpr auto kernel = mx_rows_kernel<X4, GATED, LINES, MT, NT>;
    const hipError_t e = LDS > 64 * 1024 ? allow_lds<kernel>(LDS) : hipSuccess;
    if (e != hipSuccess) return e;
    a.tiles_n = (uint32_t)((a.N + 16 * NT - 1) / (16 * NT));
    const uint64_t tiles_m = (uint32_t)((a.M + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL(kernel, op_grid(tiles_m * a.tiles_n), dim3(64 * MX_WAVES), LDS, s, a);
    return hipGetLastError();
}

// Estimated microseconds of the two kernels, in coefficients fitted to 602 measured calls (1 .. 4096 rows, 100 .. 16384 columns, K from 300 to 11008; beyond
// that they are carried on).  Over these the choice costs 1 % over the best kernel on average (at most 43 %: 192 x 400 x 8192), and 2.5 - 10 % without any one
// of the five tiles; the estimate itself is off by 5 % in the middle and 39 % at most.  A workgroup of the first kernel reads its rows of x and of the weights;
// what counts is how much the busiest CU reads (workgroups with 4 and more products share one unevenly: rounds of them count).  One of the second advances by
// stages, a little slower when all CUs work, 1.4 times as long where scales come through registers.
template <bool X4>
double rows_us(const MxArgs& a, int mt, int nt) {
    const double mats = a.w2 ? 2 : 1, products = mt * nt * mats, per_cu = (double)((a.M + 16 * mt - 1) / (16 * mt)) * ((a.N + 16 * nt - 1) / (16 * nt)) / 256;
    const double kb = 1e-3 * a.nb * (std::min(a.M, 16 * mt) * (X4 ? 17 : 64) + 16 * nt * mats * 17), times = products < 4 ? std::max(1.0, per_cu) : std::ceil(per_cu);
    return X4 ? 2.5 + 0.152 * products + 0.035 * kb * times : 2.8 + 0.276 * products + 0.031 * kb * times;
}
struct TileCost { int bm, bn; double call, round, block, full; };
constexpr TileCost MX_COST[2][5] = {
    {{64, 64, 2.2, 2.5, 0.064, 0.021}, {64, 128, 2.8, 2.0, 0.111, 0.039}, {128, 128, 2.2, 3.6, 0.173, 0.074}, {128, 256, 2.4, 3.4, 0.326, 0.111}, {256, 256, 8.9, 2.2, 0.481, 0.253}},
    {{64, 64, 2.1, 1.7, 0.026, 0.014}, {64, 128, 2.4, 1.9, 0.035, 0.025}, {128, 128, 2.1, 3.0, 0.053, 0.040}, {128, 256, 1.4, 4.2, 0.089, 0.056}, {256, 256, 5.6, 2.6, 0.146, 0.111}}};
double tiles_us(const MxArgs& a, const TileCost& c) {
    const double tiles = (double)((a.M + c.bm - 1) / c.bm) * (((a.w2 ? 2ll : 1ll) * a.N + c.bn - 1) / c.bn), rounds = std::ceil(tiles / 256);
    return c.call + rounds * (c.round + a.nb * (a.s_direct ? 1.0 : 1.4) * (c.block + c.full * std::min(1.0, tiles / 256)));
}

// The kernels: three of the first kind (in 16s of rows and columns 1 x 1, 1 x 2, and 1 x 4 or, with codes, 2 x 2: with bf16 rows more columns come before more
// rows, since a row costs what 4 columns do), then five of the second.
constexpr int MX_ROW_TILES = 3;
constexpr int MX_TALL[2][2] = {{1, 4}, {2, 2}};
template <bool X4, class F>
auto with_tile(int tile, const F& f) {
    switch (tile) {
        case 0: return f(Tile<X4, X4 ? 2 : 4, X4 ? 2 : 1, 2, X4 ? 1 : 2, 1>());
        case 1: return f(Tile<X4, 2, 2, 2, 2, 1>());
        case 2: return f(Tile<X4, 2, 2, 2, 2, 2>());
        case 3: return f(Tile<X4, 1, 4, 2, 2, 2>());
        default: return f(Tile<X4, 1, 2, 4, 4, 2>());
    }
}

// the fastest by the estimate: 0 .. 2 of the first kind, 3 .. 7 of the second
template <bool X4>
int choose(const MxArgs& a) {
    const double r1 = rows_us<X4>(a, 1, 1), r2 = rows_us<X4>(a, 1, 2), r3 = rows_us<X4>(a, MX_TALL[X4][0], MX_TALL[X4][1]), rows = std::min({r1, r2, r3});
    const int64_t x_row = X4 ? (int64_t)a.nb * 16 : a.ldx * 2;
    // the second kernel counts bytes within a workgroup's rows in 32 bits, and its threads are one dimension of a grid
    if (x_row <= 1 << 23 && a.nb <= 1 << 19 && ((a.M + 63ll) / 64) * ((a.N * (a.w2 ? 2ll : 1ll) + 63) / 64) < 1 << OP_GRID_BITS) {
        const TileCost* c = MX_COST[X4];
        double t[5];
        for (int i = 0; i < 5; ++i) t[i] = i < 3 || a.x_direct ? tiles_us(a, c[i]) : 1e30;
        const double tiles = *std::min_element(t, t + 5);
        if (tiles < rows) return MX_ROW_TILES + (int)(std::find(t, t + 5, tiles) - t);
    }
    return r1 == rows ? 0 : r2 == rows ? 1 : 2;
}

// what decides among the forms of a kernel, by addresses and strides; true: whole lines
bool product_form(MxArgs& a, bool x4) {
    a.x_direct = x4 || (op_aligned(a.x, 4) && a.ldx % 2 == 0);
    a.s_direct = a.nb % 4 == 0 && op_aligned(a.ws, 4) && op_aligned(a.ws2, 4) && op_aligned(a.xs, 4);
    return a.nb % 8 == 0 && op_aligned(a.w, 128) && op_aligned(a.w2, 128) && op_aligned(a.x, 128) && (x4 || a.ldx % 64 == 0);
}

template <bool X4, bool GATED, bool LINES>
hipError_t launch(hipStream_t s, const MxArgs& a) {
    const int kernel = choose<X4>(a);
    if (kernel == 0) return launch_rows<X4, GATED, LINES, 1, 1>(s, a);
    if (kernel == 1) return launch_rows<X4, GATED, LINES, 1, 2>(s, a);
    if (kernel == 2) return launch_rows<X4, GATED, LINES, MX_TALL[X4][0], MX_TALL[X4][1]>(s, a);
    return with_tile<X4>(kernel - MX_ROW_TILES, [&](auto tile) { return launch_tiles<GATED>(s, a, tile); });
}

hipError_t launch_products(hipStream_t s, MxArgs a, bool x4) {
    if (product_form(a, x4)) return x4 ? (a.w2 ? launch<true, true, true>(s, a) : launch<true, false, true>(s, a)) : (a.w2 ? launch<false, true, true>(s, a) : launch<false, false, true>(s, a));
    return x4 ? (a.w2 ? launch<true, true, false>(s, a) : launch<true, false, false>(s, a)) : (a.w2 ? launch<false, true, false>(s, a) : launch<false, false, false>(s, a));
}

template <bool X4>
void describe(const MxArgs& a, bool lines, int32_t* out) {
    const int kernel = choose<X4>(a), tile = kernel - MX_ROW_TILES;
    out[0] = kernel;
    out[1] = lines;
    out[2] = a.x_direct;
    out[3] = a.s_direct;
    out[4] = tile < 0 ? (a.nb + MX_WAVES * (lines ? 8 : 4) - 1) / (MX_WAVES * (lines ? 8 : 4)) : with_tile<X4>(tile, [&](auto t) {
        const int blocks = 16 / decltype(t)::GROUP;
        return (a.nb + blocks - 1) / blocks;
    });
    out[5] = tile < 0 ? 0 : with_tile<X4>(tile, [](auto t) { return (int)decltype(t)::NBUF; });
    out[6] = a.nb / 16;
    out[7] = tile < 0 ? 0 : with_tile<X4>(tile, [](auto t) { return (int)decltype(t)::AHEAD; });
}

// the checks that both products share; null: fine
const char* product_fault(int32_t M, int32_t N, int32_t K, const OpRows& x, const void* x_scales, const void* codes, const void* scales, const void* codes2, const void* scales2,
                          const void* bias, const void* bias2, const void* residual, int32_t out_dtype, const void* out) {
    if (M < 0 || N < 0 || K < 1) return "M and N must not be negative, K must be positive";
    if (std::max({M, N, K}) > 0x7FFFFFFF - 4096) return "M, N or K is too large";
    if (out_dtype != MV_BF16 && out_dtype != MV_F32) return "out_dtype must be MV_BF16 or MV_F32";
    if (M == 0 || N == 0) return nullptr;
    if (!codes || !scales || !out) return "null argument";
    if (!codes2 != !scales2) return "codes2 and scales2 go together";
    if (bias2 && !codes2) return "bias2 without codes2";
    if (!op_aligned(codes, 16) || !op_aligned(codes2, 16)) return "codes must be aligned to 16 bytes";
    const size_t esz = out_dtype == MV_F32 ? 4 : 2;
    if (!op_aligned(out, esz) || !op_aligned(residual, esz) || !op_aligned(bias, 2) || !op_aligned(bias2, 2)) return "a buffer is not aligned to its element";
    const int64_t nb = ((int64_t)K + 31) / 32;
    const OpRows y = op_bytes(out, M, (int64_t)N * (int64_t)esz);
    if (residual != out && op_overlap(y, op_bytes(residual, M, (int64_t)N * (int64_t)esz))) return "out on top of a part of the residual";
    for (const OpRows& b : {x, op_bytes(x_scales, M, nb), op_bytes(codes, N, 16 * nb), op_bytes(codes2, N, 16 * nb), op_bytes(scales, N, nb), op_bytes(scales2, N, nb),
                            op_bytes(bias, N, 2), op_bytes(bias2, N, 2)})
        if (op_overlap(y, b)) return "out on top of an input";
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
    const int64_t nb = ((int64_t)K + 31) / 32;
    const OpRows in{w, N, std::min(ldw, OP_FAR) * (int64_t)esz, K * (int64_t)esz}, c = op_bytes(codes, N, 16 * nb), s = op_bytes(scales, N, nb), d = op_bytes(dequantised, N, (int64_t)K * 2);
    const bool in_place = dequantised == w && dtype == MV_BF16 && ldw == K;
    if (op_overlap(c, in) || op_overlap(s, in) || (!in_place && op_overlap(d, in)))
        return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: an output on top of w (dequantised may be w, with bf16 and ldw = K)");
    if (op_overlap(c, s) || op_overlap(c, d) || op_overlap(s, d)) return mv_fail(MV_ERR_INVALID, "quantize_mxfp4: an output on top of another");
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
    const char* fault = ldx < K ? "ldx below K" : nullptr;
    if (!fault && M > 0 && N > 0 && (!x || !op_aligned(x, 2))) fault = "x is null or not aligned to its element";
    if (!fault) fault = product_fault(M, N, K, OpRows{x, M, std::min(ldx, OP_FAR) * 2, (int64_t)K * 2}, nullptr, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out);
    if (fault) return mv_fail(MV_ERR_INVALID, "linear_mxfp4: %s (M=%d N=%d K=%d)", fault, M, N, K);
    if (M == 0 || N == 0) return MV_OK;
    OpDevice dev((hipStream_t)stream, out);
    MX_TRY(dev.status());
    MxArgs a{x, nullptr, (const unsigned char*)codes, (const unsigned char*)scales, (const unsigned char*)codes2, (const unsigned char*)scales2,
             (const bf16_t*)bias, (const bf16_t*)bias2, residual, out, ldx, M, N, K, (K + 31) / 32, out_dtype == MV_F32, 0, 0, 0};
    MX_TRY(launch_products((hipStream_t)stream, a, false));
    return MV_OK;
}

int mv_op_gemm_mxfp4(void* stream, int32_t M, int32_t N, int32_t K, const void* x_codes, const void* x_scales, const void* codes, const void* scales,
                     const void* codes2, const void* scales2, const void* bias, const void* bias2, const void* residual, int32_t out_dtype, void* out) {
    const char* fault = M > 0 && N > 0 && (!x_codes || !x_scales || !op_aligned(x_codes, 16)) ? "x_codes must be aligned to 16 bytes, x_scales not null" : nullptr;
    if (!fault) fault = product_fault(M, N, K, op_bytes(x_codes, M, ((int64_t)K + 31) / 32 * 16), x_scales, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out);
    if (fault) return mv_fail(MV_ERR_INVALID, "gemm_mxfp4: %s (M=%d N=%d K=%d)", fault, M, N, K);
    if (M == 0 || N == 0) return MV_OK;
    OpDevice dev((hipStream_t)stream, out);
    MX_TRY(dev.status());
    MxArgs a{x_codes, (const unsigned char*)x_scales, (const unsigned char*)codes, (const unsigned char*)scales, (const unsigned char*)codes2,
             (const unsigned char*)scales2, (const bf16_t*)bias, (const bf16_t*)bias2, residual, out, 0, M, N, K, (K + 31) / 32, out_dtype == MV_F32, 0, 0, 0};
    MX_TRY(launch_products((hipStream_t)stream, a, true));
    return MV_OK;
}

int mv_debug_mxfp4_kernel(int32_t x4, int32_t M, int32_t N, int32_t K, int64_t ldx, int32_t gated, uint64_t x, uint64_t codes, uint64_t scales, int32_t* out) {
    if (M < 1 || N < 1 || K < 1 || std::max({M, N, K}) > 0x7FFFFFFF - 4096 || (!x4 && ldx < K) || !out) return mv_fail(MV_ERR_INVALID, "debug_mxfp4_kernel: bad argument");
    const unsigned char *w = (const unsigned char*)codes, *ws = (const unsigned char*)scales;
    MxArgs a{(const void*)x, x4 ? ws : nullptr, w, ws, gated ? w : nullptr, gated ? ws : nullptr, nullptr, nullptr, nullptr, nullptr, x4 ? 0 : ldx, M, N, K, (K + 31) / 32, 0, 0, 0, 0};
    const bool lines = product_form(a, x4 != 0);
    x4 ? describe<true>(a, lines, out) : describe<false>(a, lines, out);
    return MV_OK;
}

}  // extern "C"
