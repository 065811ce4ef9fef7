// Controls on next-token logits, before the sampler: guidance mix, penalties for repeated tokens, biases, grammar masks.
//
// For token v of a row, in fp32, rounded once at the end:
//   x = logits[v]                                     with `uncond`: g * logits[v] + (1 - g) * uncond[v], see lc_mix
//   v occurs in the history:                          x = x > 0 ? x / repetition : x * repetition
//   v occurs n > 0 times behind the prompt:           x = x - (n * frequency + presence)
//   v is in the bias list (its last entry holds):     x = x + bias
//   the row's mask has bit v clear:                   x = -inf, whatever stood there (NaN and infinities too)
//
// Split: one workgroup takes LC_CHUNK consecutive tokens of one row and keeps two words per token in LDS, the count from the history and the number of
// the bias entry that holds.  It scans the whole history and bias list of its row and keeps what falls into its chunk: a history is short beside the
// row (and comes from the L2 for all chunks but the first), so this replaces a count array in memory, a launch that clears it and one that fills it.
// Integer adds, ors and maxima in LDS give the same words in any order: results do not depend on timing.  Bound by memory when rows x vocab is large,
// by the latency of one launch with two dependent loads (length, then history) when it is not: 256 x 131072 fp32 in 54 us, 5.0 TB/s (a large copy: 5.1); 64 x
// 32003 bf16 to fp32 with histories of 4096 9.0 us; 1 x 2562 4.8 us.
#include "common.h"
#include "op_common.h"

#include <algorithm>
#include <type_traits>

#define LC_THREADS 512
#define LC_GROUPS 2                                // groups of 4 consecutive tokens per thread
#define LC_CHUNK (LC_THREADS * LC_GROUPS * 4)      // 4096 tokens: two words each are 32 KB of LDS

#define LC_TRY(expr)                                                                                                               \
    do {                                                                                                                           \
        hipError_t _e = (expr);                                                                                                    \
        if (_e != hipSuccess) return mv_fail(MV_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(_e), __FILE__, __LINE__); \
    } while (0)

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

struct ControlArgs {
    mv_logit_controls c;
    const void* logits;
    const void* uncond;
    void* out;
    int32_t* allowed;
    int64_t ld, ld_out;
    int32_t vocab;
    uint32_t rows, chunks, groups;  // chunks of a row, and its workgroups: one more where the mask's bits are counted
};

// 4 consecutive logits of a row from token v on, zero past the vocabulary
template <bool F32>
__device__ __forceinline__ f32x4_t lc_load(const void* base, int64_t at, int left) {
    f32x4_t r = {0, 0, 0, 0};
    if (F32) {
        const float* p = (const float*)base + at;
        if (left >= 4) return *(const f32x4_any*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) r[i] = p[i];
    } else {
        const bf16_t* p = (const bf16_t*)base + at;
        if (left >= 4) {
            const u32x2 q = *(const u32x2_any*)p;
            return f32x4_t{bf_lo(q[0]), bf_hi(q[0]), bf_lo(q[1]), bf_hi(q[1])};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) r[i] = bf2f(p[i]);
    }
    return r;
}

// Guidance mix.  An infinite logit stays, guidance 1 is the conditioned row whatever lies beside it, and beyond 1 a token that the unconditioned row alone
// excludes (u = -inf) stays too, where the formula would make it the only token.  The terms may leave the range of fp32 where the mix does not (both rows
// masked by the type's lowest value): then the difference of the rows is taken first, in halves, none of which is larger than the mix or the rows.
__device__ __forceinline__ float lc_mix(float g, float x, float u) {
    const float y = g * x + (1.f - g) * u;
    if (fabsf(y) < INFINITY) return y;
    if (fabsf(x) == INFINITY || g == 1.f || (u == -INFINITY && g > 1.f)) return x;
    return 2.f * (0.5f * x + (g - 1.f) * (0.5f * x - 0.5f * u));
}

#define LC_AHEAD 4  // history ids per thread that are asked for at once

template <bool IN32, bool OUT32, bool GUIDED>
__global__ void __launch_bounds__(LC_THREADS) logit_controls_kernel(const ControlArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t count[LC_CHUNK];  // bit 31: in the prompt; below: occurrences behind it
    __shared__ __attribute__((aligned(16))) uint32_t entry[LC_CHUNK];  // 1 + the bias entry that holds, 0: none
    const mv_logit_controls& c = a.c;
    const int tid = threadIdx.x;
    const uint32_t id = op_workgroup(), row = id / a.groups, chunk = id - row * a.groups;
    if (row >= a.rows) return;
    const int index = c.masks == nullptr ? -1 : c.mask_index ? c.mask_index[row] : (int)row;
    const uint32_t* mask = index >= 0 && index < c.n_masks ? c.masks + (int64_t)index * c.ld_mask : nullptr;

    if (chunk == a.chunks) {  // behind the chunks of a row: a workgroup that counts the bits of its mask
        int n = 0;
        if (mask) {
#pragma unroll 4
            for (int w = tid; w < (a.vocab + 31) / 32; w += LC_THREADS) {
                const int left = a.vocab - w * 32;
                n += __popc(left >= 32 ? mask[w] : mask[w] & ((1u << left) - 1u));
            }
        } else if (tid == 0) n = a.vocab;
        if (tid == 0) count[0] = 0;
        __syncthreads();
        if (n) atomicAdd(&count[0], (uint32_t)n);
        __syncthreads();
        if (tid == 0) a.allowed[row] = (int32_t)count[0];
        return;
    }

    // Everything that depends on nothing else is asked for first: logits, mask words, the first history and bias ids (a history's room is readable
    // whatever its length), so that the two rounds over LDS wait for memory once.
    const int v0 = (int)(chunk * LC_CHUNK);
    const bool counted = c.history != nullptr, biased = c.bias_ids != nullptr;
    const int len = !counted ? 0 : c.history_len ? min(max(c.history_len[row], 0), c.history_cap) : c.history_cap;
    const int prompt = counted && c.prompt_len ? c.prompt_len[row] : 0;
    const int32_t* h = c.history + (int64_t)row * c.ld_history;
    const int32_t* ids = c.bias_ids + (int64_t)row * c.ld_bias;
    f32x4_t x[LC_GROUPS], u[LC_GROUPS];
    uint32_t word[LC_GROUPS];
#pragma unroll
    for (int j = 0; j < LC_GROUPS; ++j) {
        const int v = v0 + (j * LC_THREADS + tid) * 4, left = a.vocab - v;
        x[j] = left > 0 ? lc_load<IN32>(a.logits, (int64_t)row * a.ld + v, left) : f32x4_t{0, 0, 0, 0};
        u[j] = GUIDED && left > 0 ? lc_load<IN32>(a.uncond, (int64_t)row * a.ld + v, left) : f32x4_t{0, 0, 0, 0};
        word[j] = left > 0 && mask ? mask[v >> 5] : 0xFFFFFFFFu;
    }
    int seen[LC_AHEAD], extra = -1;
#pragma unroll
    for (int k = 0; k < LC_AHEAD; ++k) seen[k] = counted && tid + k * LC_THREADS < c.history_cap ? h[tid + k * LC_THREADS] : -1;
    if (biased && tid < c.n_bias) extra = ids[tid];

    if (counted || biased) {
#pragma unroll
        for (int j = 0; j < LC_GROUPS; ++j) {
            if (counted) *(u32x4*)&count[(j * LC_THREADS + tid) * 4] = u32x4{0, 0, 0, 0};
            if (biased) *(u32x4*)&entry[(j * LC_THREADS + tid) * 4] = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
        const uint32_t width = (uint32_t)min(LC_CHUNK, a.vocab - v0);
        const auto note = [&](int id, int i) {
            const uint32_t k = (uint32_t)id - (uint32_t)v0;
            if (i >= len || k >= width) return;
            if (i < prompt) atomicOr(&count[k], 0x80000000u);
            else atomicAdd(&count[k], 1u);
        };
        if (counted) {
#pragma unroll
            for (int k = 0; k < LC_AHEAD; ++k) note(seen[k], tid + k * LC_THREADS);
            for (int i = tid + LC_AHEAD * LC_THREADS; i < len; i += LC_AHEAD * LC_THREADS) {
#pragma unroll
                for (int k = 0; k < LC_AHEAD; ++k) seen[k] = i + k * LC_THREADS < len ? h[i + k * LC_THREADS] : -1;
#pragma unroll
                for (int k = 0; k < LC_AHEAD; ++k) note(seen[k], i + k * LC_THREADS);
            }
        }
        if (biased) {
            for (int i = tid; i < c.n_bias; i += LC_THREADS) {
                const uint32_t k = (uint32_t)(i == tid ? extra : ids[i]) - (uint32_t)v0;
                if (k < width) atomicMax(&entry[k], (uint32_t)i + 1u);
            }
        }
        __syncthreads();
    }

    const float g = GUIDED ? c.guidance[row] : 0.f;
    const float rho = c.repetition ? c.repetition[row] : 1.f, pres = c.presence ? c.presence[row] : 0.f, freq = c.frequency ? c.frequency[row] : 0.f;
#pragma unroll
    for (int j = 0; j < LC_GROUPS; ++j) {
        const int k = (j * LC_THREADS + tid) * 4, v = v0 + k, left = a.vocab - v;
        if (left <= 0) break;
        if constexpr (GUIDED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = lc_mix(g, x[j][i], u[j][i]);
        }
        if (counted) {
            const u32x4 n4 = *(const u32x4*)&count[k];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (n4[i] == 0) continue;
                x[j][i] = x[j][i] > 0.f ? x[j][i] / rho : x[j][i] * rho;
                const uint32_t n = n4[i] & 0x7FFFFFFFu;
                if (n) x[j][i] -= (float)n * freq + pres;
            }
        }
        if (biased) {
            const u32x4 e4 = *(const u32x4*)&entry[k];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e4[i]) x[j][i] += c.bias[(int64_t)row * c.ld_bias + e4[i] - 1];
        }
        const uint32_t bits = word[j] >> (v & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!((bits >> i) & 1)) x[j][i] = -INFINITY;
        const int64_t at = (int64_t)row * a.ld_out + v;
        if (OUT32) {
            float* o = (float*)a.out + at;
            if (left >= 4) *(f32x4_any*)o = x[j];
            else
                for (int i = 0; i < left; ++i) o[i] = x[j][i];
        } else {
            bf16_t* o = (bf16_t*)a.out + at;
            if (left >= 4) *(u32x2_any*)o = u32x2{pack_bf2(x[j][0], x[j][1]), pack_bf2(x[j][2], x[j][3])};
            else
                for (int i = 0; i < left; ++i) o[i] = f2bf(x[j][i]);
        }
    }
}

}  // namespace

extern "C" int mv_op_logit_controls(void* stream, int32_t rows, int32_t vocab, int32_t dtype, const void* logits, const void* uncond, int64_t ld,
                                    const mv_logit_controls* controls, int32_t out_dtype, void* out, int64_t ld_out, int32_t* allowed) {
    if (rows < 0 || vocab < 1) return mv_fail(MV_ERR_INVALID, "logit_controls: bad shape rows=%d vocab=%d", rows, vocab);
    if ((dtype != MV_BF16 && dtype != MV_F32) || (out_dtype != MV_BF16 && out_dtype != MV_F32))
        return mv_fail(MV_ERR_INVALID, "logit_controls: dtype %d -> %d (MV_BF16 or MV_F32)", dtype, out_dtype);
    if (ld < vocab || ld_out < vocab) return mv_fail(MV_ERR_INVALID, "logit_controls: a row stride (%lld, %lld) is below the vocabulary %d", (long long)ld, (long long)ld_out, vocab);
    if (!controls) return mv_fail(MV_ERR_INVALID, "logit_controls: null argument");
    ControlArgs a{*controls, logits, uncond, out, allowed, ld, ld_out, vocab, (uint32_t)rows, 0, 0};
    mv_logit_controls& c = a.c;
    if (uncond && !c.guidance) return mv_fail(MV_ERR_INVALID, "logit_controls: uncond without guidance");
    if (c.history_cap < 0 || c.n_bias < 0 || c.n_masks < 0) return mv_fail(MV_ERR_INVALID, "logit_controls: a negative count");
    if (std::max({vocab, c.history_cap, c.n_bias}) > 0x7FFFFFFF - LC_CHUNK) return mv_fail(MV_ERR_INVALID, "logit_controls: vocab, history_cap or n_bias is too large");
    if (c.history && c.ld_history < c.history_cap) return mv_fail(MV_ERR_INVALID, "logit_controls: ld_history below history_cap");
    if (!c.history && c.history_cap) return mv_fail(MV_ERR_INVALID, "logit_controls: history_cap without history");
    if (!c.bias_ids != !c.bias || (!c.bias && c.n_bias)) return mv_fail(MV_ERR_INVALID, "logit_controls: bias_ids, bias and n_bias go together");
    if (c.bias && c.ld_bias != 0 && c.ld_bias < c.n_bias) return mv_fail(MV_ERR_INVALID, "logit_controls: ld_bias is neither 0 nor n_bias or more");
    if (!c.masks && (c.n_masks || c.mask_index)) return mv_fail(MV_ERR_INVALID, "logit_controls: n_masks or mask_index without masks");
    if (c.masks && c.ld_mask < (vocab + 31LL) / 32) return mv_fail(MV_ERR_INVALID, "logit_controls: ld_mask below one bit per token");
    if (c.masks && !c.mask_index && c.n_masks < rows) return mv_fail(MV_ERR_INVALID, "logit_controls: %d masks for %d rows and no mask_index", c.n_masks, rows);
    if (rows == 0) return MV_OK;
    if (!logits || !out) return mv_fail(MV_ERR_INVALID, "logit_controls: null argument");
    const size_t ein = dtype == MV_F32 ? 4 : 2, eout = out_dtype == MV_F32 ? 4 : 2;
    if (!op_aligned(logits, ein) || !op_aligned(uncond, ein) || !op_aligned(out, eout)) return mv_fail(MV_ERR_INVALID, "logit_controls: a buffer is not aligned to its element");
    for (const void* p : {(const void*)c.guidance, (const void*)c.repetition, (const void*)c.presence, (const void*)c.frequency, (const void*)c.history, (const void*)c.history_len,
                          (const void*)c.prompt_len, (const void*)c.bias_ids, (const void*)c.bias, (const void*)c.masks, (const void*)c.mask_index, (const void*)allowed})
        if (!op_aligned(p, 4)) return mv_fail(MV_ERR_INVALID, "logit_controls: a buffer is not aligned to its element");
    if ((out == logits || out == uncond) && (dtype != out_dtype || ld != ld_out))
        return mv_fail(MV_ERR_INVALID, "logit_controls: out on top of its input needs the input's dtype and stride");
    if (c.history_cap == 0 || (!c.repetition && !c.presence && !c.frequency)) c.history = nullptr;
    if (c.n_bias == 0) c.bias_ids = nullptr;
    a.chunks = (uint32_t)((vocab + (int64_t)LC_CHUNK - 1) / LC_CHUNK);
    a.groups = a.chunks + (allowed ? 1 : 0);
    if ((int64_t)a.groups * rows > 0x7FFFFFFF) return mv_fail(MV_ERR_INVALID, "logit_controls: rows=%d vocab=%d is too large", rows, vocab);
    const int64_t words = (vocab + 31LL) / 32;
    const auto row_of = [&](const void* p, int64_t stride, size_t e) { return OpRows{p, rows, std::min(stride, OP_FAR) * (int64_t)e, (int64_t)vocab * (int64_t)e}; };
    const auto per_row = [&](const void* p) { return op_bytes(p, rows, 4); };
    const OpRows y = row_of(out, ld_out, eout), n = per_row(allowed), history{c.history, rows, std::min(c.ld_history, OP_FAR) * 4, c.history_cap * 4LL};
    const OpRows ids{c.bias_ids, c.ld_bias ? rows : 1, std::min(c.ld_bias, OP_FAR) * 4, c.n_bias * 4LL}, bias{c.bias, ids.rows, ids.stride, ids.width};
    if (op_overlap(y, n) || (out != logits && op_overlap(y, row_of(logits, ld, ein))) || (out != uncond && op_overlap(y, row_of(uncond, ld, ein))))
        return mv_fail(MV_ERR_INVALID, "logit_controls: out on top of a part of its inputs or of allowed");
    for (const OpRows& b : {row_of(logits, ld, ein), row_of(uncond, ld, ein), per_row(c.guidance), per_row(c.repetition), per_row(c.presence), per_row(c.frequency),
                            per_row(c.history_len), per_row(c.prompt_len), per_row(c.mask_index), history, ids, bias, OpRows{c.masks, c.n_masks, std::min(c.ld_mask, OP_FAR) * 4, words * 4}}) {
        if (op_overlap(n, b)) return mv_fail(MV_ERR_INVALID, "logit_controls: allowed on top of an input");
        if (b.p != logits && b.p != uncond && op_overlap(y, b)) return mv_fail(MV_ERR_INVALID, "logit_controls: out on top of an input");
    }
    OpDevice dev((hipStream_t)stream, out);
    LC_TRY(dev.status());
    const dim3 grid = op_grid((uint64_t)a.groups * rows), block(LC_THREADS);
    const auto launch = [&](auto in32, auto out32) {
        if (uncond) hipLaunchKernelGGL((logit_controls_kernel<decltype(in32)::value, decltype(out32)::value, true>), grid, block, 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((logit_controls_kernel<decltype(in32)::value, decltype(out32)::value, false>), grid, block, 0, (hipStream_t)stream, a);
    };
    if (dtype == MV_F32 && out_dtype == MV_F32) launch(std::true_type{}, std::true_type{});
    else if (dtype == MV_F32) launch(std::true_type{}, std::false_type{});
    else if (out_dtype == MV_F32) launch(std::false_type{}, std::true_type{});
    else launch(std::false_type{}, std::false_type{});
    LC_TRY(hipGetLastError());
    return MV_OK;
}
