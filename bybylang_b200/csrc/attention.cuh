// attention.cuh - what the paged-attention kernels share: their parameters, which keys a row
// sees, and the score of a pair.
#pragma once

#include "kvcache.cuh"

namespace bybycu {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    const __nv_bfloat16* q;
    void* out;
    int64_t q_token, q_head, o_token, o_head;
    const float* slopes;
    const int32_t* prefix;
    int32_t q_heads, group, max_q, max_kv, window;   // group: query heads a kv head
    // scale * log2(e); softcap; scale / softcap; 2 log2(e) scale / softcap; softcap * log2(e)
    float scale_log2, cap, cap_in, cap_ex, cap_out;
};

// One sequence of the batch as a kernel reads it.  rows and kv are what may be touched: never past
// the tensors, the table or what the launch was sized for; a sequence that is longer keeps its
// positions, loses the rest and is recorded.
struct Seq {
    int q0, rows, kv, first_pos, prefix;
};

__device__ __forceinline__ Seq load_seq(const kvc::Cache& c, const Params& p, int b) {
    Seq s;
    s.q0 = c.q_start[b];
    const int nq = c.q_start[b + 1] - s.q0, kv = c.kv_lens[b], limit = min(p.max_kv, c.max_pages * c.page_size);
    s.prefix = p.prefix ? p.prefix[b] : 0;
    s.first_pos = kv - nq;
    s.rows = min(nq, p.max_q);
    if (s.q0 < 0 || s.q0 > c.n_tokens) s.rows = 0;
    else s.rows = min(s.rows, c.n_tokens - s.q0);
    s.kv = min(kv, limit);
    if ((s.rows != nq || s.kv != kv) && (threadIdx.x & 31) == 0) record_device_error(kDevErrLength);
    return s;
}

// Keys [lo, hi) that a row at position pos can see: j <= pos or j < prefix, within the cache and
// the window.  Empty (lo >= hi) for a padding row.
__device__ __forceinline__ void row_range(const Params& p, const Seq& s, int pos, int* lo, int* hi) {
    *hi = pos < 0 ? 0 : min(s.kv, max(pos + 1, s.prefix));
    *lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The smaller and the larger of two numbers, NaN where either is: a NaN score is not clamped away.
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// A capped score: cap * tanh(y) in units of log2, y = raw * scale / cap.
//   plain:  cap * (1 - 2 / (1 + e^2y)), off by some 1e-7 of the cap wherever y is.  For a bf16
//           output and caps up to kCapPlain that is 3e-5 of a score, far below the rounding of a
//           probability; at a cap of 1e6 it made probabilities wrong by 9%
//   exact:  for |y| < 0.6  s * (1 + y^2 P(y^2)), s the score without a cap, P of degree 4 (tanh(y)
//           to 4.2e-9 of itself, a Chebyshev fit), and the plain form above, where it is good to
//           2^-22 of itself: off by a few 2^-24 of the score, however large the cap.
constexpr float kCapPlain = 256.0f;
constexpr float kCapBend = 0.6f;   // where the two forms of `exact` meet
constexpr float kCapP0 = -0.333332956f, kCapP1 = 0.133318797f, kCapP2 = -0.0537803993f, kCapP3 = 0.0207851473f, kCapP4 = -0.00588323316f;

__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float capped_plain(const Params& p, float raw) {
    return fmaf(-2.0f * p.cap_out, rcp(1.0f + ex2(raw * p.cap_ex)), p.cap_out);
}
__device__ __forceinline__ float capped_small(const Params& p, float raw) {
    const float y = raw * p.cap_in, z = y * y, s = raw * p.scale_log2;
    return fmaf(s * z, fmaf(fmaf(fmaf(fmaf(kCapP4, z, kCapP3), z, kCapP2), z, kCapP1), z, kCapP0), s);
}
__device__ __forceinline__ float capped_exact(const Params& p, float raw) {
    const float small = capped_small(p, raw), large = capped_plain(p, raw);
    return fabsf(raw * p.cap_in) < kCapBend ? small : large;   // a NaN goes through
}
// The plain form of two scores with one reciprocal.  The exponents are held below 60, where tanh is
// 1 in fp32, so that the product of the two denominators stays finite.
__device__ __forceinline__ float2 capped_plain(const Params& p, float raw0, float raw1) {
    const float a = 1.0f + ex2(min_nan(raw0 * p.cap_ex, 60.0f)), b = 1.0f + ex2(min_nan(raw1 * p.cap_ex, 60.0f));
    const float r = rcp(a * b);
    return make_float2(fmaf(-2.0f * p.cap_out, r * b, p.cap_out), fmaf(-2.0f * p.cap_out, r * a, p.cap_out));
}

// The score of a pair in units of log2: raw = q . k, MOD: a cap (EXACT: for an fp32 output) and / or
// distance slopes.
template <bool MOD, bool EXACT>
__device__ __forceinline__ float score_log2(const Params& p, float raw, float slope_log2, int distance) {
    if constexpr (!MOD) {
        return raw * p.scale_log2;
    } else {
        float s = raw * p.scale_log2;
        if (p.cap > 0.0f) s = EXACT || p.cap > kCapPlain ? capped_exact(p, raw) : capped_plain(p, raw);
        return s - slope_log2 * static_cast<float>(distance < 0 ? -distance : distance);
    }
}

// Where the token at position j of sequence b is, or -1 (recorded) for a page that does not exist.
__device__ __forceinline__ int64_t slot_of(const kvc::Cache& c, int b, int j) {
    const int pg = j / c.page_size;
    const int id = c.page_table[b * c.table_stride + pg];
    if (id < 0 || id >= c.n_pages) {
        record_device_error(kDevErrPage);
        return -1;
    }
    return id * c.page_stride + (j - pg * c.page_size) * c.token_stride;
}

// Four dimensions of a finished row: sums over their total, zeros for a row that saw nothing.
template <bool F32>
__device__ __forceinline__ void store_row4(const Params& p, int64_t token, int64_t head, int d, float4 acc, float sum) {
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int64_t at = token * p.o_token + head * p.o_head + d;
    if constexpr (F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
        __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = *reinterpret_cast<const uint2*>(h);
    }
}

}  // namespace attn
}  // namespace bybycu
