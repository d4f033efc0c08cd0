// attention.cu - attention of new tokens over a paged cache: the checks, the choice of a route,
// and the SIMT route (one warp a query row, fp32 throughout).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.cuh"

namespace bybycu {
namespace attn {

// ---------------------------------------------------------------------------------------
// SIMT route: one warp per (token, head).  32 keys at a time: each lane takes the product with
// one key, the warp joins the running maximum and sum, then every lane adds the 32 probabilities
// times its own dimensions of V.  A masked key's V is never read.  Exact in fp32; for head
// dimensions that the matrix kernels are not built for.
// ---------------------------------------------------------------------------------------
constexpr int kSimtWarps = 4;

template <bool MOD, bool OUTF32>
__global__ void __launch_bounds__(kSimtWarps * 32) attention_simt_kernel(const kvc::Cache c, const Params p) {
    __shared__ __align__(16) float s_q[kSimtWarps][kvc::kMaxHeadDim];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kSimtWarps + warp;
    if (item >= static_cast<int64_t>(c.n_tokens) * p.q_heads) return;
    const int t = static_cast<int>(item / p.q_heads), h = static_cast<int>(item % p.q_heads), D = c.head_dim;
    int b = 0;
    for (int i = 0; i < c.n_seqs; i += 32) b += __popc(__ballot_sync(~0u, i + lane < c.n_seqs && c.q_start[i + lane + 1] <= t));
    if (b >= c.n_seqs || t < c.q_start[0]) return;
    const Seq s = load_seq(c, p, b);
    if (t - s.q0 >= s.rows) return;
    const int pos = s.first_pos + (t - s.q0), kvh = h / p.group;
    int lo, hi;
    row_range(p, s, pos, &lo, &hi);
    for (int d = lane; d < D; d += 32) s_q[warp][d] = __bfloat162float(p.q[t * p.q_token + h * p.q_head + d]);
    __syncwarp();
    const float slope = MOD && p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[kvc::kMaxHeadDim / 32] = {};
    for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        int64_t at = -1;
        float sc = -INFINITY;
        if (j < hi) at = slot_of(c, b, j);
        if (at >= 0) {
            at += kvh * c.head_stride;
            const uint4* kp = reinterpret_cast<const uint4*>(c.k + at);
            float dot = 0.0f;
            for (int d = 0; d < D; d += 8) {
                const uint4 w = kp[d / 8];
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dot = fmaf(s_q[warp][d + 2 * e], __uint_as_float(u[e] << 16), dot);
                    dot = fmaf(s_q[warp][d + 2 * e + 1], __uint_as_float(u[e] & 0xffff0000u), dot);
                }
            }
            sc = score_log2<MOD, true>(p, dot, slope, pos - j);
        }
        float mn = fmaxf(m, sc);
#pragma unroll
        for (int o = 16; o; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(~0u, mn, o));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float keep = exp2f(m - base), pr = exp2f(sc - base);
        m = mn;
        l = l * keep + pr;
#pragma unroll
        for (int e = 0; e < kvc::kMaxHeadDim / 32; ++e) acc[e] *= keep;
        for (int jj = 0; jj < min(32, hi - j0); ++jj) {
            const float w = __shfl_sync(~0u, pr, jj);
            const int64_t a = __shfl_sync(~0u, at, jj);
            if (a < 0) continue;
#pragma unroll
            for (int e = 0; e < kvc::kMaxHeadDim / 32; ++e)
                if (32 * e + lane < D) acc[e] = fmaf(w, __bfloat162float(c.v[a + 32 * e + lane]), acc[e]);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;   // a row that sees nothing gives zeros
#pragma unroll
    for (int e = 0; e < kvc::kMaxHeadDim / 32; ++e) {
        if (32 * e + lane >= D) break;
        const int64_t o = t * p.o_token + h * p.o_head + 32 * e + lane;
        if constexpr (OUTF32) static_cast<float*>(p.out)[o] = acc[e] * inv;
        else static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(acc[e] * inv);
    }
}

static int launch_simt(const kvc::Cache& c, const Params& p, bool mod, bool f32, cudaStream_t stream) {
    const int64_t blocks = ceil_div(static_cast<int64_t>(c.n_tokens) * p.q_heads, kSimtWarps);
    if (blocks > INT32_MAX) return set_error(BYBYCU_ERR_SHAPE, "paged_attention: too many rows");
    auto kern = mod ? (f32 ? attention_simt_kernel<true, true> : attention_simt_kernel<true, false>)
                    : (f32 ? attention_simt_kernel<false, true> : attention_simt_kernel<false, false>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kSimtWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, c, p));
    return BYBYCU_OK;
}

}  // namespace attn
}  // namespace bybycu

using namespace bybycu;

extern "C" int bybycu_paged_attention(const bybycu_paged_kv* kv, const bybycu_attention* a, void* stream) {
    kvc::Cache c;
    if (int rc = kvc::check_cache(kv, "paged_attention", &c)) return rc;
    if (!a) return set_error(BYBYCU_ERR_ARGS, "paged_attention: the arguments are NULL");
    if (a->out_dtype != BYBYCU_DT_F32 && a->out_dtype != BYBYCU_DT_BF16)
        return set_error(BYBYCU_ERR_ARGS, "paged_attention: output type must be F32 or BF16");
    if (a->q_heads <= 0 || a->q_heads % c.kv_heads)
        return set_error(BYBYCU_ERR_SHAPE, "paged_attention: %d query heads over %d kv heads", a->q_heads, c.kv_heads);
    if (a->max_q < 0 || a->max_kv < 0 || a->window < 0)
        return set_error(BYBYCU_ERR_SHAPE, "paged_attention: max_q=%d max_kv=%d window=%d", a->max_q, a->max_kv, a->window);
    if (!std::isfinite(a->scale) || !(a->softcap >= 0.0f) || !std::isfinite(a->softcap))
        return set_error(BYBYCU_ERR_ARGS, "paged_attention: scale %g, softcap %g", a->scale, a->softcap);
    if (a->route != BYBYCU_ROUTE_AUTO && a->route != BYBYCU_ROUTE_SIMT && a->route != BYBYCU_ROUTE_GEMV &&
        a->route != BYBYCU_ROUTE_TC)
        return set_error(BYBYCU_ERR_ARGS, "unknown route %d", a->route);
    if (c.n_tokens == 0 || c.n_seqs == 0) return BYBYCU_OK;
    if (!a->q || !a->out) return set_error(BYBYCU_ERR_ARGS, "paged_attention: a slot is missing");
    const int oal = a->out_dtype == BYBYCU_DT_F32 ? 4 : 8;   // 16-byte output vectors
    if (!kvc::aligned(a->q, 16) || !kvc::aligned(a->out, 16) || !kvc::aligned(a->slopes, 4) || !kvc::aligned(a->prefix_lens, 4) ||
        !kvc::strides_ok(a->q_token_stride, a->q_head_stride, a->q_heads, c.head_dim, 8) ||
        !kvc::out_strides_ok(a->out_token_stride, a->out_head_stride, c.n_tokens, a->q_heads, c.head_dim, oal))
        return set_error(BYBYCU_ERR_ARGS, "paged_attention: q and out need 16-byte aligned vectors that do not overlap");
    // no sequence has more new tokens than there are; a tile's rows (token, head of a group) are counted in 32 bits
    const int max_q = std::min(a->max_q, c.n_tokens);
    if (static_cast<int64_t>(max_q) * (a->q_heads / c.kv_heads) > INT32_MAX - 256)
        return set_error(BYBYCU_ERR_SHAPE, "paged_attention: %d new tokens of %d heads a kv head: 2^31 rows or more", max_q, a->q_heads / c.kv_heads);
    // finite even where the quotient overflows: a score of 0 stays 0 under the smallest cap
    const float cap_in = a->softcap > 0.0f ? std::clamp(a->scale / a->softcap, -FLT_MAX / 4, FLT_MAX / 4) : 0.0f;
    const attn::Params p{static_cast<const __nv_bfloat16*>(a->q), a->out, a->q_token_stride, a->q_head_stride,
                         a->out_token_stride, a->out_head_stride, a->slopes, a->prefix_lens, a->q_heads,
                         a->q_heads / c.kv_heads, max_q, a->max_kv, a->window, a->scale * attn::kLog2e, a->softcap,
                         cap_in, 2.0f * attn::kLog2e * cap_in, a->softcap * attn::kLog2e};
    const bool mod = a->softcap > 0.0f || a->slopes, f32 = a->out_dtype == BYBYCU_DT_F32;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->route == BYBYCU_ROUTE_SIMT) return attn::launch_simt(c, p, mod, f32, s);
    const bool tc = attn::tc_attention_supports(c, p, f32);
    if (a->route == BYBYCU_ROUTE_TC && !tc)
        return set_error(BYBYCU_ERR_SHAPE, "paged_attention: the tensor-core route needs bf16 output, head dimension <= 128, at most "
                                           "128 heads a group, pages of 8, 16, 32, 64 or a multiple of 128 tokens and a token stride of q");
    // A tensor-core tile costs its 128 rows however many there are, the GEMV's warps 16 each: 8
    // sequences of 4096 keys, 8 kv heads of 128, at 16, 32, 64 and 128 rows 51, 64, 88, 153 us on
    // the GEMV and 43, 46, 51, 61 on the tensor cores; heads of 64 33, 41, 53, 93 and 37, 39, 43,
    // 53; one sequence of 2048 15, 17, 21, 23 and 19, 19, 20, 23.  From 33 rows on the tensor cores
    // are ahead in all three.  Up to 32 the rule keeps the GEMV, which one short sequence is faster
    // on; a batch of 17 to 32 rows a kv head is up to 28% slower by it (the number of tiles, which
    // would tell the two apart, is not part of the rule).
    if (a->route == BYBYCU_ROUTE_TC || (a->route == BYBYCU_ROUTE_AUTO && tc && static_cast<int64_t>(max_q) * p.group > 32))
        return attn::launch_tc_attention(c, p, mod, s);
    return attn::launch_gemv(c, p, f32, s);
}
