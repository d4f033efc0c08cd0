// beam.cu - beam search's selection over beams and vocabulary.
//
// score(b, t) = scores[b] + (x[b][t] - lse[b]), lse[b] = m + log(sum_t exp(x[b][t] - m)): every
// logit is needed once for the sum, and the order of a beam's continuations is the order of its
// logits.  So one pass over the logits does both: a block reads one slice of one row into
// registers, reduces its maximum and sum, and keeps the slice's `keep` largest logits; a second,
// small kernel joins the slices of each row and then the beams of each group.
//
// Order is kept in whole numbers: a candidate is the 64-bit key (ordered bits of the logit, then
// the complement of the token), so no two keys are equal, equal logits go to the lower token and
// the result depends on no order of execution.
#include <algorithm>

#include "kvcache.cuh"

namespace bybycu {

static int scratch_pool(int device, cudaMemPool_t* pool);

namespace beam {

constexpr int kThreads = 256;
constexpr int kMaxKeep = 64;
constexpr int kMaxSlices = 128;
constexpr int kCand = 512;      // candidates of a slice that are ranked against each other

struct Params {
    const void* x;
    int64_t row_stride;
    const float* scores;
    int groups, beams, vocab, keep, slices;
    float2* part;        // [rows][slices] maximum and sum of a slice
    uint64_t* keys;      // [rows][slices][keep] the slice's best, best first; 0 = none
    float* out_scores;
    int32_t* out_beams;
    int32_t* out_tokens;
};

__device__ __forceinline__ uint32_t ordered_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // -0 orders as +0
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

// One slice of kThreads * ITEMS logits of one row, in registers.  Which of them can be among the
// slice's `keep` largest: every warp whose 32 threads all have tokens takes the r-th largest of
// its threads' own maxima, r = ceil(keep / warps); at least keep keys are not below the smallest
// of these, so it bounds the result from below, and for logits in no particular order some 2 *
// keep elements reach it.  Where more than kCand do (a warp whose tokens are all masked, a slice
// too short for a bound), a bisection over the keys finds the exact bound instead.
template <typename T, int ITEMS, bool VEC>
__global__ void __launch_bounds__(kThreads) beam_scan_kernel(const Params p) {
    __shared__ uint64_t s_cand[kCand];
    __shared__ float s_red[2][kThreads / 32];
    __shared__ uint64_t s_bound[kThreads / 32];
    __shared__ int s_count;
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kVec = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
    constexpr int kWarps = kThreads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.y, slice = blockIdx.x;
    const int base = slice * (kThreads * ITEMS);
    const T* x = static_cast<const T*>(p.x) + row * p.row_stride;
    // a thread's tokens ascend with i
    auto token = [&](int i) { return base + (i / kVec * kThreads + tid) * kVec + i % kVec; };
    auto key = [&](float v, int t) { return (static_cast<uint64_t>(ordered_bits(v)) << 32) | ~static_cast<uint32_t>(t); };
    float v[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i += kVec) {
        const int t = token(i);
        if (VEC && t + kVec <= p.vocab) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + t));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                if constexpr (sizeof(T) == 4) v[i + e] = __uint_as_float(u[e % 4]);
                else v[i + e] = __uint_as_float(e & 1 ? u[e / 2 % 4] & 0xffff0000u : u[e / 2 % 4] << 16);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[i + e] = t + e < p.vocab ? static_cast<float>(x[t + e]) : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) m = fmaxf(m, v[i]);
    float bm = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(~0u, bm, o));
    if (lane == 0) s_red[0][warp] = bm;
    if (tid == 0) s_count = 0;
    // the warp's r-th largest of its threads' maxima, taken out one by one
    const int threads_used = min(kThreads, (p.vocab - base + kVec - 1) / kVec);
    const int full = threads_used / 32;
    const bool bounded = full * 32 >= p.keep;
    if (bounded && warp < full) {
        int first = 0;
#pragma unroll
        for (int i = ITEMS - 1; i >= 0; --i) first = v[i] == m ? token(i) : first;
        uint32_t hi = ordered_bits(m), lo = ~static_cast<uint32_t>(first);
        const int rounds = (p.keep + full - 1) / full;
        uint32_t bh = 0, bl = 0;
        for (int r = 0; r < rounds; ++r) {
            bh = __reduce_max_sync(~0u, hi);
            bl = __reduce_max_sync(~0u, hi == bh ? lo : 0u);
            if (hi == bh && lo == bl) hi = lo = 0;
        }
        if (lane == 0) s_bound[warp] = (static_cast<uint64_t>(bh) << 32) | bl;
    }
    __syncthreads();
    bm = s_red[0][0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bm = fmaxf(bm, s_red[0][w]);
    // sum of exp(v - bm); a NaN or +inf logit makes it NaN, which kills the row
    float sum = 0.0f;
    if (bm != -INFINITY) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) sum += __expf(v[i] - bm);   // a place past the vocabulary adds 0
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) sum += isnan(v[i]) ? v[i] : 0.0f;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) s_red[1][warp] = sum;
    uint64_t bound = 0;
    if (bounded) {
        bound = s_bound[0];
        for (int w = 1; w < full; ++w) bound = s_bound[w] < bound ? s_bound[w] : bound;
    }
    auto collect = [&]() {
        const float bound_value = bound ? from_ordered(static_cast<uint32_t>(bound >> 32)) : -INFINITY;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!(v[i] < bound_value) && token(i) < p.vocab) {
                const uint64_t k = key(v[i], token(i));
                if (k >= bound) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < kCand) s_cand[at] = k;
                }
            }
    };
    collect();
    __syncthreads();
    if (s_count > kCand) {   // the same for every thread
        // the largest bound that keep keys reach, one bit at a time
        bound = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t tried = bound | (1ull << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) n += token(i) < p.vocab && key(v[i], token(i)) >= tried;
            n = __reduce_add_sync(~0u, n);
            __syncthreads();
            if (lane == 0) s_bound[warp] = n;
            __syncthreads();
            n = 0;
            for (int w = 0; w < kWarps; ++w) n += static_cast<int>(s_bound[w]);
            if (n >= p.keep) bound = tried;
        }
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        collect();
        __syncthreads();
    }
    const int n = s_count;
    uint64_t* out = p.keys + (static_cast<int64_t>(row) * p.slices + slice) * p.keep;
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t k = s_cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_cand[j] > k;
        if (rank < p.keep) out[rank] = k;
    }
    for (int i = n + tid; i < p.keep; i += kThreads) out[i] = 0;
    if (tid == 0) {
        float total = 0.0f;
        for (int w = 0; w < kWarps; ++w) total += s_red[1][w];
        p.part[static_cast<int64_t>(row) * p.slices + slice] = make_float2(bm, total);
    }
}

// The `keep` largest of n_lists sorted lists of `keep` keys each, by one warp, into out[keep]
// (sorted, 0 where there are fewer).  Every list's e-th entry, e = ceil(keep / n_lists), bounds
// the result from below through the smallest of them, as does any list's last entry.
__device__ __forceinline__ void warp_merge(const uint64_t* lists, int n_lists, int keep, uint64_t* buf, uint64_t* out,
                                           int lane) {
    const int e = (keep + n_lists - 1) / n_lists - 1;
    uint64_t lo = ~0ull, hi = 0;
    for (int l = lane; l < n_lists; l += 32) {
        const uint64_t a = lists[l * keep + e], z = lists[l * keep + keep - 1];
        lo = a < lo ? a : lo;
        hi = z > hi ? z : hi;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(~0u, lo, o), z = __shfl_xor_sync(~0u, hi, o);
        lo = a < lo ? a : lo;
        hi = z > hi ? z : hi;
    }
    const uint64_t bound = lo > hi ? lo : hi;
    int n = 0;
    const int total = n_lists * keep;
    for (int i0 = 0; i0 < total; i0 += 32) {
        const uint64_t k = i0 + lane < total ? lists[i0 + lane] : 0;
        const bool in = k != 0 && k >= bound;
        const uint32_t mask = __ballot_sync(~0u, in);
        if (in) buf[n + __popc(mask & ((1u << lane) - 1))] = k;
        n += __popc(mask);
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const uint64_t k = buf[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += buf[j] > k;
        if (rank < keep) out[rank] = k;
    }
    for (int i = n + lane; i < keep; i += 32) out[i] = 0;
    __syncwarp();
}

// One block per group: each warp joins the slices of its beams, then warp 0 the beams.
// Dynamic shared memory: [beams][keep] tokens' keys, [beams][keep] final keys, and a buffer of
// buf_keys keys per warp.
__global__ void beam_merge_kernel(const Params p, int buf_keys) {
    extern __shared__ __align__(16) uint64_t s_mem[];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int g = blockIdx.x, K = p.keep;
    uint64_t* s_list = s_mem;
    uint64_t* s_final = s_list + p.beams * K;
    uint64_t* buf = s_final + p.beams * K + warp * buf_keys;
    for (int b = warp; b < p.beams; b += warps) {
        const int64_t row = static_cast<int64_t>(g) * p.beams + b;
        float m = -INFINITY;
        for (int s = lane; s < p.slices; s += 32) m = fmaxf(m, p.part[row * p.slices + s].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float sum = 0.0f;
        for (int s = lane; s < p.slices; s += 32) {
            const float2 v = p.part[row * p.slices + s];
            sum += v.x == -INFINITY ? v.y : v.y * __expf(v.x - m);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        const float lse = m + logf(sum);
        const float prior = p.scores[row];
        uint64_t* list = s_list + b * K;
        // every continuation of a dead beam scores -inf: its tokens count in their own order
        const bool dead = !(fabsf(lse) < INFINITY) || isnan(prior) || prior == -INFINITY;
        if (dead) {
            for (int i = lane; i < K; i += 32)
                list[i] = i < p.vocab ? (static_cast<uint64_t>(ordered_bits(-INFINITY)) << 32) | ~static_cast<uint32_t>(i) : 0;
        } else {
            warp_merge(p.keys + row * p.slices * K, p.slices, K, buf, list, lane);
        }
        __syncwarp();
        for (int i = lane; i < K; i += 32) {
            const uint64_t k = list[i];
            float sc = dead ? -INFINITY : prior + (from_ordered(static_cast<uint32_t>(k >> 32)) - lse);
            if (isnan(sc)) sc = -INFINITY;
            s_final[b * K + i] = k ? (static_cast<uint64_t>(ordered_bits(sc)) << 32) | ~static_cast<uint32_t>(b * kMaxKeep + i) : 0;
        }
    }
    __syncthreads();
    if (warp) return;
    uint64_t* best = s_final + p.beams * K + buf_keys - K;   // the end of warp 0's buffer
    warp_merge(s_final, p.beams, K, buf, best, lane);
    for (int i = lane; i < K; i += 32) {
        const uint64_t k = best[i];
        const uint32_t place = ~static_cast<uint32_t>(k);
        const int b = place / kMaxKeep, r = place % kMaxKeep;
        const int64_t at = static_cast<int64_t>(g) * K + i;
        p.out_scores[at] = from_ordered(static_cast<uint32_t>(k >> 32));
        p.out_beams[at] = b;
        p.out_tokens[at] = static_cast<int32_t>(~static_cast<uint32_t>(s_list[b * K + r]));
    }
}

template <typename T, int ITEMS>
static int launch(const Params& p, bool vec, cudaStream_t stream) {
    auto scan = vec ? beam_scan_kernel<T, ITEMS, true> : beam_scan_kernel<T, ITEMS, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.slices), static_cast<unsigned>(p.groups * p.beams));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, scan, p));
    // a warp's buffer holds every key of a beam's slices, or of the beams, and the final list
    const int buf = std::max(p.slices, p.beams) * p.keep + p.keep;
    const size_t lists = static_cast<size_t>(2) * p.beams * p.keep * 8;
    const int warps = std::max(1, std::min({8, p.beams, static_cast<int>((200 * 1024 - lists) / (static_cast<size_t>(buf) * 8))}));
    const size_t smem = lists + static_cast<size_t>(warps) * buf * 8;
    if (smem > 48 * 1024)
        BYBYCU_CUDA_TRY(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024));
    cfg.gridDim = dim3(static_cast<unsigned>(p.groups));
    cfg.blockDim = dim3(static_cast<unsigned>(warps * 32));
    cfg.dynamicSmemBytes = smem;
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, beam_merge_kernel, p, buf));
    return BYBYCU_OK;
}

}  // namespace beam
}  // namespace bybycu

using namespace bybycu;

extern "C" int bybycu_beam_select(const void* logits, int logits_dtype, int64_t row_stride, const float* scores,
                                  int groups, int beams, int vocab, int keep, float* out_scores, int32_t* out_beams,
                                  int32_t* out_tokens, void* stream) {
    if (logits_dtype != BYBYCU_DT_F32 && logits_dtype != BYBYCU_DT_BF16)
        return set_error(BYBYCU_ERR_ARGS, "beam_select: logits must be F32 or BF16");
    if (groups < 0 || beams < 1 || beams > 64 || vocab < 1 || keep < 1 || keep > beam::kMaxKeep ||
        keep > static_cast<int64_t>(beams) * vocab || vocab > beam::kThreads * 32 * beam::kMaxSlices)
        return set_error(BYBYCU_ERR_SHAPE, "beam_select: groups=%d beams=%d vocab=%d keep=%d", groups, beams, vocab, keep);
    if (static_cast<int64_t>(groups) * beams > 65535)
        return set_error(BYBYCU_ERR_SHAPE, "beam_select: more than 65535 rows (%d groups of %d beams)", groups, beams);
    if (groups == 0) return BYBYCU_OK;
    if (!logits || !scores || !out_scores || !out_beams || !out_tokens)
        return set_error(BYBYCU_ERR_ARGS, "beam_select: a slot is missing");
    const int esz = logits_dtype == BYBYCU_DT_F32 ? 4 : 2;
    if (row_stride < vocab || !kvc::aligned(logits, esz) || !kvc::aligned(scores, 4) || !kvc::aligned(out_scores, 4) ||
        !kvc::aligned(out_beams, 4) || !kvc::aligned(out_tokens, 4))
        return set_error(BYBYCU_ERR_ARGS, "beam_select: rows overlap or a slot is misaligned");
    DeviceInfo info;
    if (int rc = current_device_info(&info)) return rc;
    const int64_t rows = static_cast<int64_t>(groups) * beams;
    // 32 logits a thread, or 8 where that would leave the card half empty
    const bool small = rows * ceil_div(vocab, beam::kThreads * 32) < 2 * info.sm_count &&
                       ceil_div(vocab, beam::kThreads * 8) <= beam::kMaxSlices;
    beam::Params p{};
    p.x = logits;
    p.row_stride = row_stride;
    p.scores = scores;
    p.groups = groups; p.beams = beams; p.vocab = vocab; p.keep = keep;
    p.slices = static_cast<int>(ceil_div(vocab, beam::kThreads * (small ? 8 : 32)));
    p.out_scores = out_scores; p.out_beams = out_beams; p.out_tokens = out_tokens;
    const bool vec = kvc::aligned(logits, 16) && row_stride * esz % 16 == 0;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaMemPool_t pool = nullptr;
    if (int rc = scratch_pool(info.device, &pool)) return rc;
    const size_t key_bytes = static_cast<size_t>(rows) * p.slices * keep * 8;
    void* scratch = nullptr;
    BYBYCU_CUDA_TRY(cudaMallocFromPoolAsync(&scratch, key_bytes + static_cast<size_t>(rows) * p.slices * 8, pool, s));
    p.keys = static_cast<uint64_t*>(scratch);
    p.part = reinterpret_cast<float2*>(static_cast<char*>(scratch) + key_bytes);
    int rc;
    if (logits_dtype == BYBYCU_DT_F32) rc = small ? beam::launch<float, 8>(p, vec, s) : beam::launch<float, 32>(p, vec, s);
    else rc = small ? beam::launch<__nv_bfloat16, 8>(p, vec, s) : beam::launch<__nv_bfloat16, 32>(p, vec, s);
    const cudaError_t fe = cudaFreeAsync(scratch, s);
    if (rc) return rc;
    if (fe != cudaSuccess) return cuda_fail(fe, "cudaFreeAsync(beam scratch)");
    return BYBYCU_OK;
}
