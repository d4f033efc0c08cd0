// beam.cu - beam search's selection over beams and vocabulary.
//
// score(b, t) = scores[b] + ((x[b][t] - m[b]) - log(sum_t exp(x[b][t] - m[b]))), m the row's largest:
// every logit is needed once for the sum, and the order of a beam's continuations is the order of its
// logits.  So one pass over the logits does both: a block walks one slice of one row, each thread
// with a running maximum and sum, and collects the logits that can still be among the slice's
// `keep` largest; a second, small kernel joins the slices of each row and then the beams of each
// group.
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
constexpr int kWarps = kThreads / 32;
constexpr int kMaxKeep = 64;
constexpr int kMaxSlices = 32;
constexpr int kItems = 8;                       // logits of a lane in one chunk
constexpr int kChunk = 32 * kItems;             // of a warp
constexpr int kSoft = 2 * kMaxKeep;             // candidates above which a warp cuts them down to the best `keep`
constexpr int kCand = kSoft + kChunk;           // so that a whole chunk always finds room

struct Params {
    const void* x;
    int64_t row_stride;
    const float* scores;
    int groups, beams, vocab, keep, slices, slice_len;   // slice_len: a multiple of kWarps * kChunk
    float2* part;        // [rows][slices] maximum and sum of a slice
    uint64_t* keys;      // [rows][slices][keep] the slice's best, best first; 0 = none
    float* out_scores;
    int32_t* out_beams;
    int32_t* out_tokens;
};

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t ordered_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // -0 orders as +0
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

// Writes the best `keep` of a warp's n candidates to `list`, sorted, by counting for each the
// larger ones; how many there are.
__device__ __forceinline__ int warp_best(const uint64_t* cand, int n, int keep, uint64_t* list, int lane) {
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const uint64_t k = cand[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += cand[j] > k;
        if (rank < keep) list[rank] = k;
    }
    __syncwarp();
    return min(n, keep);
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
    uint64_t bound = lo > hi ? lo : hi;
    if (n_lists > 2 * keep) {   // of many short lists the keep-th largest head bounds better
        uint64_t head[2];   // up to 64 lists
#pragma unroll
        for (int i = 0; i < 2; ++i) head[i] = 32 * i + lane < n_lists ? lists[(32 * i + lane) * keep] : 0;
        uint64_t kth = 0;
        for (int r = 0; r < keep; ++r) {
            const uint64_t top = head[0] > head[1] ? head[0] : head[1];
            const uint32_t bh = __reduce_max_sync(~0u, static_cast<uint32_t>(top >> 32));
            const uint32_t bl = __reduce_max_sync(~0u, static_cast<uint32_t>(top >> 32) == bh ? static_cast<uint32_t>(top) : 0u);
            kth = (static_cast<uint64_t>(bh) << 32) | bl;
#pragma unroll
            for (int i = 0; i < 2; ++i) head[i] = head[i] == kth ? 0 : head[i];
        }
        bound = kth > bound ? kth : bound;
    }
    int n = 0;
    const int total = n_lists * keep;
    for (int i0 = 0; i0 < total; i0 += 256) {   // eight loads in flight a lane
        uint64_t k[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) k[u] = i0 + 32 * u + lane < total ? lists[i0 + 32 * u + lane] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool in = k[u] != 0 && k[u] >= bound;
            const uint32_t mask = __ballot_sync(~0u, in);
            if (in) buf[n + __popc(mask & ((1u << lane) - 1))] = k[u];
            n += __popc(mask);
        }
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const uint64_t k = buf[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += buf[j] > k;
        if (rank < keep) out[rank] = k;
    }
    for (int i = n + lane; i < keep; i += 32) out[i] = 0;
    __syncwarp();
}

// One slice of one row.  Each warp walks its own chunks with its own candidates: a logit is one
// when it is not below the warp's bound.  The first bound comes from all warps' first chunks: each
// takes the r-th largest of its lanes' maxima, r = ceil(keep / warps), and at least keep keys are
// not below the smallest of these.  After 2, 4, 8, 16 and 32 chunks the same with the r-th best
// candidates, so that for logits in no particular order some 2 * keep / c elements of the c-th
// chunks become candidates.  A warp that has more than kSoft cuts them down to its best keep.
// 256 rows of 128256 bf16 (66 MB) take 43 us with the second kernel, 1.5 TB/s: bound by the 20
// instructions a logit, of which the conversion, maximum, sum and comparison need about 8 (block-wide
// bounds met at a barrier every 2048 logits took 61 us, a warp's bound from its own first 256 logits
// 80 us).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) beam_scan_kernel(const Params p) {
    __shared__ uint64_t s_cand[kWarps * kCand];
    __shared__ uint64_t s_list[kWarps * kMaxKeep];
    __shared__ uint64_t s_bound[kWarps];
    __shared__ float s_max[kWarps], s_sum[kWarps];
    __shared__ int s_count[kWarps];
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kVec = VEC ? 16 / static_cast<int>(sizeof(T)) : 1, kLoads = kItems / kVec;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y, slice = blockIdx.x;
    const int lo = slice * p.slice_len, hi = min(p.vocab, lo + p.slice_len);
    const T* x = static_cast<const T*>(p.x) + row * p.row_stride;
    uint64_t* cand = s_cand + warp * kCand;
    uint64_t* list = s_list + warp * p.keep;
    int* count = s_count + warp;
    // a lane's tokens of the warp's c-th chunk ascend with i
    auto token = [&](int c, int i) { return lo + (c * kWarps + warp) * kChunk + (i / kVec * 32 + lane) * kVec + i % kVec; };
    // chunks of this warp that lie in the slice whole: loaded as vectors ahead of time; the ragged
    // end is read by itself
    const int left = hi - lo - warp * kChunk;   // of this warp's part
    const int whole = VEC && left >= kChunk ? (left - kChunk) / (kWarps * kChunk) + 1 : 0;
    const T* mine = x + lo + warp * kChunk + lane * kVec;
    auto fetch = [&](int c, uint4 (&raw)[kLoads]) {
        if (c < whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                raw[i] = __ldcs(reinterpret_cast<const uint4*>(mine + c * (kWarps * kChunk) + i * 32 * kVec));
        }
    };
    auto unpack = [&](int c, const uint4 (&raw)[kLoads], float (&v)[kItems]) {
        if (c < whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if constexpr (sizeof(T) == 4) v[i * kVec + e] = __uint_as_float(u[e % 4]);
                    else v[i * kVec + e] = __uint_as_float(e & 1 ? u[e / 2 % 4] & 0xffff0000u : u[e / 2 % 4] << 16);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int t = token(c, i);
                v[i] = t < hi ? static_cast<float>(x[t]) : -INFINITY;
            }
        }
    };
    const int chunks = left > 0 ? (left + kWarps * kChunk - 1) / (kWarps * kChunk) : 0;
    uint4 raw[2][kLoads];
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if (c < chunks) fetch(c, raw[c]);
    if (lane == 0) *count = 0;
    __syncwarp();
    const bool bounded = hi - lo >= kWarps * kChunk;   // every lane of every warp has a whole first chunk
    const int share = (p.keep + kWarps - 1) / kWarps;
    // the smallest of the warps' keys; every warp calls
    auto join_bounds = [&](uint64_t mine) {
        if (lane == 0) s_bound[warp] = mine;
        __syncthreads();
        uint64_t least = s_bound[0];
        for (int w = 1; w < kWarps; ++w) least = s_bound[w] < least ? s_bound[w] : least;
        __syncthreads();
        return least;
    };
    const int common = (hi - lo) / (kWarps * kChunk);   // chunks that every warp has in whole
    float m = -INFINITY, sum = 0.0f, bound_value = -INFINITY;
    uint64_t bound = 0;
    for (int c0 = 0; c0 < chunks; c0 += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + h;
            if (c >= chunks) break;
            float v[kItems];
            unpack(c, raw[h], v);
            if (c + 2 < chunks) fetch(c + 2, raw[h]);
            float top = v[0];
#pragma unroll
            for (int i = 1; i < kItems; ++i) top = fmaxf(top, v[i]);
            if (top > m) {
                sum *= ex2((m - top) * kLog2e);
                m = top;
            }
            // The difference from the maximum comes before the scaling: it is exact near the maximum,
            // whatever their size, where the rounding of m * log2e alone would be an exponent of 2^8
            // and more beside a mask of -1e10, and overflows for the lowest numbers.  A NaN or +inf
            // logit makes the sum NaN, which kills the row.
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < kItems; ++i) sum += ex2((v[i] - base) * kLog2e);   // a place past the slice adds 0
            if (c == 0 && left >= 32 * kVec && (bounded || p.keep <= 32)) {
                int first = 0;
#pragma unroll
                for (int i = kItems - 1; i >= 0; --i) first = v[i] == top ? token(0, i) : first;
                uint32_t high = ordered_bits(top), low = ~static_cast<uint32_t>(first), bh = 0, bl = 0;
                const int rounds = bounded ? share : p.keep;   // a short slice: each warp for itself
                for (int r = 0; r < rounds; ++r) {   // the maxima, taken out one by one
                    bh = __reduce_max_sync(~0u, high);
                    bl = __reduce_max_sync(~0u, high == bh ? low : 0u);
                    if (high == bh && low == bl) high = low = 0;
                }
                bound = (static_cast<uint64_t>(bh) << 32) | bl;
                if (bounded) bound = join_bounds(bound);
                bound_value = from_ordered(static_cast<uint32_t>(bound >> 32));
            }
            if (__any_sync(~0u, top >= bound_value)) {
                uint32_t some = 0;
#pragma unroll
                for (int i = 0; i < kItems; ++i) some |= v[i] >= bound_value ? 1u << i : 0u;
                if (c >= whole) {   // not what stands for tokens past the slice
#pragma unroll
                    for (int i = 0; i < kItems; ++i)
                        if (token(c, i) >= hi) some &= ~(1u << i);
                }
                while (some) {   // few: read again rather than kept in reach of an index
                    const int t = token(c, __ffs(some) - 1);
                    const uint64_t k = (static_cast<uint64_t>(ordered_bits(static_cast<float>(x[t]))) << 32) | ~static_cast<uint32_t>(t);
                    if (k >= bound) cand[atomicAdd(count, 1)] = k;
                    some &= some - 1;
                }
                __syncwarp();
                const int n = *count;
                if (c + 1 < chunks && n > kSoft) {
                    const int now = warp_best(cand, n, p.keep, list, lane);
                    for (int i = lane; i < now; i += 32) cand[i] = list[i];
                    if (lane == 0) *count = now;
                    if (now == p.keep) {
                        bound = list[p.keep - 1];
                        bound_value = from_ordered(static_cast<uint32_t>(bound >> 32));
                    }
                }
                __syncwarp();
            }
            if (bounded && c + 1 < common && (c == 1 || c == 3 || c == 7 || c == 15 || c == 31)) {
                // the bound follows: the share-th best of each warp so far
                const int now = warp_best(cand, *count, p.keep, list, lane);
                for (int i = lane; i < now; i += 32) cand[i] = list[i];
                if (lane == 0) *count = now;
                __syncwarp();
                const uint64_t joint = join_bounds(now >= share ? list[share - 1] : 0);
                if (joint > bound) {
                    bound = joint;
                    bound_value = from_ordered(static_cast<uint32_t>(bound >> 32));
                }
            }
        }
    }
    const int n = warp_best(cand, *count, p.keep, list, lane);
    for (int i = n + lane; i < p.keep; i += 32) list[i] = 0;
    float bm = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(~0u, bm, o));
    sum *= m == -INFINITY ? 1.0f : ex2((m - bm) * kLog2e);   // a lane that saw -inf only has 0, or NaN
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
        s_max[warp] = bm;
        s_sum[warp] = sum;
    }
    __syncthreads();
    const int64_t at = static_cast<int64_t>(row) * p.slices + slice;
    if (warp == 0) {
        warp_merge(s_list, kWarps, p.keep, s_cand, p.keys + at * p.keep, lane);   // the warps' candidates are done with
    } else if (threadIdx.x == 32) {
        float all = s_max[0], total = 0.0f;
        for (int w = 1; w < kWarps; ++w) all = fmaxf(all, s_max[w]);
        for (int w = 0; w < kWarps; ++w) total += s_max[w] == -INFINITY ? s_sum[w] : s_sum[w] * ex2((s_max[w] - all) * kLog2e);
        p.part[at] = make_float2(all, total);
    }
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
        const float prior = p.scores[row];
        const float2 part = lane < p.slices ? p.part[row * p.slices + lane] : make_float2(-INFINITY, 0.0f);
        float m = part.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float sum = part.x == -INFINITY ? part.y : part.y * ex2((part.x - m) * kLog2e);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        // m and log(sum) stay apart: their sum would round at the size of m
        const float log_sum = logf(sum);
        uint64_t* list = s_list + b * K;
        // every continuation of a dead beam scores -inf: its tokens count in their own order
        const bool dead = !(fabsf(m) < INFINITY) || !(sum < INFINITY) || isnan(prior) || prior == -INFINITY;
        if (dead) {
            for (int i = lane; i < K; i += 32)
                list[i] = i < p.vocab ? (static_cast<uint64_t>(ordered_bits(-INFINITY)) << 32) | ~static_cast<uint32_t>(i) : 0;
        } else {
            warp_merge(p.keys + row * p.slices * K, p.slices, K, buf, list, lane);
        }
        __syncwarp();
        for (int i = lane; i < K; i += 32) {
            const uint64_t k = list[i];
            float sc = dead ? -INFINITY : prior + ((from_ordered(static_cast<uint32_t>(k >> 32)) - m) - log_sum);
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

template <typename T>
static int launch(const Params& p, bool vec, cudaStream_t stream) {
    auto scan = vec ? beam_scan_kernel<T, true> : beam_scan_kernel<T, false>;
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
        keep > static_cast<int64_t>(beams) * vocab || vocab > (1 << 20))
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
    // Slices of whole chunks: two blocks an SM or a few more (1, 2, 4 times as many: 48, 53, 56 us then, at
    // 256 rows of 128256 bf16), but no more than a warp of the second kernel joins at once.
    constexpr int kPiece = beam::kWarps * beam::kChunk;
    const int chunks = static_cast<int>(ceil_div(vocab, kPiece));
    const int wanted = static_cast<int>(std::min<int64_t>({chunks, beam::kMaxSlices, std::max<int64_t>(1, ceil_div(2 * info.sm_count, rows))}));
    beam::Params p{};
    p.x = logits;
    p.row_stride = row_stride;
    p.scores = scores;
    p.groups = groups; p.beams = beams; p.vocab = vocab; p.keep = keep;
    p.slice_len = static_cast<int>(ceil_div(chunks, wanted)) * kPiece;
    p.slices = static_cast<int>(ceil_div(vocab, p.slice_len));
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
    if (logits_dtype == BYBYCU_DT_F32) rc = beam::launch<float>(p, vec, s);
    else rc = beam::launch<__nv_bfloat16>(p, vec, s);
    const cudaError_t fe = cudaFreeAsync(scratch, s);
    if (rc) return rc;
    if (fe != cudaSuccess) return cuda_fail(fe, "cudaFreeAsync(beam scratch)");
    return BYBYCU_OK;
}
