// kvcache.cu - rotary positions with the append of new keys and values to a paged cache, and the
// copies of pages (forks, compaction).  Both are pure data movement for the memory system.
#include <algorithm>
#include <vector>

#include "kvcache.cuh"

namespace bybycu {
namespace kvc {

// ---------------------------------------------------------------------------------------
// rope_append
//
// Of token t at position p: (x, y) -> m (x cos a - y sin a, x sin a + y cos a) for each pair i,
// a = 2 pi frac(p * turns[i]).  The product is taken in fp64 and only its fraction converted to
// fp32: an fp32 angle at position 30000 is off by up to 2^-10 rad, which a bf16 key still shows.
// One block per token: its angles once (an fp64 product and sincospif a pair, shared by all heads),
// then every vector of 8 values of q, k and v, the first of them loaded before the angles are
// worked out.  Bound by HBM for prompts (6521 tokens of 32 + 2 x 8 heads of 128, fp32 in, 240 MB:
// 45 us, 5.3 TB/s; 256 threads a block 47), by latency for single tokens (6 us).
// ---------------------------------------------------------------------------------------
struct RopeParams {
    const void *q, *k, *v;
    __nv_bfloat16* q_out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    const double* turns;
    const int32_t* positions;
    int32_t q_heads, pairs;
    float magnitude;
};

constexpr int kRopeThreads = 128;

// VEC values as they lie in memory: loads that are issued long before their values are needed.
template <typename T, int VEC>
struct RawVec {
    static constexpr int kWords = VEC * static_cast<int>(sizeof(T)) / 16;   // 16-byte words of a whole vector
    uint4 w[kWords > 0 ? kWords : 1];
    T s[1];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC == 1) {
            s[0] = *p;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        }
    }
    __device__ __forceinline__ void values(float (&x)[VEC]) const {
        if constexpr (VEC == 1) {
            x[0] = static_cast<float>(s[0]);
        } else {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(u[i]);
                else x[i] = __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
            }
        }
    }
};

template <int N>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&x)[N]) {
    if constexpr (N == 8) {
        uint4 a;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = a;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = __float2bfloat16_rn(x[i]);
    }
}

// VEC: values of a vector access (8 where the layout allows 16-byte accesses, else 1).  A unit is
// one vector, or the two that a rotation pairs: i and i + pairs (half layout), or for single
// values 2i and 2i + 1 (whole vectors of the interleaved layout hold their own pairs).
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const Cache c, const RopeParams p) {
    __shared__ float s_cos[kMaxHeadDim / 2], s_sin[kMaxHeadDim / 2];
    constexpr bool kTwo = !INTERLEAVED || VEC == 1;          // a turned unit is two vectors
    constexpr int kStep = INTERLEAVED && VEC == 1 ? 2 : VEC; // dimensions between turned units
    constexpr int kBatch = 2;                                // units of a thread in flight
    const int t = blockIdx.x, D = c.head_dim, R = 2 * p.pairs;
    const int turned = INTERLEAVED ? R / kStep : p.pairs / VEC, units = turned + (D - R) / VEC;
    const int qk = (p.q_heads + c.kv_heads) * units, total = qk + c.kv_heads * (D / VEC);
    struct Unit {
        RawVec<T, VEC> x, y;
        int h, d;            // head (q, then k, then v), first dimension
        bool pair;
    };
    const int apart = INTERLEAVED ? 1 : p.pairs;
    auto fetch = [&](int u, Unit& n) {
        const T* src;
        n.pair = false;
        if (u >= qk) {
            n.h = p.q_heads + c.kv_heads + (u - qk) / (D / VEC);
            n.d = (u - qk) % (D / VEC) * VEC;
            src = static_cast<const T*>(p.v) + t * p.v_token + (n.h - p.q_heads - c.kv_heads) * p.v_head + n.d;
        } else {
            const int i = u % units;
            n.h = u / units;
            n.pair = i < turned;
            n.d = n.pair ? i * kStep : R + (i - turned) * VEC;
            src = (n.h < p.q_heads ? static_cast<const T*>(p.q) + t * p.q_token + n.h * p.q_head
                                   : static_cast<const T*>(p.k) + t * p.k_token + (n.h - p.q_heads) * p.k_head) + n.d;
        }
        n.x.load(src);
        if (kTwo && n.pair) n.y.load(src + apart);
    };
    pdl_launch_dependents();
    pdl_wait();
    // the first units are on their way while the token's place and angles are worked out
    Unit unit[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (static_cast<int>(threadIdx.x) + i * kRopeThreads < total) fetch(threadIdx.x + i * kRopeThreads, unit[i]);
    const int b = block_seq_of(c, t);
    if (b >= c.n_seqs || t < c.q_start[0]) return;   // a row of no sequence
    const int pos = c.kv_lens[b] - (c.q_start[b + 1] - t);
    const int turn_pos = p.positions ? p.positions[t] : pos;
    for (int i = threadIdx.x; i < p.pairs; i += kRopeThreads) {
        const double turn = static_cast<double>(turn_pos) * p.turns[i];
        float sn, cs;
        sincospif(2.0f * static_cast<float>(turn - rint(turn)), &sn, &cs);
        s_cos[i] = p.magnitude * cs;
        s_sin[i] = p.magnitude * sn;
    }
    // the new token's slot
    int64_t slot = -1;
    if (pos >= 0) {
        const int pg = pos / c.page_size;
        const int id = pg < c.max_pages ? c.page_table[b * c.table_stride + pg] : -1;
        if (id >= 0 && id < c.n_pages) slot = id * c.page_stride + (pos - pg * c.page_size) * c.token_stride;
        else if (threadIdx.x == 0) record_device_error(kDevErrPage);
    }
    __syncthreads();
    auto finish = [&](const Unit& n) {
        __nv_bfloat16* dst;
        if (n.h < p.q_heads) dst = p.q_out + t * p.o_token + n.h * p.o_head;
        else if (slot < 0) return;
        else if (n.h < p.q_heads + c.kv_heads) dst = c.k + slot + (n.h - p.q_heads) * c.head_stride;
        else dst = c.v + slot + (n.h - p.q_heads - c.kv_heads) * c.head_stride;
        float x[VEC], y[VEC];
        n.x.values(x);
        if constexpr (kTwo) {
            if (n.pair) {
                n.y.values(y);
                const int i0 = INTERLEAVED ? n.d / 2 : n.d;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float cs = s_cos[i0 + e], sn = s_sin[i0 + e], a = x[e] * cs - y[e] * sn;
                    y[e] = x[e] * sn + y[e] * cs;
                    x[e] = a;
                }
            }
        } else if (n.pair) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float cs = s_cos[(n.d + e) / 2], sn = s_sin[(n.d + e) / 2], a = x[e] * cs - x[e + 1] * sn;
                x[e + 1] = x[e] * sn + x[e + 1] * cs;
                x[e] = a;
            }
        }
        if (pos < 0) {   // a padding token's q row is zero
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = y[e] = 0.0f;
        }
        store_vec<VEC>(dst + n.d, x);
        if (kTwo && n.pair) store_vec<VEC>(dst + n.d + apart, y);
    };
    for (int u = threadIdx.x; u < total; u += kBatch * kRopeThreads) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (u + i * kRopeThreads < total) finish(unit[i]);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (u + (kBatch + i) * kRopeThreads < total) fetch(u + (kBatch + i) * kRopeThreads, unit[i]);
    }
}

template <typename T>
static int launch_rope(const Cache& c, const RopeParams& p, bool interleaved, bool vec, cudaStream_t stream) {
    auto kern = vec ? (interleaved ? rope_append_kernel<T, 8, true> : rope_append_kernel<T, 8, false>)
                    : (interleaved ? rope_append_kernel<T, 1, true> : rope_append_kernel<T, 1, false>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.n_tokens));
    cfg.blockDim = dim3(kRopeThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, c, p));
    return BYBYCU_OK;
}

// ---------------------------------------------------------------------------------------
// copy_pages
//
// Each block moves one piece of one page of one layer of K or V.  The pairs ride in the launch's
// parameters, so a call needs no copy to the device and keeps nothing alive after it returns.
// Bound by HBM: 256 pages of 8 layers (2 x 537 MB) in 166 us, 6.5 TB/s; 4 small pages 4 us.
// ---------------------------------------------------------------------------------------
constexpr int kCopyPairs = 1000;       // pairs of one launch: 8000 bytes of parameters,
constexpr int kCopyFew = 56;           // or 448 where there are few (the launch copies them all)
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;         // 16-byte loads in flight per thread
constexpr int kCopyPiece = kCopyThreads * kCopyUnroll * 16;   // 16 KiB

template <int N>
struct CopyParams {
    char* base[2];
    int64_t layer_stride, page_stride, page_bytes;
    int32_t pieces, n_tensors, n_layers;
    int32_t pairs[2 * N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
    pdl_launch_dependents();
    pdl_wait();
    const int pair = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    char* base = (blockIdx.z ? p.base[1] : p.base[0]) + blockIdx.y * p.layer_stride;
    const uint4* src = reinterpret_cast<const uint4*>(base + p.pairs[2 * pair] * p.page_stride);
    uint4* dst = reinterpret_cast<uint4*>(base + p.pairs[2 * pair + 1] * p.page_stride);
    const int64_t n = p.page_bytes / 16;
    const int64_t i0 = static_cast<int64_t>(piece) * (kCopyPiece / 16) + threadIdx.x;
    uint4 x[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (i0 + u * kCopyThreads < n) x[u] = __ldcs(src + i0 + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (i0 + u * kCopyThreads < n) __stcs(dst + i0 + u * kCopyThreads, x[u]);
}

template <int N>
static int launch_copy(CopyParams<N>& p, const int32_t* pairs, int n, cudaStream_t stream) {
    std::copy(pairs, pairs + 2 * n, p.pairs);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(n * p.pieces), static_cast<unsigned>(p.n_layers), p.n_tensors);
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, copy_pages_kernel<N>, p));
    return BYBYCU_OK;
}

template <int N>
static int copy_all(void* k, void* v, int n_layers, int64_t layer_stride, int64_t page_stride, int64_t page_bytes,
                    int pieces, const int32_t* pairs, int n_pairs, cudaStream_t stream) {
    CopyParams<N> p;
    p.base[0] = static_cast<char*>(k);
    p.base[1] = static_cast<char*>(v);
    p.layer_stride = layer_stride;
    p.page_stride = page_stride;
    p.page_bytes = page_bytes;
    p.pieces = pieces;
    p.n_layers = n_layers;
    p.n_tensors = v ? 2 : 1;
    for (int at = 0; at < n_pairs; at += N)
        if (int rc = launch_copy(p, pairs + 2 * at, std::min(N, n_pairs - at), stream)) return rc;
    return BYBYCU_OK;
}

}  // namespace kvc
}  // namespace bybycu

using namespace bybycu;

extern "C" {

int bybycu_rope_append(const bybycu_paged_kv* kv, const bybycu_rope* r, void* stream) {
    kvc::Cache c;
    if (int rc = kvc::check_cache(kv, "rope_append", &c)) return rc;
    if (!r) return set_error(BYBYCU_ERR_ARGS, "rope_append: the arguments are NULL");
    if (r->in_dtype != BYBYCU_DT_F32 && r->in_dtype != BYBYCU_DT_BF16)
        return set_error(BYBYCU_ERR_ARGS, "rope_append: element type must be F32 or BF16");
    if (r->reserved) return set_error(BYBYCU_ERR_ARGS, "rope_append: reserved fields must be 0");
    if (r->q_heads <= 0 || r->q_heads > 65535 || c.kv_heads > 65535 || r->pairs < 0 || r->pairs > c.head_dim / 2)
        return set_error(BYBYCU_ERR_SHAPE, "rope_append: %d query heads, %d pairs of a head of %d", r->q_heads, r->pairs,
                         c.head_dim);
    if (c.n_tokens == 0 || c.n_seqs == 0) return BYBYCU_OK;
    if (!r->q || !r->k || !r->v || !r->q_out || (!r->turns && r->pairs))
        return set_error(BYBYCU_ERR_ARGS, "rope_append: a slot is missing");
    const int esz = r->in_dtype == BYBYCU_DT_F32 ? 4 : 2;
    if (!kvc::aligned(r->q, esz) || !kvc::aligned(r->k, esz) || !kvc::aligned(r->v, esz) || !kvc::aligned(r->q_out, 2) ||
        !kvc::aligned(r->turns, 8) || !kvc::aligned(r->positions, 4))
        return set_error(BYBYCU_ERR_ARGS, "rope_append: misaligned slot");
    if (!kvc::strides_ok(r->q_token_stride, r->q_head_stride, r->q_heads, c.head_dim, 1) ||
        !kvc::strides_ok(r->k_token_stride, r->k_head_stride, c.kv_heads, c.head_dim, 1) ||
        !kvc::strides_ok(r->v_token_stride, r->v_head_stride, c.kv_heads, c.head_dim, 1) ||
        !kvc::out_strides_ok(r->out_token_stride, r->out_head_stride, c.n_tokens, r->q_heads, c.head_dim, 1))
        return set_error(BYBYCU_ERR_ARGS, "rope_append: negative or overlapping strides");
    const kvc::RopeParams p{r->q, r->k, r->v, static_cast<__nv_bfloat16*>(r->q_out),
                            r->q_token_stride, r->q_head_stride, r->k_token_stride, r->k_head_stride,
                            r->v_token_stride, r->v_head_stride, r->out_token_stride, r->out_head_stride,
                            r->turns, r->positions, r->q_heads, r->pairs, r->magnitude};
    // 16-byte accesses: whole vectors on either side of every split, and every vector aligned
    const int64_t in_all = r->q_token_stride | r->q_head_stride | r->k_token_stride | r->k_head_stride |
                           r->v_token_stride | r->v_head_stride;
    const bool vec = r->pairs % (r->interleaved ? 4 : 8) == 0 && (in_all * esz) % 16 == 0 &&
                     (r->out_token_stride | r->out_head_stride) % 8 == 0 && kvc::aligned(r->q, 16) &&
                     kvc::aligned(r->k, 16) && kvc::aligned(r->v, 16) && kvc::aligned(r->q_out, 16);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return r->in_dtype == BYBYCU_DT_F32 ? kvc::launch_rope<float>(c, p, r->interleaved != 0, vec, s)
                                        : kvc::launch_rope<__nv_bfloat16>(c, p, r->interleaved != 0, vec, s);
}

int bybycu_copy_pages(void* k, void* v, int n_layers, int64_t layer_stride, int64_t page_stride, int64_t page_bytes,
                      int n_pages, const int32_t* pairs, int n_pairs, void* stream) {
    if (n_layers <= 0 || n_layers > 65535 || n_pages <= 0 || page_bytes <= 0 || page_bytes % 16)
        return set_error(BYBYCU_ERR_SHAPE, "copy_pages: layers=%d pages=%d page bytes=%lld", n_layers, n_pages,
                         static_cast<long long>(page_bytes));
    if (n_pairs < 0 || (n_pairs && (!pairs || !k))) return set_error(BYBYCU_ERR_ARGS, "copy_pages: a slot is missing");
    if (layer_stride % 16 || page_stride % 16 || layer_stride < 0 || page_stride < page_bytes ||
        !kvc::aligned(k, 16) || !kvc::aligned(v, 16))
        return set_error(BYBYCU_ERR_ARGS, "copy_pages: pointers and strides must be multiples of 16 bytes, pages "
                                          "page_bytes apart at least");
    // bit 0: source of a pair, bit 1: destination of one
    std::vector<uint8_t> role;
    try {
        role.assign(static_cast<size_t>(n_pages), 0);
    } catch (const std::bad_alloc&) {
        return set_error(BYBYCU_ERR_RANGE, "copy_pages: no host memory for %d pages", n_pages);
    }
    for (int i = 0; i < n_pairs; ++i) {
        const int a = pairs[2 * i], b = pairs[2 * i + 1];
        if (a < 0 || a >= n_pages || b < 0 || b >= n_pages)
            return set_error(BYBYCU_ERR_RANGE, "copy_pages: pair %d (%d, %d) is outside the %d pages", i, a, b, n_pages);
        if (role[b] || (role[a] & 2) || a == b)
            return set_error(BYBYCU_ERR_ARGS, "copy_pages: page %d is the destination of one pair and in another", role[b] || a == b ? b : a);
        role[a] |= 1;
        role[b] |= 2;
    }
    const int64_t pieces = ceil_div(page_bytes, kvc::kCopyPiece);
    if (pieces > (1 << 20)) return set_error(BYBYCU_ERR_SHAPE, "copy_pages: pages of %lld bytes", static_cast<long long>(page_bytes));
    auto all = n_pairs <= kvc::kCopyFew ? kvc::copy_all<kvc::kCopyFew> : kvc::copy_all<kvc::kCopyPairs>;
    return all(k, v, n_layers, layer_stride, page_stride, page_bytes, static_cast<int>(pieces), pairs, n_pairs,
               static_cast<cudaStream_t>(stream));
}

}  // extern "C"
