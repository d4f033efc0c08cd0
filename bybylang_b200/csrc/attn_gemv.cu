// attn_gemv.cu - the GEMV route of paged attention: few query rows a kv head over a long cache.
//
// At one token and a group of G query heads the work is 4 G flop for every 4 bytes of K and V, so
// the cache's stream from HBM is all there is (6.5 TB/s; at G = 8 that is 52 TFLOP/s, above what
// fp32 FMAs with their conversions keep up with), and warp-level bf16 MMAs (m16n8k16) with the
// group's rows as M take it along.
//
//   * A CTA is WK key groups of WM warps; a warp holds 16 query rows, a group streams its own
//     chunks of KC = 16 WM keys through its own cp.async ring, so that no barrier joins the groups
//     until the end.  WM = 1 for up to 16 rows, 2 and 4 above (rows then share the chunk).
//   * Keys come through the page table, a 16-byte piece of a slot per copy; slots outside the
//     rows' common range and pages that do not exist are filled with zeros instead of read.
//   * Every warp keeps the running maximum and sum of its rows (online softmax); scores and
//     probabilities stay in registers: the accumulator layout of S is the A layout of P.
//   Measured: 64 sequences of up to 8192 keys, 32/8 heads of 128 (721 MB), 132 us with the joining
//     launch, 5.5 TB/s; one of 131071 keys, fp32 out (537 MB), 106 us, 5.1 TB/s.  DRAM runs at two
//     thirds of its cycles; eight warps an SM wait mostly on their own chains of dependent
//     instructions, and neither more CTAs nor deeper rings changed that.
//   * fp32 output: P enters as three bf16 terms (24 bits), so the product with V is exact to fp32
//     rounding.  bf16 output: one term, 2.3e-3 of the output's norm from the exact one; two terms
//     gave 1.7e-3, the output's own rounding, at 135 us for 132 and prompts of 700 tokens at 278
//     for 245.
//   * The cache axis is cut over the grid as well.  Up to 8 pieces are the CTAs of a cluster,
//     which cuts each sequence's own keys evenly and joins its sums through distributed shared
//     memory; more are splits of a fixed number of keys that leave unnormalised sums with their
//     maximum for a second, dependent launch.  Both join in a fixed order.
#include <algorithm>

#include "attention.cuh"

namespace bybycu {

static int scratch_pool(int device, cudaMemPool_t* pool);

namespace attn {

// What a split leaves for the joining kernel: row = (token * q_heads + head).
struct Partials {
    float* o;        // [splits][tokens * q_heads][head_dim]
    float2* ml;      // [splits][tokens * q_heads]: maximum (log2 units) and sum
    int64_t rows;
};

// The keys that a tile of `rows` rows (row r: token r / group, head r % group) can see, aligned
// down to the chunk grid, and how many splits of split_keys they take.
struct TileRange {
    int lo, hi, lo_aligned, splits;
};
__device__ __forceinline__ TileRange tile_range(const Params& p, const Seq& s, int first_row, int rows, int align,
                                                int split_keys) {
    TileRange r{0, 0, 0, 1};
    const int t0 = first_row / p.group, t1 = (first_row + rows - 1) / p.group;
    int lo0, hi0, lo1, hi1;
    row_range(p, s, s.first_pos + t0, &lo0, &hi0);
    row_range(p, s, s.first_pos + t1, &lo1, &hi1);
    // rows at negative positions see nothing and come first
    if (hi1 <= 0) return r;
    r.lo = hi0 > 0 ? lo0 : 0;
    r.hi = hi1;
    r.lo_aligned = r.lo / align * align;
    r.splits = r.hi > r.lo_aligned ? 1 + (r.hi - r.lo_aligned - 1) / split_keys : 1;
    return r;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Reads of the same shared-memory place in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes from src, or zeros.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
    const int n = real ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

template <int HD, int WM>
struct GemvCfg {
    static constexpr int kWarps = 4;
    static constexpr int kWK = kWarps / WM;
    static constexpr int kKC = 16 * WM;                          // keys of a chunk
    static constexpr int kPitch = HD * 2 + 16;                   // a row's bytes: 16 more keep ldmatrix free of conflicts
    static constexpr int kTensorBytes = kKC * kPitch;            // one chunk of K or of V
    static constexpr int kChunkBytes = 2 * kTensorBytes;
    // about 100 KB, so that two CTAs share an SM, but three chunks a group (two where three do not fit)
    static constexpr int kQBytes = HD > 128 ? 16 * WM * kPitch : 0;
    static constexpr int kFit = 104 * 1024 / (kWK * kChunkBytes);
    static constexpr int kLeast = 3 * kWK * kChunkBytes + kQBytes <= 227 * 1024 ? 3 : 2;
    static constexpr int kStages = kFit < kLeast ? kLeast : kFit > 8 ? 8 : kFit;
    static constexpr int kRingBytes = kWK * kStages * kChunkBytes;
    // the end: every warp's sums [16][HD] fp32, and in a cluster the CTA's [16 WM][HD], in the ring's place
    static constexpr int kCtaSums = kWarps * 16 * HD * 4;
    static constexpr int kJoinBytes = kCtaSums + 16 * WM * HD * 4;
    static constexpr int kSmem = (kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes) + kQBytes;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// P16: pages of whole 16-slot granules.  The address of a granule is then looked up once, 32
// granules at a time and a batch ahead, so that no copy waits for the page table.
template <int HD, int WM, bool F32, bool P16>
__global__ void __launch_bounds__(128) attention_gemv_kernel(const kvc::Cache c, const Params p, const Partials part,
                                                             int split_keys, int tile0, int row_tiles, int cluster) {
    using C = GemvCfg<HD, WM>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ float2 s_ml[16 * WM];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int wm = warp % WM, wk = warp / WM;
    const int kvh = blockIdx.y / row_tiles, first_row = (tile0 + blockIdx.y % row_tiles) * (16 * WM), b = blockIdx.z, split = blockIdx.x;
    const Seq s = load_seq(c, p, b);
    const int rows = min(16 * WM, s.rows * p.group - first_row);
    if (rows <= 0) return;   // every CTA of a cluster has the same rows
    TileRange range = tile_range(p, s, first_row, rows, 16, cluster ? INT32_MAX : split_keys);
    if (cluster) {   // this tile's own keys, evenly, in whole rounds of the CTA's chunks
        const int last = max(range.hi - range.lo_aligned, 1) - 1;
        split_keys = (last / cluster / 64 + 1) * 64;
        range.splits = last / split_keys + 1;
    }
    if (split >= range.splits && !cluster) return;
    // a CTA of a cluster without keys has an empty segment
    const int seg_lo = split < range.splits ? range.lo_aligned + split * split_keys : range.hi;
    const int seg_hi = seg_lo + min(range.hi - seg_lo, split_keys);
    const int D = c.head_dim;

    // this thread's two rows of its warp's sixteen
    int row_lo[2], row_hi[2], row_pos[2];
    float slope[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = wm * 16 + g + 8 * i;
        row_pos[i] = s.first_pos + (first_row + r) / p.group;
        row_lo[i] = row_hi[i] = 0;
        slope[i] = 0.0f;
        if (r < rows) {
            row_range(p, s, row_pos[i], &row_lo[i], &row_hi[i]);
            if (p.slopes) slope[i] = p.slopes[kvh * p.group + (first_row + r) % p.group] * kLog2e;
        }
    }
    // the plain form takes the maximum of unscaled scores: a scale above 0 only
    const bool mod = p.cap > 0.0f || p.slopes || !(p.scale_log2 > 0.0f);
    const float unit = mod ? 1.0f : p.scale_log2;
    // keys that every row of the warp sees need no mask
    int all_lo = max(row_lo[0], row_lo[1]), all_hi = min(row_hi[0], row_hi[1]);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        all_lo = max(all_lo, __shfl_xor_sync(~0u, all_lo, o));
        all_hi = min(all_hi, __shfl_xor_sync(~0u, all_hi, o));
    }

    // Q as A fragments: registers up to 128 dimensions, shared memory above
    constexpr int kSteps = HD / 16;
    uint32_t qf[HD > 128 ? 1 : kSteps][4];
    const uint32_t ring = smem_u32(smem), qs = ring + (C::kSmem - C::kQBytes);
    if constexpr (HD > 128) {
        for (int i = threadIdx.x; i < 16 * WM * (HD / 8); i += 128) {
            const int r = i / (HD / 8), d = i % (HD / 8) * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < rows && d < D)
                v = *reinterpret_cast<const uint4*>(p.q + (s.q0 + (first_row + r) / p.group) * p.q_token +
                                                    (kvh * p.group + (first_row + r) % p.group) * p.q_head + d);
            *reinterpret_cast<uint4*>(smem + (C::kSmem - C::kQBytes) + r * C::kPitch + d * 2) = v;
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = wm * 16 + g + 8 * i;
            const __nv_bfloat16* q = p.q + (s.q0 + (first_row + r) / p.group) * p.q_token +
                                     (kvh * p.group + (first_row + r) % p.group) * p.q_head;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = k * 16 + e * 8 + t4 * 2;
                    qf[k][e * 2 + i] = r < rows && d < D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                }
        }
    }

    // the group's chunks: wk, wk + WK, ... of the segment
    const int n_all = seg_hi > seg_lo ? (seg_hi - seg_lo + C::kKC - 1) / C::kKC : 0;
    const int n_mine = n_all > wk ? (n_all - wk + C::kWK - 1) / C::kWK : 0;
    const uint32_t my_ring = ring + wk * C::kStages * C::kChunkBytes;
    const int gt = wm * 32 + lane;   // thread of the group
    const int32_t* table = c.page_table + b * c.table_stride;
    const int64_t head_off = static_cast<int64_t>(kvh) * c.head_stride;
    // One slot row is HD / 8 pieces of 16 bytes; a thread copies the same piece of every
    // (32 WM / pieces)-th slot.
    constexpr int kPieces = HD / 8, kRowStep = 32 * WM / kPieces;
    static_assert(kRowStep >= 1 && 16 % kRowStep == 0, "copy layout");
    const int piece = gt % kPieces, row0 = gt / kPieces;
    const bool piece_real = piece * 8 < D;
    // The copies of chunk i into its ring slot, one commit group.  Chunks are fetched in order.
    constexpr int kBatch = 32 / WM;   // chunks whose granules' pages one batch of lanes looks up
    int batch_id = -1, next_id = -1;
    auto granule_key = [&](int batch) {   // the first key of this lane's granule of a batch
        return seg_lo + (wk + (batch * kBatch + lane / WM) * C::kWK) * C::kKC + lane % WM * 16;
    };
    auto look_up = [&](int batch) {
        const int j = granule_key(batch);
        return j < seg_hi && j + 16 > range.lo ? table[j / c.page_size] : 0;
    };
    if constexpr (P16) {
        if (n_mine > 0) next_id = look_up(0);
    }
    int64_t granule = -1;   // this lane's granule: element offset of its first slot, -1 without one
    // dense slots of the kernel's own head dimension: every copy's address is one base and a constant
    const bool dense = P16 && D == HD && c.token_stride == HD;
    const int64_t mine_off = head_off + row0 * c.token_stride + piece * 8;
    const uint32_t mine_dst = my_ring + row0 * C::kPitch + piece * 16;
    int fetch_stage = 0;
    auto fetch = [&](int i) {
        if (i < n_mine) {
            const int j0 = seg_lo + (wk + i * C::kWK) * C::kKC;
            const uint32_t dst = mine_dst + fetch_stage * C::kChunkBytes;
            fetch_stage = fetch_stage + 1 == C::kStages ? 0 : fetch_stage + 1;
            if constexpr (P16) {
                if (i % kBatch == 0) {
                    batch_id = next_id;
                    const int j = granule_key(i / kBatch);
                    const bool in = j < seg_hi && j + 16 > range.lo;
                    if (batch_id < 0 || batch_id >= c.n_pages) {
                        if (in) record_device_error(kDevErrPage);
                        batch_id = -1;
                    }
                    granule = in && batch_id >= 0 ? batch_id * c.page_stride + j % c.page_size * c.token_stride : -1;
                    if (i + kBatch < n_mine) next_id = look_up(i / kBatch + 1);
                }
                int64_t at[WM];
#pragma unroll
                for (int w = 0; w < WM; ++w) at[w] = __shfl_sync(~0u, granule, i % kBatch * WM + w);
                const bool whole = j0 >= range.lo && j0 + C::kKC <= seg_hi;
                bool pages = true;
#pragma unroll
                for (int w = 0; w < WM; ++w) pages = pages && at[w] >= 0;
                if (dense && whole && pages) {
#pragma unroll
                    for (int w = 0; w < WM; ++w) {
                        const __nv_bfloat16 *kp = c.k + (at[w] + mine_off), *vp = c.v + (at[w] + mine_off);
#pragma unroll
                        for (int r = 0; r < 16 / kRowStep; ++r) {
                            const uint32_t to = dst + (w * 16 + r * kRowStep) * C::kPitch;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(kp + r * kRowStep * HD) : "memory");
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + C::kTensorBytes), "l"(vp + r * kRowStep * HD) : "memory");
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    return;
                }
#pragma unroll
                for (int r = 0; r < C::kKC / kRowStep; ++r) {
                    const int j = row0 + r * kRowStep;   // its granule is r * kRowStep / 16: kRowStep divides 16
                    const int64_t base = at[r * kRowStep / 16];
                    const bool real = base >= 0 && piece_real && (whole || (j0 + j >= range.lo && j0 + j < seg_hi));
                    const int64_t off = real ? base + j % 16 * c.token_stride + head_off + piece * 8 : 0;
                    cp_async16_or_zero(dst + r * kRowStep * C::kPitch, c.k + off, real);
                    cp_async16_or_zero(dst + C::kTensorBytes + r * kRowStep * C::kPitch, c.v + off, real);
                }
            } else {
                int pg_have = -1, id = -1;
#pragma unroll
                for (int r = 0; r < C::kKC / kRowStep; ++r) {
                    const int j = j0 + row0 + r * kRowStep;
                    const bool in = j >= range.lo && j < seg_hi;
                    const int pg = in ? j / c.page_size : -1;
                    if (in && pg != pg_have) {
                        id = table[pg];
                        pg_have = pg;
                        if (id < 0 || id >= c.n_pages) {
                            record_device_error(kDevErrPage);
                            id = -1;
                        }
                    }
                    const bool real = in && id >= 0 && piece_real;
                    const int64_t off = real ? id * c.page_stride + (j - pg * c.page_size) * c.token_stride + head_off + piece * 8 : 0;
                    cp_async16_or_zero(dst + r * kRowStep * C::kPitch, c.k + off, real);
                    cp_async16_or_zero(dst + C::kTensorBytes + r * kRowStep * C::kPitch, c.v + off, real);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto group_sync = [&]() {
        if constexpr (WM == 1) __syncwarp();
        else named_barrier(1 + wk, 32 * WM);
    };

    float o[HD / 8][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) fetch(i);
    int stage = 0;
    for (int i = 0; i < n_mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
        group_sync();   // the chunk is whole, and the slot that the next fetch fills is free
        fetch(i + C::kStages - 1);
        const int j0 = seg_lo + (wk + i * C::kWK) * C::kKC;
        const uint32_t kc = my_ring + stage * C::kChunkBytes, vc = kc + C::kTensorBytes;
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        float sc[C::kKC / 8][4] = {};
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            uint32_t a[4];
            if constexpr (HD > 128) ldsm4(qs + (wm * 16 + (lane & 15)) * C::kPitch + k * 32 + (lane >> 4) * 16, a);
            else { a[0] = qf[k][0]; a[1] = qf[k][1]; a[2] = qf[k][2]; a[3] = qf[k][3]; }
#pragma unroll
            for (int n = 0; n < C::kKC / 16; ++n) {
                uint32_t kf[4];
                ldsm4(kc + (n * 16 + (lane >> 4) * 8 + (lane & 7)) * C::kPitch + k * 32 + ((lane >> 3) & 1) * 16, kf);
                mma_bf16(sc[2 * n], a, kf[0], kf[1]);
                mma_bf16(sc[2 * n + 1], a, kf[2], kf[3]);
            }
        }
        const bool masked = j0 < all_lo || j0 + C::kKC > all_hi;
        if (mod) {
#pragma unroll
            for (int n = 0; n < C::kKC / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[n][e] = score_log2<true, F32>(p, sc[n][e], slope[e >> 1], row_pos[e >> 1] - (j0 + n * 8 + t4 * 2 + (e & 1)));
        }
        if (masked) {
#pragma unroll
            for (int n = 0; n < C::kKC / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + n * 8 + t4 * 2 + (e & 1);
                    if (j < row_lo[e >> 1] || j >= row_hi[e >> 1]) sc[n][e] = -INFINITY;
                }
        }
        float mn[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < C::kKC / 8; ++n) {
            mn[0] = fmaxf(mn[0], fmaxf(sc[n][0], sc[n][1]));
            mn[1] = fmaxf(mn[1], fmaxf(sc[n][2], sc[n][3]));
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mn[r] = fmaxf(mn[r], __shfl_xor_sync(~0u, mn[r], 1));
            mn[r] = fmaxf(mn[r], __shfl_xor_sync(~0u, mn[r], 2));
            mn[r] = fmaxf(m[r], mn[r] * unit);
        }
        // The sums follow a new maximum only when one grew by more than 2^8 (probabilities are then
        // below 2^8 with the same relative rounding): hardly ever after the first chunks.
        if (__any_sync(~0u, mn[0] > m[0] + 8.0f || mn[1] > m[1] + 8.0f)) {
            float keep[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                keep[r] = mn[r] == -INFINITY ? 1.0f : ex2(m[r] - mn[r]);
                l[r] *= keep[r];
                m[r] = mn[r];
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                o[n][0] *= keep[0];
                o[n][1] *= keep[0];
                o[n][2] *= keep[1];
                o[n][3] *= keep[1];
            }
        }
        const float off[2] = {m[0] == -INFINITY ? 0.0f : -m[0], m[1] == -INFINITY ? 0.0f : -m[1]};
#pragma unroll
        for (int n = 0; n < C::kKC / 8; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = ex2(fmaf(sc[n][e], unit, off[e >> 1]));
            l[0] += sc[n][0] + sc[n][1];
            l[1] += sc[n][2] + sc[n][3];
        }
#pragma unroll
        for (int n = 0; n < C::kKC / 16; ++n) {
            constexpr int kTerms = F32 ? 3 : 1;
            uint32_t pf[kTerms][4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {   // a0 a1: keys 0-7 (rows g, g + 8); a2 a3: keys 8-15
                float x = sc[2 * n + (f >> 1)][(f & 1) * 2], y = sc[2 * n + (f >> 1)][(f & 1) * 2 + 1];
#pragma unroll
                for (int w = 0; w < kTerms; ++w) {
                    pf[w][f] = pack_bf16(x, y);
                    x -= bf16_lo(pf[w][f]);
                    y -= bf16_hi(pf[w][f]);
                }
            }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t vf[4];
                ldsm4_t(vc + (n * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * C::kPitch + d * 32 + (lane >> 4) * 16, vf);
if constexpr (F32) {
                    // The tensor core truncates as it accumulates: over thousands of keys that is
                    // a bias of several 2^-22, so a chunk's product is summed apart, its smallest
                    // term first, and added with a rounding.
                    float x[4] = {}, y[4] = {};
#pragma unroll
                    for (int w = kTerms - 1; w >= 0; --w) {
                        mma_bf16(x, pf[w], vf[0], vf[1]);
                        mma_bf16(y, pf[w], vf[2], vf[3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[2 * d][e] += x[e];
                        o[2 * d + 1][e] += y[e];
                    }
                } else {
                    mma_bf16(o[2 * d], pf[0], vf[0], vf[1]);
                    mma_bf16(o[2 * d + 1], pf[0], vf[2], vf[3]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(~0u, l[r], 1);
        l[r] += __shfl_xor_sync(~0u, l[r], 2);
    }
    // join the key groups: every warp's sums into shared memory, in the ring's place
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);   // [warp][16][HD]
    if (t4 == 0) {
        s_m[warp][g] = m[0]; s_m[warp][g + 8] = m[1];
        s_l[warp][g] = l[0]; s_l[warp][g + 8] = l[1];
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
        *reinterpret_cast<float2*>(so + (warp * 16 + g) * HD + n * 8 + t4 * 2) = make_float2(o[n][0], o[n][1]);
        *reinterpret_cast<float2*>(so + (warp * 16 + g + 8) * HD + n * 8 + t4 * 2) = make_float2(o[n][2], o[n][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (HD / 4); i += 128) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4, w0 = r / 16, rr = r % 16;
        if (d >= D) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < C::kWK; ++k) mx = fmaxf(mx, s_m[k * WM + w0][rr]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < C::kWK; ++k) {
            const int w = k * WM + w0;
            const float f = ex2(s_m[w][rr] - base);
            const float4 v = *reinterpret_cast<const float4*>(so + (w * 16 + rr) * HD + d);
            sum = fmaf(f, s_l[w][rr], sum);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
        }
        if (cluster) {
            *reinterpret_cast<float4*>(smem + C::kCtaSums + (r * HD + d) * 4) = acc;
            if (d == 0) s_ml[r] = make_float2(mx, sum);
            continue;
        }
        const int64_t token = s.q0 + (first_row + r) / p.group, head = kvh * p.group + (first_row + r) % p.group;
        if (range.splits > 1) {
            const int64_t at = split * part.rows + token * p.q_heads + head;
            *reinterpret_cast<float4*>(part.o + at * D + d) = acc;
            if (d == 0) part.ml[at] = make_float2(mx, sum);
            continue;
        }
        store_row4<F32>(p, token, head, d, acc, sum);
    }
    if (!cluster) return;
    cluster_barrier();
    for (int i = split * 128 + threadIdx.x; i < rows * (HD / 4); i += cluster * 128) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        if (d >= D) continue;
        float mx = -INFINITY;
        for (int k = 0; k < range.splits; ++k) mx = fmaxf(mx, cluster_load2(cluster_addr(&s_ml[r], k)).x);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < range.splits; ++k) {
            const float2 ml = cluster_load2(cluster_addr(&s_ml[r], k));
            const float4 v = cluster_load4(cluster_addr(smem + C::kCtaSums + (r * HD + d) * 4, k));
            const float f = ex2(ml.x - base);
            sum = fmaf(f, ml.y, sum);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
        }
        store_row4<F32>(p, s.q0 + (first_row + r) / p.group, kvh * p.group + (first_row + r) % p.group, d, acc, sum);
    }
    cluster_barrier();   // no CTA leaves while another may read its sums
}

// Joins the splits of a row (token, head): WARPS warps of a block take equal runs of them, and are
// added in order.  Four warps for many splits and few rows (a warp alone took 22 us for 37), one a
// row for many rows.
template <bool F32, int WARPS>
__global__ void __launch_bounds__(128) attention_join_kernel(const kvc::Cache c, const Params p, const Partials part,
                                                             int split_keys, int tile_rows, int align) {
    __shared__ float s_sum[4];
    __shared__ float4 s_acc[3][kvc::kMaxHeadDim / 4];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / WARPS) + warp / WARPS;
    if (row >= part.rows) return;
    const int t = static_cast<int>(row / p.q_heads), h = static_cast<int>(row % p.q_heads), D = c.head_dim;
    int b = 0;
    for (int i = 0; i < c.n_seqs; i += 32) b += __popc(__ballot_sync(~0u, i + lane < c.n_seqs && c.q_start[i + lane + 1] <= t));
    if (b >= c.n_seqs || t < c.q_start[0]) return;
    const Seq s = load_seq(c, p, b);
    if (t - s.q0 >= s.rows) return;
    // the tile that the row was in: key range and splits as that kernel had them
    const int first_row = ((t - s.q0) * p.group + h % p.group) / tile_rows * tile_rows;
    const TileRange range = tile_range(p, s, first_row, min(tile_rows, s.rows * p.group - first_row), align, split_keys);
    if (range.splits == 1) return;   // written by the first kernel
    float mx = -INFINITY;
    for (int k = lane; k < range.splits; k += 32) mx = fmaxf(mx, part.ml[k * part.rows + row].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
    const float base = mx == -INFINITY ? 0.0f : mx;
    const int per = (range.splits + WARPS - 1) / WARPS, k0 = warp % WARPS * per, k1 = min(range.splits, k0 + per);
    for (int d0 = 0; d0 < D; d0 += 128) {
        const int d = d0 + lane * 4;
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (d < D) {
#pragma unroll 4
            for (int k = k0; k < k1; ++k) {
                const float2 ml = part.ml[k * part.rows + row];
                const float4 v = *reinterpret_cast<const float4*>(part.o + (k * part.rows + row) * D + d);
                const float f = exp2f(ml.x - base);
                sum = fmaf(f, ml.y, sum);
                acc.x = fmaf(f, v.x, acc.x);
                acc.y = fmaf(f, v.y, acc.y);
                acc.z = fmaf(f, v.z, acc.z);
                acc.w = fmaf(f, v.w, acc.w);
            }
        }
        if constexpr (WARPS == 4) {   // the whole block has one row
            if (warp && d < D) s_acc[warp - 1][d / 4] = acc;
            if (lane == 0) s_sum[warp] = sum;
            __syncthreads();
            if (warp == 0 && d < D) {
                for (int w = 0; w < 3; ++w) {
                    const float4 v = s_acc[w][d / 4];
                    acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
                }
                store_row4<F32>(p, t, h, d, acc, s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);
            }
            __syncthreads();
        } else if (d < D) {
            store_row4<F32>(p, t, h, d, acc, sum);
        }
    }
}

// The launch of a route's kernel and, where the grid splits the cache, of the joining one.
static cudaLaunchConfig_t pdl_config(dim3 grid, int threads, size_t smem, cudaStream_t stream, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

static int launch_join(const kvc::Cache& c, const Params& p, const Partials& part, int split_keys, int tile_rows,
                       int align, bool f32, cudaStream_t stream) {
    const bool wide = part.rows <= 4096;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(wide ? part.rows : ceil_div(part.rows, 4))), 128, 0, stream, attr);
    auto kern = wide ? (f32 ? attention_join_kernel<true, 4> : attention_join_kernel<false, 4>)
                     : (f32 ? attention_join_kernel<true, 1> : attention_join_kernel<false, 1>);
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, c, p, part, split_keys, tile_rows, align));
    return BYBYCU_OK;
}

// Scratch of a split launch, stream-ordered.
struct SplitScratchMem {
    void* ptr = nullptr;
    cudaStream_t stream = nullptr;
    int take(int device, int64_t rows, int splits, int dim, cudaStream_t s, Partials* part) {
        cudaMemPool_t pool = nullptr;
        if (int rc = scratch_pool(device, &pool)) return rc;
        const size_t o_bytes = static_cast<size_t>(rows) * splits * dim * 4;
        BYBYCU_CUDA_TRY(cudaMallocFromPoolAsync(&ptr, o_bytes + static_cast<size_t>(rows) * splits * 8, pool, s));
        stream = s;
        part->o = static_cast<float*>(ptr);
        part->ml = reinterpret_cast<float2*>(static_cast<char*>(ptr) + o_bytes);
        part->rows = rows;
        return BYBYCU_OK;
    }
    ~SplitScratchMem() {
        if (ptr) cudaFreeAsync(ptr, stream);
    }
};

// The longest stretch of keys that one row tile can visit.
static int64_t longest_span(const Params& p, int tile_rows) {
    int64_t span = p.max_kv;
    if (p.window > 0 && !p.prefix) span = std::min<int64_t>(span, static_cast<int64_t>(p.window) + ceil_div(tile_rows, p.group) + 16);
    return std::max<int64_t>(span, 1);
}

template <int HD, int WM, bool F32, bool P16>
static int launch_gemv_tile(const kvc::Cache& c, const Params& p, const DeviceInfo& info, cudaStream_t stream) {
    using C = GemvCfg<HD, WM>;
    auto kern = attention_gemv_kernel<HD, WM, F32, P16>;
    static std::once_flag once[64];
    static cudaError_t prep[64];
    if (info.device < 0 || info.device >= 64) return set_error(BYBYCU_ERR_ARGS, "device %d out of range", info.device);
    std::call_once(once[info.device], [&] {
        prep[info.device] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    });
    if (prep[info.device] != cudaSuccess) return cuda_fail(prep[info.device], "attention_gemv_kernel shared memory");
    const int row_tiles = static_cast<int>(ceil_div(static_cast<int64_t>(p.max_q) * p.group, 16 * WM));
    // a launch's grid has 65535 rows and layers at most
    constexpr int kGrid = 65535;
    if (c.kv_heads > kGrid) return set_error(BYBYCU_ERR_SHAPE, "paged_attention: %d kv heads", c.kv_heads);
    const int64_t units = static_cast<int64_t>(row_tiles) * c.kv_heads * c.n_seqs;
    const int slots = info.sm_count * std::max(1, std::min(3, static_cast<int>(227 * 1024 / (C::kSmem + 2048))));
    const int64_t span = longest_span(p, 16 * WM);
    // One sequence: as many pieces as fill the card once.  More: their lengths may differ up to the
    // longest, so pieces of a sixth of a CTA's share of half of the most there can be, whatever the
    // lengths, keep the tail short.  128 keys at least (two rounds of a CTA's chunks).
    const int64_t share = std::max<int64_t>(c.n_seqs == 1 ? ceil_div(span * units, slots) : ceil_div(span * units, 12 * slots), 128);
    const int64_t pieces = ceil_div(span, share);
    // A cluster where one wave holds them all: with more work than that its CTAs, which end
    // together, keep SM slots from others (64 sequences of up to 8192: 216 us against 142).
    const int fit = pieces == 1 || pieces > 12 ? 0 : pieces == 2 ? 2 : pieces <= 4 ? 4 : 8;
    const int cluster = units * fit <= slots ? fit : 0;
    // splits of the second kernel: 256 keys at least, below a split's own sums weigh
    const int split_keys = static_cast<int>(std::min<int64_t>(std::max<int64_t>(ceil_div(share, 64) * 64, 256), INT32_MAX / 2 / 64 * 64));
    const int splits = cluster ? cluster : pieces == 1 ? 1 : static_cast<int>(ceil_div(span + 16, split_keys));
    Partials part{};
    SplitScratchMem scratch;
    if (splits > 1 && !cluster)
        if (int rc = scratch.take(info.device, static_cast<int64_t>(c.n_tokens) * p.q_heads, splits, c.head_dim, stream, &part)) return rc;
    cudaLaunchAttribute attr[2];
    const int tiles_step = std::min(row_tiles, kGrid / c.kv_heads);
    for (int64_t seq0 = 0; seq0 < c.n_seqs; seq0 += kGrid) {
        kvc::Cache cc = c;   // the sequences from seq0 on
        Params pp = p;
        cc.page_table += seq0 * c.table_stride;
        cc.q_start += seq0;
        cc.kv_lens += seq0;
        if (pp.prefix) pp.prefix += seq0;
        for (int tile0 = 0; tile0 < row_tiles; tile0 += tiles_step) {
            const int tiles = std::min(tiles_step, row_tiles - tile0);
            cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(splits), static_cast<unsigned>(tiles * c.kv_heads),
                                                     static_cast<unsigned>(std::min<int64_t>(kGrid, c.n_seqs - seq0))), 128, C::kSmem, stream, attr);
            if (cluster) {
                attr[1].id = cudaLaunchAttributeClusterDimension;
                attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
                attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
                cfg.numAttrs = 2;
            }
            BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, cc, pp, part, splits == 1 ? INT32_MAX : split_keys, tile0, tiles, cluster));
        }
    }
    return splits > 1 && !cluster ? launch_join(c, p, part, split_keys, 16 * WM, 16, F32, stream) : BYBYCU_OK;
}

template <int HD, bool F32>
static int launch_gemv_rows(const kvc::Cache& c, const Params& p, const DeviceInfo& info, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.max_q) * p.group;
    const bool p16 = c.page_size % 16 == 0;
    if (rows <= 16) return p16 ? launch_gemv_tile<HD, 1, F32, true>(c, p, info, stream) : launch_gemv_tile<HD, 1, F32, false>(c, p, info, stream);
    if (rows <= 32) return p16 ? launch_gemv_tile<HD, 2, F32, true>(c, p, info, stream) : launch_gemv_tile<HD, 2, F32, false>(c, p, info, stream);
    return p16 ? launch_gemv_tile<HD, 4, F32, true>(c, p, info, stream) : launch_gemv_tile<HD, 4, F32, false>(c, p, info, stream);
}

static int launch_gemv(const kvc::Cache& c, const Params& p, bool f32, cudaStream_t stream) {
    if (p.max_q == 0) return BYBYCU_OK;
    DeviceInfo info;
    if (int rc = current_device_info(&info)) return rc;
    if (c.head_dim <= 64) return f32 ? launch_gemv_rows<64, true>(c, p, info, stream) : launch_gemv_rows<64, false>(c, p, info, stream);
    if (c.head_dim <= 128) return f32 ? launch_gemv_rows<128, true>(c, p, info, stream) : launch_gemv_rows<128, false>(c, p, info, stream);
    return f32 ? launch_gemv_rows<256, true>(c, p, info, stream) : launch_gemv_rows<256, false>(c, p, info, stream);
}

}  // namespace attn
}  // namespace bybycu
