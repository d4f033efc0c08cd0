// attn_tc.cu - the TC route of paged attention: many query rows a kv head, on the
// 5th-generation tensor cores.
//
// A CTA (one per SM) takes two tiles of up to 128 query rows of one kv head - row r is token
// r / G, head r % G, so the G heads of a group share every key they read - and walks the keys in
// blocks of 128:
//   warps 0-7, 8-15  one softmax group per query tile: two threads a row, 64 keys each
//   warp 16          brings Q and the K and V blocks in by TMA, page by page through the table
//   warp 17          issues the MMAs: S = Q K^T (both from shared memory) into tensor memory,
//                    O += P V with P from tensor memory (bf16, over the scores it came from)
//                    and V as it lies in its pages (N-major)
// While the tensor core works on one tile's O += P V and next S, the other tile's group is at its
// exponentials: at 128 dimensions a block's two products take the tensor core about as long
// (2 * 128^3 multiplies at 4096 a cycle) as its 128^2 exponentials take the SM's special-function
// units (16 a cycle), so neither may wait for the other.
//   Measured: 2 sequences of 4096 tokens, 32 heads of 128, 281 us (980 TFLOP/s) alone, 323 us where
// call follows call and the clocks give way; with 8 kv heads 274 us; heads of 64 at half of that
// rate (the exponentials are the same).  A pair of blocks takes
// some 3300 cycles where its MMAs alone are 2048: a tile's softmax (1700, issue and latency of four
// warps on a scheduler) and its own P V and S (1350) follow one another, and only the other tile's
// run beside them.
//
//   * The running maximum is only followed when it grew by more than 2^8: probabilities then stay
//     below 2^8, with the same relative rounding in bf16 and sums in fp32, and the accumulators in
//     tensor memory are hardly ever rescaled.
//   * Products of a tile past its rows' last visible key are skipped; within the last and first
//     blocks the P V product runs over the 16-key steps that hold a visible key, and V rows of
//     these steps outside the common range are zeroed in shared memory (0 * NaN would be NaN).
//   * bf16 output only: the tensor core truncates when it accumulates, and over thousands of keys
//     that costs an fp32 output two digits.
//   * Fewer bits than fp32, for a bf16 output: probabilities in bf16 (16 bits would take half as much
//     tensor work again), the cubic of ex2_fma, the truncation, a cap up to 256 in its
//     plain form.  2.0e-3 of the output's norm together, of which its own rounding is 1.7e-3.
//
// Every wait is bounded: on a timeout the kernel records the error, drains its copies and MMAs,
// frees its tensor memory and returns.
#include <algorithm>
#include <type_traits>

#include "attention.cuh"

namespace bybycu {
namespace attn {
namespace tcore {

constexpr int kThreads = 576;   // 18 warps, five on a quarter of the SM: 96 registers a thread
constexpr int kLoadWarp = 16, kMmaWarp = 17;
constexpr int kHalf = 64;       // keys of a softmax thread
constexpr int kFma = 3;         // of 16 exponentials that the FMA units take over: 0, 2, 4, 5, 7 of 16
                                // measured 267, 265, 266, 267, 272 us (2 x 4096 tokens, 32/8 heads of 128)
constexpr int kRows = 128;      // query rows of a tile (MMA M)
constexpr int kKeys = 128;      // keys of a block
constexpr uint32_t kTmemCols = 512;

template <int HD>
struct Cfg {
    static constexpr int kHalves = HD / 64;                              // 128-byte swizzled boxes a row
    static constexpr uint32_t kQTile = kRows * HD * 2;
    static constexpr uint32_t kBlock = kKeys * HD * 2;                   // one K or V block
    static constexpr int kStages = HD == 128 ? 5 : 8;
    static constexpr uint32_t kOffRing = 2 * kQTile;
    static constexpr uint32_t kOffBar = kOffRing + kStages * kBlock;
    // barriers: q; full, empty [stages]; s_full, p_half, p_full [2]; done
    static constexpr uint32_t kNumBars = 1 + 2 * kStages + 6 + 1;
    static constexpr uint32_t kOffSlot = kOffBar + kNumBars * 8;
    static constexpr uint32_t kOffRow = kOffSlot + 8;                    // a float per query row
    static constexpr uint32_t kSmem = kOffRow + 2 * kRows * 4 + 1024;    // + alignment slack
    static_assert(kSmem <= 227 * 1024 && kSmem > 114 * 1024, "one CTA per SM");
    // instruction descriptors of kind::f16: D fp32, A and B bf16, M = 128
    static constexpr uint32_t kBase = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kRows >> 4) << 24);
    static constexpr uint32_t kIdescS = kBase | (uint32_t(kKeys >> 3) << 17);               // K: keys x dims, K-major
    static constexpr uint32_t kIdescO = kBase | (1u << 16) | (uint32_t(HD >> 3) << 17);     // V: N-major
    // tensor memory: S0 S1 (P over them) O0 O1
    static constexpr uint32_t kTmemO = 2 * kKeys;
};

struct Maps {
    CUtensorMap q;   // bf16 (dim, head, token), box 64 x group x tokens of a tile
    CUtensorMap k;   // bf16 (dim, slot, kv head, page), box 64 x slots x 1 x 1
    CUtensorMap v;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}

// The MMA warp stays converged; elect.sync picks the lane that issues.  Four products at a time
// (an instruction of its own to elect for each would cost as much as the issue).
__device__ __forceinline__ void mma_ss4(uint32_t d, const uint64_t (&a)[4], const uint64_t (&b)[4], uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred e, p, q;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %2, 0;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %3, %7, %1, p;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %4, %8, %1, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %9, %1, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %6, %10, %1, q;\n\t}"
                 ::"r"(d), "r"(idesc), "r"(accumulate), "l"(a[0]), "l"(a[1]), "l"(a[2]), "l"(a[3]), "l"(b[0]), "l"(b[1]), "l"(b[2]), "l"(b[3])
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Probabilities lie over the scores they came from, each half of 64 keys over its own columns:
// 16-key step st at column p_column(st).
__device__ __forceinline__ uint32_t p_column(int st) { return (st >> 2) * kHalf + (st & 3) * 8; }
// The same from tensor memory: four 16-key steps from `a` and `b` (2048 bytes of V a step).
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred e, p, q;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %2, 0;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%3], %7, %1, p;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%4], %8, %1, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%5], %9, %1, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%6], %10, %1, q;\n\t}"
                 ::"r"(d), "r"(idesc), "r"(accumulate), "r"(a), "r"(a + 8), "r"(a + 16), "r"(a + 24), "l"(b), "l"(b + 128), "l"(b + 256),
                 "l"(b + 384)
                 : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait that also ends when another warp of the CTA has given up (without reading its
// flag where the phase is complete already: a shared-memory read costs the chain of waits some
// 100 cycles while the tensor core streams its operands).
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t err) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            record_device_error(err);
            *abort = 1;
            return false;
        }
    }
}

// Whether any thread of a pair of warps says so; their barrier.
__device__ __forceinline__ bool pair_any(uint32_t id, bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"(static_cast<uint32_t>(mine)), "r"(id) : "memory");
    return any != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 2^x of two numbers below 128 on the FMA units: x = n + f with n the nearest whole number (the
// low bits of x + 1.5 * 2^23), 2^f by the cubic of least relative error on [-1/2, 1/2] (7.5e-5, by
// Remez exchange; a bf16 probability is rounded by up to 3.9e-3 after it), n added to the exponent.
// Below 2^-125 it stays there: masked scores, whose 2^x has to be 0, do not come here.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
    const float magic = 12582912.0f;
    x.x = fmaxf(x.x, -125.0f);
    x.y = fmaxf(x.y, -125.0f);
    const float2 t = add2(x, make_float2(magic, magic));
    const float2 n = add2(t, make_float2(-magic, -magic));
    const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
    float2 y = fma2(f, make_float2(0.0551716685f, 0.0551716685f), make_float2(0.242611125f, 0.242611125f));
    y = fma2(y, f, make_float2(0.693260968f, 0.693260968f));
    y = fma2(y, f, make_float2(0.999928057f, 0.999928057f));
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}

template <int HD, bool MOD>
__global__ void __launch_bounds__(kThreads, 1) attention_tc_kernel(const __grid_constant__ Maps maps, const kvc::Cache c,
                                                                   const Params p, const Partials part, int split_keys, int splits,
                                                                   int tiles, int band, int tile_rows, int box_slots) {
    using C = Cfg<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Order of the grid: bands of (sequence, kv head, split) whose keys and values fit into L2
    // together; within a band the late tiles, which see the most keys, come first.
    const int64_t units = static_cast<int64_t>(c.n_seqs) * c.kv_heads * splits;
    const int64_t first_unit = blockIdx.x / (static_cast<int64_t>(band) * tiles) * band;
    const int in_band = static_cast<int>(units - first_unit < band ? units - first_unit : band);
    const int at = static_cast<int>(blockIdx.x - first_unit * tiles);
    const int64_t unit_id = first_unit + at % in_band;
    const int split = static_cast<int>(unit_id % splits), kvh = static_cast<int>(unit_id / splits % c.kv_heads);
    const int b = static_cast<int>(unit_id / splits / c.kv_heads);
    const int first_row = (tiles - 1 - at / in_band) * 2 * tile_rows;
    const Seq s = load_seq(c, p, b);
    const int rows = min(2 * tile_rows, s.rows * p.group - first_row);
    if (rows <= 0) return;
    const TileRange range = tile_range(p, s, first_row, rows, kKeys, split_keys);
    if (split >= range.splits) return;
    const int seg_lo = range.lo_aligned + split * split_keys;
    const int seg_hi = seg_lo + min(range.hi - seg_lo, split_keys);
    // key blocks of each query tile in this segment (none for a tile without rows)
    int n_blocks[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int left = min(tile_rows, rows - i * tile_rows);
        n_blocks[i] = 0;
        if (left > 0) {
            const TileRange mine = tile_range(p, s, first_row + i * tile_rows, left, kKeys, split_keys);
            n_blocks[i] = max(0, (min(mine.hi, seg_hi) - seg_lo + kKeys - 1) / kKeys);
        }
    }
    const int n_all = max(n_blocks[0], n_blocks[1]);

    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + C::kStages;
    uint64_t* s_full = empty + C::kStages;   // [2] scores (after the last block: the output) ready
    uint64_t* p_half = s_full + 2;           // [2] output rescaled, probabilities of keys 0-63 written
    uint64_t* p_full = p_half + 2;           // [2] of keys 64-127
    uint64_t* done = p_full + 2;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::kOffSlot);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::kOffSlot + 4);
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_half[i], 4);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(done, 1);
        *s_abort = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= kLoadWarp) {
        if (warp == kLoadWarp) {
            // ----------------------------------------------------------------- loads
            if (n_all > 0) {
                if (lane == 0) {
                    const int tokens = tile_rows / p.group;
                    const uint32_t bytes = static_cast<uint32_t>(tile_rows) * 128u * C::kHalves;
                    mbar_arrive_expect_tx(q_full, n_blocks[1] > 0 ? 2 * bytes : bytes);
                    for (int i = 0; i < (n_blocks[1] > 0 ? 2 : 1); ++i)
                        for (int h = 0; h < C::kHalves; ++h)
                            tma_load_3d(base + i * C::kQTile + h * kRows * 128, &maps.q, q_full, h * 64, kvh * p.group,
                                        s.q0 + first_row / p.group + i * tokens);
                }
                // lane l looks after the block's slots [l * box, l * box + box)
                const int boxes = kKeys / box_slots;
                const int32_t* table = c.page_table + b * c.table_stride;
                auto look_up = [&](int j, int* slot) {
                    const int key = seg_lo + j * kKeys + lane * box_slots;
                    if (lane >= boxes || key >= seg_hi || key + box_slots <= range.lo) return -1;
                    const int pg = key / c.page_size;
                    *slot = key - pg * c.page_size;
                    return table[pg];
                };
                int slot = 0, next_slot = 0, issued = 0;
                int next_id = look_up(0, &next_slot);
                bool ok = true;
                for (int j = 0; j < n_all && ok; ++j) {
                    const int key = seg_lo + j * kKeys + lane * box_slots;
                    const bool mine = lane < boxes && key < seg_hi && key + box_slots > range.lo;
                    int id = next_id;
                    slot = next_slot;
                    if (j + 1 < n_all) next_id = look_up(j + 1, &next_slot);
                    if (mine && (id < 0 || id >= c.n_pages)) {
                        record_device_error(kDevErrPage);
                        id = c.n_pages;   // past the tensor: the copy fills zeros
                    }
                    const uint32_t n_boxes = __popc(__ballot_sync(~0u, mine));
                    for (int kv = 0; kv < 2; ++kv, ++issued) {
                        const int st = issued % C::kStages, r = issued / C::kStages;
                        if (r > 0) ok = __all_sync(~0u, wait_or_abort(&empty[st], (r - 1) & 1, s_abort, kDevErrEmptyWait));
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[st], n_boxes * static_cast<uint32_t>(box_slots) * 128u * C::kHalves);
                        __syncwarp();
                        if (mine)
                            for (int h = 0; h < C::kHalves; ++h)
                                tma_load_4d(base + C::kOffRing + st * C::kBlock + h * kKeys * 128 + lane * box_slots * 128,
                                            kv ? &maps.v : &maps.k, &full[st], h * 64, slot, kvh, id);
                    }
                }
                if (!ok) *s_abort = 1;
                // leave no copy in flight
                if (!tc::wait_bar(q_full, 0, kDevErrDrainWait)) *s_abort = 1;
                for (int it = max(0, issued - C::kStages); it < issued; ++it)
                    if (!tc::wait_bar(&full[it % C::kStages], (it / C::kStages) & 1, kDevErrDrainWait)) break;
            }
        } else if (warp == kMmaWarp) {
            // ----------------------------------------------------------------- MMAs
            bool ok = n_all > 0 && __all_sync(~0u, wait_or_abort(q_full, 0, s_abort, kDevErrFullWait));
            auto wait_stage = [&](int it) { return __all_sync(~0u, wait_or_abort(&full[it % C::kStages], (it / C::kStages) & 1, s_abort, kDevErrFullWait)); };
            auto issue_s = [&](int i, int it) {
                const uint64_t q = tc::sw128_desc(base + i * C::kQTile);
                const uint64_t kk = tc::sw128_desc(base + C::kOffRing + it % C::kStages * C::kBlock);
#pragma unroll
                for (int h = 0; h < C::kHalves; ++h) {
                    uint64_t qd[4], kd[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {   // 16 dimensions are 32 bytes inside a swizzled row, 64 the next box
                        qd[k] = q + static_cast<uint64_t>(h * (kRows * 128 >> 4) + k * 2);
                        kd[k] = kk + static_cast<uint64_t>(h * (kKeys * 128 >> 4) + k * 2);
                    }
                    mma_ss4(tmem + i * kKeys, qd, kd, C::kIdescS, h != 0);
                }
            };
            if (ok) {
                ok = wait_stage(0);
                if (ok) {
                    tc::tc_fence_after();
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (n_blocks[i] > 0) {
                            issue_s(i, 0);
                            commit(&s_full[i]);
                        }
                    commit(&empty[0]);
                }
            }
            for (int j = 0; j < n_all && ok; ++j) {
                const int v_it = 2 * j + 1, k_it = 2 * j + 2;
                // the 16-key steps that hold a key which some row sees
                const int t0 = seg_lo + j * kKeys;
                const int lo = max(0, range.lo - t0), hi = min(kKeys, seg_hi - t0);
                const int step0 = lo / 16, step1 = (hi + 15) / 16;
                const uint32_t v_smem = base + C::kOffRing + v_it % C::kStages * C::kBlock;
                // the loads first, so that nothing but the issue follows the probabilities
                ok = wait_stage(v_it) && (j + 1 >= n_all || wait_stage(k_it));
                if (!ok) break;
                if (lo > step0 * 16 || hi < step1 * 16) {
                    // V rows of the outer steps that belong to no visible key
                    const int n0 = lo - step0 * 16, n1 = step1 * 16 - hi, per = HD / 8;
                    for (int e = lane; e < (n0 + n1) * per; e += 32) {
                        const int r = e / per < n0 ? step0 * 16 + e / per : hi + e / per - n0, d = e % per;
                        const uint32_t at = v_smem + (d >> 3) * (kKeys * 128) + r * 128 + ((d & 7) ^ (r & 7)) * 16;
                        sts_v4(at, 0.0f, 0.0f, 0.0f, 0.0f);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                // V is [key][dim]: N-major, 64-dim boxes kKeys * 128 bytes apart, 8-key groups 1024
                const uint64_t vd = (static_cast<uint64_t>((v_smem >> 4) & 0x3FFFu)) |
                                    (static_cast<uint64_t>(kKeys * 128 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (j >= n_blocks[i]) continue;
                    const uint32_t o = tmem + C::kTmemO + i * HD, pr = tmem + i * kKeys;
                    const bool whole = step0 == 0 && step1 == kKeys / 16;
                    ok = __all_sync(~0u, wait_or_abort(&p_half[i], j & 1, s_abort, kDevErrMmaWait));
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (whole) mma_ts4(o, pr, vd, C::kIdescO, j > 0);
                    ok = __all_sync(~0u, wait_or_abort(&p_full[i], j & 1, s_abort, kDevErrMmaWait));
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (whole) {
                        mma_ts4(o, pr + kHalf, vd + 4 * (2048 >> 4), C::kIdescO, 1);
                    } else {
                        for (int st = step0; st < step1; ++st)
                            mma_ts(o, pr + p_column(st), vd + st * (2048 >> 4), C::kIdescO, j > 0 || st > step0);
                    }
                    if (j + 1 < n_blocks[i]) issue_s(i, k_it);
                    commit(&s_full[i]);
                }
                if (!ok) break;
                commit(&empty[v_it % C::kStages]);
                if (j + 1 < n_all) commit(&empty[k_it % C::kStages]);
            }
            if (!ok && n_all > 0) *s_abort = 1;
            commit(done);
            __all_sync(~0u, tc::wait_bar(done, 0, kDevErrMmaWait));
        }
    } else {
        // ----------------------------------------------------------------- softmax, two threads a row
        const int i = warp >> 3, half = (warp >> 2) & 1, r = threadIdx.x & 127;
        const int my_rows = min(tile_rows, rows - i * tile_rows);
        const int row = first_row + i * tile_rows + r;
        const bool real = r < my_rows;
        // a thread without a row looks where the tile's last row does, so that it needs no mask there
        const int like = first_row + i * tile_rows + max(0, min(r, my_rows - 1));
        const int pos = s.first_pos + like / p.group;
        int row_lo, row_hi;
        row_range(p, s, pos, &row_lo, &row_hi);
        const float slope = MOD && p.slopes ? p.slopes[kvh * p.group + like % p.group] * kLog2e : 0.0f;
        // f(this thread's value, its row's other value), the same in both: by the second half's thread
        float* place = reinterpret_cast<float*>(smem + C::kOffRow) + i * kRows + r;
        auto join = [&](float mine, auto f) {
            if (half == 0) *place = mine;
            named_barrier(1 + i * 4 + (warp & 3), 64);
            if (half == 1) *place = f(*place, mine);
            named_barrier(1 + i * 4 + (warp & 3), 64);
            return *place;
        };
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;   // this warp's 32 tensor-memory lanes
        const uint32_t ts = tmem + lanes + i * kKeys + half * kHalf, to = tmem + lanes + C::kTmemO + i * HD;
        const float unit = MOD ? 1.0f : p.scale_log2;
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < n_blocks[i]; ++j) {
            // after a timeout anywhere no wait is entered, but the group's barriers are all met
            wait_or_abort(&s_full[i], j & 1, s_abort, kDevErrMmaWait);
            __syncwarp();
            tc::tc_fence_after();
            const int t0 = seg_lo + j * kKeys + half * kHalf;
            // 32 of this thread's scores as the tensor core left them
            auto load = [&](int q, uint32_t (&sc)[32]) {
                tc::tmem_ld32(ts + 32 * q, sc);
                tc::tc_wait_ld();
            };
            // in the units of the sum to come (MOD), -inf where the row may not look; whether that is anywhere
            auto score = [&](int q, uint32_t (&sc)[32], bool mod) {
                const int lo = row_lo - t0 - 32 * q, hi = row_hi - t0 - 32 * q;
                const bool masked = __any_sync(~0u, lo > 0 || hi < 32);
                if (mod) {
                    if (p.cap > 0.0f) {
                        if (masked) {   // two scores share a reciprocal: nothing may come of a slot past the cache
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e < lo || e >= hi) sc[e] = 0u;
                        }
                        if (p.cap <= kCapPlain) {
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float2 t = capped_plain(p, __uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
                                sc[e] = __float_as_uint(t.x);
                                sc[e + 1] = __float_as_uint(t.y);
                            }
                        } else {
                            // under such a cap hardly a score comes to where it bends: a warp whose
                            // 32 rows have none takes the polynomial alone
                            float largest = 0.0f;
#pragma unroll
                            for (int e = 0; e < 32; ++e) largest = fmaxf(largest, fabsf(__uint_as_float(sc[e])));
                            if (__all_sync(~0u, largest * fabsf(p.cap_in) < kCapBend)) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) sc[e] = __float_as_uint(capped_small(p, __uint_as_float(sc[e])));
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) sc[e] = __float_as_uint(capped_exact(p, __uint_as_float(sc[e])));
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) sc[e] = __float_as_uint(__uint_as_float(sc[e]) * p.scale_log2);
                    }
                    if (p.slopes) {
                        const float dist = static_cast<float>(pos - t0 - 32 * q);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            sc[e] = __float_as_uint(fmaf(-slope, fabsf(dist - static_cast<float>(e)), __uint_as_float(sc[e])));
                    }
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (e < lo || e >= hi) sc[e] = 0xff800000u;
                }
                return masked;
            };
            auto top = [&](const uint32_t (&sc)[32]) {
                float mx[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mx[q] = max_nan(__uint_as_float(sc[q]), __uint_as_float(sc[q + 4]));
#pragma unroll
                    for (int e = q + 8; e < 32; e += 8) mx[q] = e + 4 < 32 ? max3(mx[q], __uint_as_float(sc[e]), __uint_as_float(sc[e + 4])) : mx[q];
                }
                return max_nan(max3(mx[0], mx[1], mx[2]), mx[3]);
            };
            // The second 32 scores come again after the maximum is known (registers left free let the
            // exponentials overlap); scores that took work go back to tensor memory for that.
            uint32_t first[32], second[32];
            load(0, first);
            const bool masked0 = score(0, first, MOD);
            float mn = top(first);
            if constexpr (MOD) tc::tmem_st32(ts, first);
            load(1, second);
            const bool masked1 = score(1, second, MOD);
            mn = max_nan(m, unit * max_nan(mn, top(second)));   // a NaN score makes the row NaN
            if constexpr (MOD) {
                tc::tmem_st32(ts + 32, second);
                tc::tc_wait_st();
            }
            // Whether a row of this pair of warps (the two halves of 32 rows) needs a new maximum
            if (pair_any(1 + i * 4 + (warp & 3), real && !(mn <= m + 8.0f) && mn != -INFINITY)) {
                mn = join(mn, [](float a, float b) { return max_nan(a, b); });
                const float f = mn == -INFINITY ? 1.0f : ex2(m - mn);
                l *= f;
                m = mn;
                if (j > 0 && half == 0) {
                    // the product of the last block is done: its commit came with these scores
#pragma unroll
                    for (int q = 0; q < HD / 16; ++q) {
                        uint32_t o[32], w[16];   // sixteen columns at a time: the scores hold their registers
                        tc::tmem_ld16(to + 16 * q, o);
                        tc::tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tc::tmem_st16(to + 16 * q, w);
                    }
                }
            }
            const float off = m == -INFINITY ? 0.0f : m;
            const float2 unit2 = make_float2(unit, unit), off2 = make_float2(-off, -off);
            float2 sum = make_float2(0.0f, 0.0f);
            // 32 probabilities over the first 16 (q = 0) or the next 16 columns of this half's scores
            auto probabilities = [&](const uint32_t (&sc)[32], int q, auto split) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 x = fma2(make_float2(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), unit2, off2);
                    if (decltype(split)::value && e * kFma / 16 != (e + 1) * kFma / 16) {
                        x = ex2_fma(x);
                    } else {
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                    }
                    sum = add2(sum, x);
                    pk[e] = pack_bf16(x.x, x.y);
                }
                tc::tmem_st16(ts + 16 * q, pk);
            };
            if constexpr (MOD) load(0, first);
            if (masked0) probabilities(first, 0, std::false_type{});
            else probabilities(first, 0, std::true_type{});
            load(1, second);
            if constexpr (!MOD) score(1, second, false);
            if (masked1) probabilities(second, 1, std::false_type{});
            else probabilities(second, 1, std::true_type{});
            tc::tc_wait_st();
            tc::tc_fence_before();
            __syncwarp();
            // of two warps on a scheduler the lower one runs ahead: keys 0-63 are done first, and
            // the tensor core starts on them
            if (lane == 0) mbar_arrive(half ? &p_full[i] : &p_half[i]);
            l += sum.x + sum.y;
        }
        if (n_blocks[i] > 0) {
            wait_or_abort(&s_full[i], n_blocks[i] & 1, s_abort, kDevErrMmaWait);
            __syncwarp();
            tc::tc_fence_after();
        }
        named_barrier(1 + i * 4 + (warp & 3), 64);   // every place has been read
        l = join(l, [](float a, float b) { return a + b; });
        if (my_rows > 0) {
            const int64_t token = s.q0 + row / p.group, head = kvh * p.group + row % p.group;
            const int D = c.head_dim;
            const int64_t at = split * part.rows + token * p.q_heads + head;
            if (real && half == 0 && range.splits > 1) part.ml[at] = make_float2(m, l);
#pragma unroll
            for (int q = 0; q < HD / 64; ++q) {
                uint32_t o[32];
                if (n_blocks[i] > 0) {
                    tc::tmem_ld32(to + half * (HD / 2) + 32 * q, o);
                    tc::tc_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    const int d = half * (HD / 2) + 32 * q + e;
                    if (!real || d >= D) continue;
                    const float4 x = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                    const float4 y = make_float4(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]), __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
                    if (range.splits > 1) {
                        *reinterpret_cast<float4*>(part.o + at * D + d) = x;
                        *reinterpret_cast<float4*>(part.o + at * D + d + 4) = y;
                    } else {
                        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
                        const uint4 w = make_uint4(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv),
                                                   pack_bf16(y.x * inv, y.y * inv), pack_bf16(y.z * inv, y.w * inv));
                        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + token * p.o_token + head * p.o_head + d) = w;
                    }
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// A bf16 tensor map of `rank` dimensions, the first one dense; strides in elements.
static int encode_map(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const int* box) {
    EncodeTiledFn fn = nullptr;
    if (int rc = encode_tiled_entry(&fn)) return rc;
    cuuint64_t d[4], st[3];
    cuuint32_t bx[4], es[4];
    for (int i = 0; i < rank; ++i) {
        d[i] = static_cast<cuuint64_t>(dims[i]);
        bx[i] = static_cast<cuuint32_t>(box[i]);
        es[i] = 1;
        if (i) st[i - 1] = static_cast<cuuint64_t>(std::max<int64_t>(strides[i] * 2, 16));   // 0 only along a dimension of 1, never stepped
    }
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, st, bx, es,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(BYBYCU_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for a cache or query tensor", static_cast<int>(r));
    return BYBYCU_OK;
}

template <int HD, bool MOD>
static int launch(const kvc::Cache& c, const Params& p, const DeviceInfo& info, cudaStream_t stream) {
    using C = Cfg<HD>;
    auto kern = attention_tc_kernel<HD, MOD>;
    static std::once_flag once[64];
    static cudaError_t prep[64];
    if (info.device < 0 || info.device >= 64) return set_error(BYBYCU_ERR_ARGS, "device %d out of range", info.device);
    std::call_once(once[info.device], [&] {
        prep[info.device] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem));
    });
    if (prep[info.device] != cudaSuccess) return cuda_fail(prep[info.device], "attention_tc_kernel shared memory");
    const int tokens = kRows / p.group, tile_rows = tokens * p.group;
    const int box_slots = std::min(c.page_size, kKeys);
    Maps maps;
    {
        const int64_t dims[3] = {c.head_dim, p.q_heads, c.n_tokens}, strides[3] = {1, p.q_head, p.q_token};
        const int box[3] = {64, p.group, tokens};
        if (int rc = encode_map(&maps.q, p.q, 3, dims, strides, box)) return rc;
    }
    {
        const int64_t dims[4] = {c.head_dim, c.page_size, c.kv_heads, c.n_pages}, strides[4] = {1, c.token_stride, c.head_stride, c.page_stride};
        const int box[4] = {64, box_slots, 1, 1};
        if (int rc = encode_map(&maps.k, c.k, 4, dims, strides, box)) return rc;
        if (int rc = encode_map(&maps.v, c.v, 4, dims, strides, box)) return rc;
    }
    const int64_t tiles = ceil_div(static_cast<int64_t>(p.max_q) * p.group, 2 * tile_rows);
    const int64_t units = tiles * c.kv_heads * c.n_seqs;
    const int64_t span = longest_span(p, 2 * tile_rows) + kKeys;
    // Split the keys only where the tiles that can have rows leave SMs idle, in pieces of four blocks
    // at least.  With more tiles than SMs the partial sums cost more than the even end gives (4
    // sequences of up to 1000 tokens over 3000 keys, 32/8 heads of 128: 87 us whole, 123 in two).
    const int64_t active = std::min(units, (ceil_div(static_cast<int64_t>(c.n_tokens) * p.group, 2 * tile_rows) + c.n_seqs) * c.kv_heads);
    int64_t splits = active < info.sm_count ? info.sm_count / active : 1;
    const int64_t split_keys64 = std::max<int64_t>(ceil_div(ceil_div(span, splits), kKeys) * kKeys, 4 * kKeys);
    splits = splits == 1 ? 1 : ceil_div(span, split_keys64);
    const int split_keys = splits == 1 ? INT32_MAX / kKeys * kKeys : static_cast<int>(split_keys64);   // one split: any cache's keys
    if (units * splits > INT32_MAX)
        return set_error(BYBYCU_ERR_SHAPE, "paged_attention: %d sequences, %d kv heads, %d new tokens", c.n_seqs, c.kv_heads, p.max_q);
    Partials part{};
    SplitScratchMem scratch;
    if (splits > 1)
        if (int rc = scratch.take(info.device, static_cast<int64_t>(c.n_tokens) * p.q_heads, static_cast<int>(splits), c.head_dim, stream, &part)) return rc;
    cudaLaunchAttribute attr[1];
    // K and V of a band: about half of the 126 MB L2; bands of one size, so that none is short
    const int64_t unit_bytes = std::min<int64_t>(span, split_keys) * c.head_dim * 4;
    const int64_t kv_units = static_cast<int64_t>(c.n_seqs) * c.kv_heads * splits;
    const int64_t bands = ceil_div(kv_units, std::max<int64_t>(1, (64 << 20) / unit_bytes));
    const int band = static_cast<int>(ceil_div(kv_units, bands));
    const cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(units * splits)), kThreads, C::kSmem, stream, attr);
    BYBYCU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, c, p, part, split_keys, static_cast<int>(splits), static_cast<int>(tiles), band,
                                       tile_rows, box_slots));
    return splits > 1 ? launch_join(c, p, part, split_keys, 2 * tile_rows, kKeys, false, stream) : BYBYCU_OK;
}

}  // namespace tcore

// Head dimensions up to 128, groups up to 128 heads, pages that tile a block of 128 keys (or are
// tiled by it) in whole swizzle atoms of 8 slots, and queries that step from token to token (a tensor
// map's strides are 16 bytes at least).
static bool tc_attention_supports(const kvc::Cache& c, const Params& p, bool f32) {
    const bool pages = c.page_size % 8 == 0 && (tcore::kKeys % c.page_size == 0 || c.page_size % tcore::kKeys == 0);
    return !f32 && c.head_dim <= 128 && p.group <= tcore::kRows && pages && (p.q_token > 0 || c.n_tokens == 1);
}

static int launch_tc_attention(const kvc::Cache& c, const Params& p, bool mod, cudaStream_t stream) {
    if (p.max_q == 0) return BYBYCU_OK;
    DeviceInfo info;
    if (int rc = current_device_info(&info)) return rc;
    // the plain kernel takes the maximum of unscaled scores: a scale above 0 only
    mod = mod || !(p.scale_log2 > 0.0f);
    if (c.head_dim <= 64) return mod ? tcore::launch<64, true>(c, p, info, stream) : tcore::launch<64, false>(c, p, info, stream);
    return mod ? tcore::launch<128, true>(c, p, info, stream) : tcore::launch<128, false>(c, p, info, stream);
}

}  // namespace attn
}  // namespace bybycu
