// kvcache.cuh - what the paged-cache operators share: the cache and batch as the kernels see
// them, the checks of their arguments, and where a token of a sequence lives.
#pragma once

#include "kernels.h"

namespace bybycu {
namespace kvc {

constexpr int kMaxHeadDim = 256;
// Positions of a sequence: below 2^31 by more than a kernel looks ahead in 32 bits.
constexpr int kMaxPositions = INT32_MAX - 8192;

// bybycu_paged_kv by value (kernel parameter).
struct Cache {
    __nv_bfloat16* k;
    __nv_bfloat16* v;
    int64_t page_stride, head_stride, token_stride;
    const int32_t* page_table;
    int64_t table_stride;
    const int32_t* q_start;
    const int32_t* kv_lens;
    int32_t n_pages, page_size, kv_heads, head_dim, max_pages, n_seqs, n_tokens;
};

inline bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// The checks of the cache and batch that every operator on them makes.
inline int check_cache(const bybycu_paged_kv* kv, const char* op, Cache* c) {
    if (!kv) return set_error(BYBYCU_ERR_ARGS, "%s: the cache is NULL", op);
    if (kv->kv_heads <= 0 || kv->page_size <= 0 || kv->n_pages <= 0 || kv->max_pages <= 0 || kv->n_seqs < 0 ||
        kv->n_tokens < 0)
        return set_error(BYBYCU_ERR_SHAPE, "%s: heads=%d page=%d pages=%d table=%d seqs=%d tokens=%d", op, kv->kv_heads,
                         kv->page_size, kv->n_pages, kv->max_pages, kv->n_seqs, kv->n_tokens);
    if (kv->head_dim < 8 || kv->head_dim > kMaxHeadDim || kv->head_dim % 8)
        return set_error(BYBYCU_ERR_SHAPE, "%s: head dimension %d is not a multiple of 8 up to %d", op, kv->head_dim,
                         kMaxHeadDim);
    if (static_cast<int64_t>(kv->max_pages) * kv->page_size > kMaxPositions)
        return set_error(BYBYCU_ERR_SHAPE, "%s: %d pages of %d tokens a sequence exceed 2^31 - 8193 positions", op,
                         kv->max_pages, kv->page_size);
    if (kv->reserved) return set_error(BYBYCU_ERR_ARGS, "%s: reserved fields must be 0", op);
    if (!kv->k || !kv->v || ((!kv->page_table || !kv->kv_lens) && kv->n_seqs > 0) || !kv->q_start)
        return set_error(BYBYCU_ERR_ARGS, "%s: a cache slot is missing", op);
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->page_table, 4) || !aligned(kv->q_start, 4) ||
        !aligned(kv->kv_lens, 4))
        return set_error(BYBYCU_ERR_ARGS, "%s: misaligned cache slot", op);
    if (kv->page_stride % 8 || kv->head_stride % 8 || kv->token_stride % 8 || kv->page_stride < 0 ||
        kv->head_stride < 0 || kv->token_stride < 0 || kv->table_stride < kv->max_pages)
        return set_error(BYBYCU_ERR_ARGS, "%s: cache strides must be non-negative multiples of 8 elements, table rows "
                                          "max_pages apart at least", op);
    // no two of a page's (head, slot) vectors may overlap, nor two pages
    const bool token_inner = kv->token_stride <= kv->head_stride;
    const int64_t inner = token_inner ? kv->token_stride : kv->head_stride;
    const int64_t outer = token_inner ? kv->head_stride : kv->token_stride;
    const int n_in = token_inner ? kv->page_size : kv->kv_heads, n_out = token_inner ? kv->kv_heads : kv->page_size;
    const int64_t span = (n_in > 1 ? (n_in - 1) * inner : 0) + kv->head_dim;
    const int64_t page = (n_out > 1 ? (n_out - 1) * outer : 0) + span;
    if ((n_in > 1 && inner < kv->head_dim) || (n_out > 1 && outer < span) || (kv->n_pages > 1 && kv->page_stride < page))
        return set_error(BYBYCU_ERR_ARGS, "%s: cache strides let slots overlap", op);
    *c = Cache{static_cast<__nv_bfloat16*>(kv->k), static_cast<__nv_bfloat16*>(kv->v), kv->page_stride,
               kv->head_stride, kv->token_stride, kv->page_table, kv->table_stride, kv->q_start, kv->kv_lens,
               kv->n_pages, kv->page_size, kv->kv_heads, kv->head_dim, kv->max_pages, kv->n_seqs, kv->n_tokens};
    return BYBYCU_OK;
}

// The strides of a [tokens, heads, head_dim] tensor whose vectors must be `align` elements apart.
inline bool strides_ok(int64_t token, int64_t head, int heads, int dim, int align) {
    return token >= 0 && head >= 0 && token % align == 0 && head % align == 0 && (heads == 1 || head >= dim);
}
// The same of an output: no two of its vectors may share an element, whichever of tokens and heads
// lies inside the other.
inline bool out_strides_ok(int64_t token, int64_t head, int tokens, int heads, int dim, int align) {
    if (!strides_ok(token, head, heads, dim, align)) return false;
    if (heads == 1) return tokens == 1 || token >= dim;
    if (tokens == 1 || (token >= dim && (head - dim) / (tokens - 1) >= token)) return true;
    return token >= dim && (token - dim) / (heads - 1) >= head;
}

// Number of the n ends q_start[1..n] that are <= t, counted by a whole block (every thread
// calls): the sequence of token t, n_seqs when it belongs to none.  The loads of one round are
// independent, where a binary search would chain eight of them.
__device__ __forceinline__ int block_seq_of(const Cache& c, int t) {
    int b = 0;
    for (int i = 0; i < c.n_seqs; i += blockDim.x) {
        const int s = i + static_cast<int>(threadIdx.x);
        b += __syncthreads_count(s < c.n_seqs && c.q_start[s + 1] <= t);
    }
    return b;
}

}  // namespace kvc
}  // namespace bybycu
