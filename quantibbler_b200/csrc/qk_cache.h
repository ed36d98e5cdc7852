// What the kernels over key/value caches share: the cache as the device sees it, the arguments of an attention call.
#pragma once

#include "qk_common.h"

namespace qk {

struct CacheView {
    void *k, *v;               // [n_seq][n_kv][rows][d]
    float *k_scale, *v_scale;  // INT8: [n_seq][n_kv][rows]
    uint32_t rows, n_seq, n_kv, d;
    int32_t dtype;
};

struct AttendArgs {
    const float *q;
    size_t q_stride;
    float *out;
    size_t out_stride;
    const int32_t *kv_len;     // one query per sequence: its rows; null: a portion, query t sees rows 0 .. first_row + t of `seq`
    uint32_t n_queries, n_heads;
    size_t seq;
    uint32_t first_row;
    uint32_t prefix_len;       // rows of the prefix's slot prefix_seq, seen by every query
    size_t prefix_seq;
    float *scratch;
};

// INT8: weights times value scales go into the products as two float16 terms, scaled so that 2^14 stands for a weight of one
// times 2^(e_max + 1), e_max the exponent of the largest value scale so far; the second term is held 2^11 times larger.  A
// weight times its scale that is 2^-27 of that or more is held to 2^-22 of itself, a smaller one to 2^-50 of that, which is
// 2^-33 of the key's own scale or less while the scales lie within 2^kScaleSpread of one another.  Where they do not (a row
// of zeros, whose scale is one, among small ones; an outlier that nearly nobody attends to), or are near the ends of
// float32's range, three bfloat16 terms take over, which hold any to 2^-24 of itself.  (`least`: the bits, less one, of the
// smallest scale that is not zero, so that zeros, whose rows add nothing, are the largest.)
constexpr int kScaleSpread = 16;
__device__ __forceinline__ bool scales_apart(int e_max, uint32_t least) {
    return e_max >= 120 || (least != 0xffffffffu && e_max - ((int)((least + 1) >> 23) - 127) > kScaleSpread);
}

// One launch of the tile kernel (qk_cache_tile.cu): all queries against rows of one slot.
struct TileArgs {
    const float *q;
    size_t q_stride;
    float *out;
    size_t out_stride;
    float *scratch;            // partial results where n_slots > 1: outputs [query][head][slot][d], then {maximum, sum}
    uint32_t n_queries, n_heads;
    size_t seq;
    int32_t causal;            // query t sees rows 0 .. first_row + t; else all see rows 0 .. n_keys - 1
    uint32_t first_row, n_keys;
    uint32_t n_splits, slot0, n_slots;  // the keys' splits go to slots slot0 .. of the n_slots of a (query, head)
    int *error;
    uint32_t wait_limit;
};
// INT8 or bfloat16, head_dim 64 or 128, everything on 16-byte boundaries; the context's error word exists.
qk_status attend_tiles(qk_ctx *c, const CacheView &cache, TileArgs a);

}  // namespace qk
