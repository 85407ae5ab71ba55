// What the gated recurrence, attention and paged attention share: the element types, and their conversions, which round to nearest even.
#pragma once

#include "common.h"

namespace rwkv {

struct bf16_t { uint16_t bits; };
typedef _Float16 half_t;

DEVINL float to_f(bf16_t x) { return bf2f(x.bits); }
DEVINL float to_f(half_t x) { return static_cast<float>(x); }
DEVINL float to_f(float x) { return x; }
template <class E> DEVINL E from_f(float x) {
    if constexpr (std::is_same_v<E, bf16_t>) return {f2bf(x)};
    else return static_cast<E>(x);
}

// What the scores' arithmetic holds for: the capped score is made as cap - 2 cap / (1 + e^z), which is off by 2^-23 cap, and e^z's argument must not overflow.
// (attention's biases on keys behind a query are divided by the scale: check_attn.)
inline bool scores_ok(const float scale, const float cap) { return scale > 0.f && scale <= 0x1p60f && (cap == 0.f || (cap >= 0x1p-20f && cap <= 4096.f)); }

// Attention's tokens are less than this many elements apart: a tile of 64 rows is addressed with 31 bits.
constexpr int MAX_TOKEN_STRIDE = 1 << 24;

// The documents of a tile of 64 positions, made by a kernel of its own before the others.
struct Range {
    int lo, hi;                                                 // of the tokens that are no padding; INT_MAX and -1 without one
    int whole;                                                  // 64 tokens, none of them padding
    int unused;
};
// How the work of few queries or keys is spread over the card (a rule on sizes alone, for the kernels and for the size of their workspace).  `query_parts`: the keys of
// a query in as many parts, joined by a kernel of its own; `key_parts`: the heads that share a key in as many groups, whose sums are added by a kernel of its own.
struct AttnPlan {
    int query_parts, key_parts;
    bool eight;                                                 // heads of 128: 256 keys a workgroup of attn_dkv
    int q_items, k_items;                                       // blocks of queries, of keys, that are ordered by their work (0: they are not)
    int delta_blocks;                                           // workgroups of attn_delta for a batch element, fp16, each of which leaves its largest lengths
    size_t ranges, q_order, k_order, forward, backward;         // bytes: documents of tiles; the orders; workspace of either direction
    size_t delta, lengths;                                      // ... of delta; of the largest lengths of gradients and of values
};
constexpr int MAX_ORDER = 1024;
AttnPlan attn_plan(int B, int Tq, int Tk, int H, int Hk, int N, bool doc);
// attn_bwd.hip: tile i of `out`'s row b has positions first + 64 i .. of doc's row b, below T
void launch_attn_ranges(hipStream_t st, const int* doc, int B, int T, int first, Range* out);
// attn_bwd.hip: the blocks of queries and of keys, of which either may be null, in the order of their work
void launch_attn_order(hipStream_t st, const rwkv_attn_args& p, const Range* keys, const Range* queries, const AttnPlan& plan, int* q_order, int* k_order);
// attn_fwd.hip, attn_bwd.hip (arguments checked)
int launch_attn_fwd(hipStream_t st, const rwkv_attn_args& p);
int launch_attn_bwd(hipStream_t st, const rwkv_attn_args& p);

}  // namespace rwkv
