// Attention with capped scores, distance bias, documents and prefixes: the entry points (the arguments are explained in rwkv_hip.h).  Kernels:
// attn_fwd.hip, attn_bwd.hip.  Backward, with p the softmax's weights, dp = dy.v and delta = dy.y:  ds = p (dp - delta) (1 - tanh^2);
// dv = p^T dy;  dq = scale ds k;  dk = scale ds^T q.
#include <algorithm>
#include <climits>

#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

bool multiples_of_8(std::initializer_list<int64_t> xs) {
    for (const int64_t x : xs) if (x % 8 != 0) return false;
    return true;
}
bool wide_rows(const rwkv_attn_args& p) {
    for (const int64_t s : {p.q_st, p.k_st, p.v_st, static_cast<int64_t>(p.H) * p.N}) if (s < 0 || s >= MAX_TOKEN_STRIDE) return true;
    return false;
}
}  // namespace

// A CU runs two workgroups of attn_fwd with heads of 128, four with heads of 64.  B1 Tq512 Tk16384 H32 N128, 128 workgroups: 0.30 ms whole, 0.144 ms in four parts.
// attn_dkv: B1 T3001 H32 Hk8 N128 with five documents, 192 workgroups: 0.30 ms whole, 0.18 ms in four groups.
AttnPlan attn_plan(int B, int Tq, int Tk, int H, int Hk, int N, bool doc) {
    const int64_t width = N <= 64 ? 64 : 128, tiles = (static_cast<int64_t>(Tk) + 63) / 64;
    const auto blocks = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    AttnPlan a{};
    const int64_t queries = blocks(Tq, 128) * H * B, room = width == 64 ? 1024 : 512;
    a.query_parts = static_cast<int>(std::max<int64_t>(1, std::min({room / queries, tiles / 8, int64_t{16}})));
    const int G = H / Hk;
    const int64_t keys = blocks(Tk, width == 64 ? 128 : 256) * Hk * B, want = width == 64 ? 512 : 256;
    a.key_parts = 1;
    for (int x = 2; x <= G; ++x)
        if (G % x == 0 && keys * a.key_parts < want) a.key_parts = x;
    a.eight = width == 128 && keys * a.key_parts >= 256;
    a.ranges = doc ? static_cast<size_t>(B) * tiles * sizeof(Range) : 0;
    // Documents make unequal blocks: the most work first, where there are more than the card takes at once.  Forward + backward with H32 Hk8 N128 in ms, in their own
    // order / sorted: B1 T3001 0.357 / 0.266, B4 T4096 1.54 / 1.19, B8 T4096 2.24 / 1.91, B1 T16384 2.70 / 2.21; B1 T700, all at once, 0.105 / 0.112.
    const int64_t q_items = blocks(Tq, 128) * B, k_items = blocks(Tk, a.eight ? 256 : 128) * B;
    const auto ordered = [&](int64_t items, int64_t heads, int64_t at_once) { return doc && items <= MAX_ORDER && items * heads > at_once; };
    a.q_items = ordered(q_items, H, 512) && a.query_parts == 1 ? static_cast<int>(q_items) : 0;
    a.k_items = ordered(k_items, static_cast<int64_t>(Hk) * a.key_parts, 256) ? static_cast<int>(k_items) : 0;
    const auto order = [](int items) { return (static_cast<size_t>(items) * sizeof(int) + 15) / 16 * 16; };
    a.q_order = order(a.q_items);
    a.k_order = order(a.k_items);
    a.forward = a.ranges + a.q_order + (a.query_parts > 1 ? static_cast<size_t>(B) * H * Tq * a.query_parts * (width + 4) * sizeof(float) : 0);
    // enough workgroups to fill the card, and few enough for each of attn_dkv to look at what they leave
    a.delta_blocks = static_cast<int>(std::min(blocks(static_cast<int64_t>(Tq) * H, 2048 / width), blocks(2048, B)));
    a.delta = (static_cast<size_t>(B) * Tq * H * sizeof(float) + 15) / 16 * 16;
    a.lengths = (static_cast<size_t>(B) * a.delta_blocks * 2 * sizeof(float) + static_cast<size_t>(B) * Hk * blocks(Tk, a.eight ? 256 : 128) * sizeof(float) + 15) / 16 * 16;
    a.backward = a.ranges + a.q_order + a.k_order + (doc ? static_cast<size_t>(B) * blocks(Tq, 64) * sizeof(Range) : 0) + a.delta + a.lengths +
                 (a.key_parts > 1 ? 2 * static_cast<size_t>(a.key_parts) * B * Tk * Hk * N * sizeof(float) : 0);
    return a;
}

namespace {

int check_attn(const rwkv_attn_args* p, bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->Tq <= 0 || p->Tk < p->Tq || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 ||
        p->N <= 0 || p->N > 128 || p->N % 8 != 0 || p->B > 65535 || p->H > 65535 || wide_rows(*p) || !scores_ok(p->scale, p->cap) || p->Tk > INT_MAX - 65536 ||
        (p->slopes != nullptr && (p->Tk > 1 << 24 || p->scale < 0x1p-60f)) || (p->prefix != nullptr && !p->causal)) return RWKV_ERR_SHAPE;
    if (!multiples_of_8({p->q_sb, p->q_st, p->q_sh, p->k_sb, p->k_st, p->k_sh, p->v_sb, p->v_st, p->v_sh})) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k, p->v, p->y})) return rc;
    if (backward) {
        if (const int rc = check_ptrs({p->dy, p->dq, p->dk, p->dv, p->y_rest})) return rc;
        if (p->lse == nullptr) return RWKV_ERR_NULL;
        if (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < attn_plan(p->B, p->Tq, p->Tk, p->H, p->Hk, p->N, p->doc != nullptr).backward) return RWKV_ERR_WORKSPACE;
    } else {
        if (!aligned16(p->y_rest)) return RWKV_ERR_ALIGN;
        const size_t need = attn_plan(p->B, p->Tq, p->Tk, p->H, p->Hk, p->N, p->doc != nullptr).forward;
        if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) return RWKV_ERR_WORKSPACE;
    }
    for (const void* q : {static_cast<const void*>(p->slopes), static_cast<const void*>(p->doc), static_cast<const void*>(p->prefix), static_cast<const void*>(p->lse)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    return RWKV_OK;
}

int attn_any(void* stream, const rwkv_attn_args* p, bool backward) {
    if (const int rc = check_attn(p, backward)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return backward ? launch_attn_bwd(st, *p) : launch_attn_fwd(st, *p);
}

}  // namespace
}  // namespace rwkv

extern "C" {

size_t rwkv_attn_workspace_bytes(int B, int Tq, int Tk, int H, int Hk, int N, int doc, int backward) {
    if (B <= 0 || Tq <= 0 || Tk < Tq || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || N > 128 || B > 65535 || H > 65535) return 0;
    const rwkv::AttnPlan a = rwkv::attn_plan(B, Tq, Tk, H, Hk, N, doc != 0);
    return backward ? a.backward : a.forward;
}
int rwkv_attn_forward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, false); }
int rwkv_attn_backward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, true); }

}  // extern "C"
