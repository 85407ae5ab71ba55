// Attention with capped scores, distance bias, documents and prefixes: the entry points (the arguments are explained in rwkv_hip.h).  Kernels:
// attn_fwd.hip, attn_bwd.hip.  Backward, with p the softmax's weights, dp = dy.v and delta = dy.y:  ds = p (dp - delta) (1 - tanh^2);
// dv = p^T dy;  dq = scale ds k;  dk = scale ds^T q.
#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

bool multiples_of_8(std::initializer_list<int64_t> xs) {
    for (const int64_t x : xs) if (x % 8 != 0) return false;
    return true;
}
// a tile of 64 rows is addressed with 31 bits
bool wide_rows(const rwkv_attn_args& p) {
    for (const int64_t s : {p.q_st, p.k_st, p.v_st, static_cast<int64_t>(p.H) * p.N}) if (s < 0 || s >= 1 << 24) return true;
    return false;
}
int check_attn(const rwkv_attn_args* p, bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->Tq <= 0 || p->Tk < p->Tq || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 ||
        p->N <= 0 || p->N > 128 || p->N % 8 != 0 || p->B > 65535 || p->H > 65535 || wide_rows(*p) || !(p->scale > 0.f) || !(p->cap >= 0.f) || (p->prefix != nullptr && !p->causal)) return RWKV_ERR_SHAPE;
    if (!multiples_of_8({p->q_sb, p->q_st, p->q_sh, p->k_sb, p->k_st, p->k_sh, p->v_sb, p->v_st, p->v_sh})) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k, p->v, p->y})) return rc;
    if (backward) {
        if (const int rc = check_ptrs({p->dy, p->dq, p->dk, p->dv, p->y_rest})) return rc;
        if (p->lse == nullptr) return RWKV_ERR_NULL;
        if (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < rwkv_attn_workspace_bytes(p->B, p->Tq, p->Tk, p->H, p->doc != nullptr, 1)) return RWKV_ERR_WORKSPACE;
    } else {
        if (!aligned16(p->y_rest)) return RWKV_ERR_ALIGN;
        if (p->doc != nullptr && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < rwkv_attn_workspace_bytes(p->B, p->Tq, p->Tk, p->H, 1, 0))) return RWKV_ERR_WORKSPACE;
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

// the documents of tiles of 64 keys (16 bytes each), in the backward also of tiles of queries, and a sum of each query and head
size_t rwkv_attn_workspace_bytes(int B, int Tq, int Tk, int H, int doc, int backward) {
    if (B <= 0 || Tq <= 0 || Tk < Tq || H <= 0) return 0;
    size_t n = doc ? static_cast<size_t>(B) * ((static_cast<int64_t>(Tk) + 63) / 64) * 16 : 0;
    if (backward) n += (doc ? static_cast<size_t>(B) * ((static_cast<int64_t>(Tq) + 63) / 64) * 16 : 0) + static_cast<size_t>(B) * Tq * H * sizeof(float);
    return n;
}
int rwkv_attn_forward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, false); }
int rwkv_attn_backward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, true); }

}  // extern "C"
