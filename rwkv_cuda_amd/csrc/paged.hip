// Attention of one new token a sequence over a cache in pages (the arguments are explained in rwkv_hip.h).
#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

constexpr int64_t L(int x) { return x; }

// one wave a query; lane = token of a tile of 64, then lane = channel
template <class E> __global__ __launch_bounds__(64) void paged_plain(const rwkv_paged_args p, const int shift) {
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x, hk = h / (p.H / p.Hk);
    __shared__ float w[64];
    __shared__ const E* at[64];
    const E* q = static_cast<const E*>(p.q) + (L(b) * p.H + h) * p.N;
    const int all = p.lens[b], n = static_cast<int>(all < L(p.M) << shift ? all : L(p.M) << shift);
    float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane, pg = j < n ? p.table[L(b) * p.M + (j >> shift)] : -1, row = j & (p.page - 1);
        const bool on = pg >= 0 && pg < p.P;
        float s = -INFINITY;
        if (on) {
            E* kr = static_cast<E*>(p.k_pages) + pg * p.k_sp + row * p.k_st + hk * p.k_sh;
            E* vr = static_cast<E*>(p.v_pages) + pg * p.v_sp + row * p.v_st + hk * p.v_sh;
            const E *kx = kr, *vx = vr;
            if (p.k != nullptr && j == all - 1) {
                kx = static_cast<const E*>(p.k) + (L(b) * p.Hk + hk) * p.N;
                vx = static_cast<const E*>(p.v) + (L(b) * p.Hk + hk) * p.N;
                if (h % (p.H / p.Hk) == 0)
                    for (int d = 0; d < p.N; ++d) { kr[d] = kx[d]; vr[d] = vx[d]; }
            }
            s = 0.f;
            for (int d = 0; d < p.N; ++d) s += to_f(q[d]) * to_f(kx[d]);
            s *= p.scale;
            if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
            if (p.slopes) s -= p.slopes[h] * static_cast<float>(all - 1 - j);
            at[lane] = vx;
        }
        float top = s;
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        top = fmaxf(m, top);
        if (top == -INFINITY) continue;
        const float grow = m == -INFINITY ? 0.f : __expf(m - top), x = on ? __expf(s - top) : 0.f;
        l = l * grow + group_sum<64>(x);
        m = top;
        w[lane] = x;
        __syncthreads();
        for (int e = 0; e < 2; ++e) {
            const int d = lane + 64 * e;
            if (d >= p.N) continue;
            acc[e] *= grow;
            for (int t = 0; t < 64; ++t) if (w[t] != 0.f) acc[e] += w[t] * to_f(at[t][d]);
        }
        __syncthreads();
    }
    for (int e = 0; e < 2; ++e) {
        const int d = lane + 64 * e;
        if (d < p.N) static_cast<E*>(p.y)[(L(b) * p.H + h) * p.N + d] = from_f<E>(l == 0.f ? 0.f : acc[e] / l);
    }
}

int check_paged(const rwkv_paged_args* p) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 || p->N <= 0 || p->N > 128 || p->N % 8 != 0 ||
        p->P <= 0 || p->M <= 0 || p->page <= 0 || (p->page & (p->page - 1)) != 0 || p->B > 65535 || p->H > 65535 || !(p->scale > 0.f) || !(p->cap >= 0.f)) return RWKV_ERR_SHAPE;
    for (const int64_t s : {p->k_sp, p->k_st, p->k_sh, p->v_sp, p->v_st, p->v_sh}) if (s % 8 != 0) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k_pages, p->v_pages, p->y})) return rc;
    if (p->table == nullptr || p->lens == nullptr || (p->k == nullptr) != (p->v == nullptr)) return RWKV_ERR_NULL;
    if (!aligned16(p->k) || !aligned16(p->v)) return RWKV_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(p->table), static_cast<const void*>(p->lens), static_cast<const void*>(p->slopes)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    const size_t need = rwkv_paged_workspace_bytes(p->B, p->H, p->Hk, p->N, p->page, p->M);
    if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" {

size_t rwkv_paged_workspace_bytes(int, int, int, int, int, int) { return 0; }

int rwkv_paged_attn(void* stream, const rwkv_paged_args* args) {
    using namespace rwkv;
    if (const int rc = check_paged(args)) return rc;
    const rwkv_paged_args& p = *args;
    const dim3 grid(p.H, p.B), block(64);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int shift = __builtin_ctz(p.page);
    if (p.dtype == RWKV_DTYPE_BF16) hipLaunchKernelGGL((paged_plain<bf16_t>), grid, block, 0, st, p, shift);
    else hipLaunchKernelGGL((paged_plain<half_t>), grid, block, 0, st, p, shift);
    return launch_status();
}

}  // extern "C"
