// Gated delta rule (the arguments are explained in rwkv_hip.h):  S = e^g S;  u = beta (v - S^T k);  S += k u^T;  y = scale S^T q.
//
// Token by token: the columns of the state (its value channels) do not depend on each other, so a workgroup keeps 32 of them in registers, a thread
// four columns of every 32nd row.  Both sums over the rows, S^T k and S^T q, are made from the state before the update, y = scale (e^g S^T q + (q.k) u), so that a token
// costs one exchange between the waves.  A token of 32 rows, 32 heads of 128: 27.7 us, the states read and written at 4.9 TB/s.
#include <algorithm>
#include <climits>

#include "delta.h"

namespace rwkv {
namespace {

template <class E, int ROWS>
__global__ __launch_bounds__(256) void delta_steps(const rwkv_delta_args p) {
    __shared__ float sums[2][4][64 + 4];
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk), tid = threadIdx.x, c0 = blockIdx.x * 32 + 4 * (tid & 7), r0 = tid >> 3, wave = tid >> 6, N = p.N;
    const int64_t head = wide(b) * p.H + h;
    const E *q = static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh, *k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh, *v = static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh;
    const E *g = static_cast<const E*>(p.g) + b * p.g_sb + h, *beta = static_cast<const E*>(p.beta) + b * p.beta_sb + h;
    E* y = static_cast<E*>(p.y) + (wide(b) * p.T * p.H + h) * N;
    const bool on = c0 < N;
    f32x4 s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + 32 * i;
        s[i] = p.s0 && on && r < N ? *reinterpret_cast<const f32x4*>(p.s0 + (head * N + r) * N + c0) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int t = 0, turn = 0; t < p.T; ++t) {
        const DeltaToken token = delta_token(p.doc, wide(b) * p.T, t, p.T);
        if (!token.real) {
            if (on && r0 == 0)
#pragma unroll
                for (int c = 0; c < 4; ++c) y[wide(t) * p.H * N + c0 + c] = from_f<E>(0.f);
            continue;
        }
        const float lg = to_f(g[t * p.g_st]), a = token.cut || lg < DELTA_NONE ? 0.f : expf(lg), bt = to_f(beta[t * p.beta_st]);
        float kr[ROWS], qr[ROWS], qk = 0.f;
        f32x4 ks{0.f, 0.f, 0.f, 0.f}, qs = ks, vt = ks;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = r0 + 32 * i;
            kr[i] = r < N ? to_f(k[t * p.k_st + r]) : 0.f;
            qr[i] = r < N ? to_f(q[t * p.q_st + r]) : 0.f;
            s[i] = a == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : s[i] * a;        // (what is no number goes with it)
            ks += kr[i] * s[i];
            qs += qr[i] * s[i];
            qk = fmaf(kr[i], qr[i], qk);
        }
        if (on)
#pragma unroll
            for (int c = 0; c < 4; ++c) vt[c] = to_f(v[t * p.v_st + c0 + c]);
#pragma unroll
        for (int x = 8; x <= 32; x <<= 1) {
#pragma unroll
            for (int c = 0; c < 4; ++c) ks[c] += __shfl_xor(ks[c], x, 64), qs[c] += __shfl_xor(qs[c], x, 64);
            qk += __shfl_xor(qk, x, 64);
        }
        float(&out)[4][68] = sums[turn ^= 1];
        if ((tid & 63) < 8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) out[wave][4 * tid % 32 + c] = ks[c], out[wave][32 + 4 * tid % 32 + c] = qs[c];
            if ((tid & 63) == 0) out[wave][64] = qk;
        }
        __syncthreads();
        f32x4 u;
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) all += out[w][64];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float x = 0.f, z = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x += out[w][4 * (tid & 7) + c], z += out[w][32 + 4 * (tid & 7) + c];
            u[c] = bt * (vt[c] - x);
            if (on && r0 == 0) y[wide(t) * p.H * N + c0 + c] = from_f<E>(p.scale * fmaf(all, u[c], z));
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) s[i] += kr[i] * u;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (on && r0 + 32 * i < N) *reinterpret_cast<f32x4*>(p.sT + (head * N + r0 + 32 * i) * N + c0) = s[i];
}

// dq and dk of a key head: the sums over the heads that share it
template <class E> __global__ __launch_bounds__(256) void delta_sum(const rwkv_delta_args p, const float* dq_of, const float* dk_of) {
    const int64_t n = wide(p.B) * p.T * p.Hk * p.N;
    const int G = p.H / p.Hk;
    for (int64_t x = blockIdx.x * 256ll + threadIdx.x; x < n; x += gridDim.x * 256ll) {
        const int c = static_cast<int>(x % p.N);
        const int64_t from = x / p.N * G * p.N + c;
        float q = 0.f, k = 0.f;
        for (int i = 0; i < G; ++i) q += dq_of[from + i * p.N], k += dk_of[from + i * p.N];
        static_cast<E*>(p.dq)[x] = from_f<E>(q);
        static_cast<E*>(p.dk)[x] = from_f<E>(k);
    }
}

// Few tokens go one by one: a chunk costs the same whatever it holds.  us with 1, 2, 4, 6, 8 tokens, 32 heads, a row and 32 rows: heads of 64 3.8 5.2 8.0 10.8 13.6 beside 6.8 of a chunk, and 9.0 12.6
// 21 29 39 beside 26.5; heads of 128 4.5 6.5 10.0 13.5 17.3 beside 8.4, and 27 36 53 72 90 beside 65 (of whose first 27 are the states, read and written at 4.9 TB/s).
// One number for all batches, so that a sequence's results do not depend on how many others there are; for a single row 3 would do, where four tokens take 1.2 and 1.6 us longer so.
constexpr int FEW = 4;
template <class E> int run_fwd(hipStream_t st, const rwkv_delta_args& p) {
    if (p.saved != nullptr || p.T > FEW) return launch_delta_fwd(st, p);
    const dim3 grid((p.N + 31) / 32, p.H, p.B);
    if (p.N <= 64) hipLaunchKernelGGL((delta_steps<E, 2>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((delta_steps<E, 4>), grid, dim3(256), 0, st, p);
    return launch_status();
}
template <class E> int run_bwd(hipStream_t st, const rwkv_delta_args& p) {
    const DeltaTiles tiles(p);
    float *dS = static_cast<float*>(p.workspace), *dZ = dS + tiles.states(), *dq = nullptr, *dk = nullptr;
    if (p.Hk != p.H) dq = dZ + tiles.updates(), dk = dq + static_cast<size_t>(p.B) * p.T * p.H * p.N;
    if (const int rc = launch_delta_bwd(st, p, dS, dZ)) return rc;
    if (const int rc = launch_delta_grads(st, p, dS, dZ, dq, dk)) return rc;
    if (dq) hipLaunchKernelGGL(delta_sum<E>, dim3(2048), dim3(256), 0, st, p, dq, dk);
    return launch_status();
}

// The sizes that the kernels hold for.
bool delta_sizes(int B, int T, int H, int Hk, int N) {
    return B > 0 && T > 0 && H > 0 && Hk > 0 && H % Hk == 0 && N > 0 && N <= 128 && N % 8 == 0 && B <= 65535 && H <= 65535 && T <= INT_MAX - 65536 &&
           (T + 63.0) * B * H < 0x1p37;                             // (chunks by 31 bits; what is kept of them, by 64)
}
int check_delta(const rwkv_delta_args* p, const bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || !delta_sizes(p->B, p->T, p->H, p->Hk, p->N) || !(p->scale > 0.f && p->scale <= 0x1p60f)) return RWKV_ERR_SHAPE;
    for (const int64_t s : {p->q_sb, p->q_st, p->q_sh, p->k_sb, p->k_st, p->k_sh, p->v_sb, p->v_st, p->v_sh}) if (s % 8 != 0) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k, p->v})) return rc;
    if (p->g == nullptr || p->beta == nullptr) return RWKV_ERR_NULL;
    if ((reinterpret_cast<uintptr_t>(p->g) & 1) || (reinterpret_cast<uintptr_t>(p->beta) & 1) || (reinterpret_cast<uintptr_t>(p->doc) & 3)) return RWKV_ERR_ALIGN;
    if (backward) {
        if (const int rc = check_ptrs({p->saved, p->dq, p->dk, p->dv})) return rc;
        if (p->dg == nullptr || p->dbeta == nullptr) return RWKV_ERR_NULL;
        if ((reinterpret_cast<uintptr_t>(p->dg) & 1) || (reinterpret_cast<uintptr_t>(p->dbeta) & 1) || !aligned16(p->dy) || !aligned16(p->dsT) || !aligned16(p->ds0)) return RWKV_ERR_ALIGN;
    } else {
        if (const int rc = check_ptrs({p->y, p->sT})) return rc;
        if (!aligned16(p->s0) || !aligned16(p->saved)) return RWKV_ERR_ALIGN;
    }
    if (p->saved && p->saved_bytes < rwkv_delta_saved_bytes(p->B, p->T, p->H, p->Hk, p->N)) return RWKV_ERR_WORKSPACE;
    const size_t need = rwkv_delta_workspace_bytes(p->B, p->T, p->H, p->Hk, p->N, backward);
    if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" {

size_t rwkv_delta_saved_bytes(int B, int T, int H, int Hk, int N) {
    using namespace rwkv;
    if (!delta_sizes(B, T, H, Hk, N)) return 0;
    const DeltaTiles tiles(B, T, H, N);
    return (tiles.states() + tiles.updates()) * sizeof(float);
}

size_t rwkv_delta_workspace_bytes(int B, int T, int H, int Hk, int N, int backward) {
    using namespace rwkv;
    if (!delta_sizes(B, T, H, Hk, N) || !backward) return 0;
    const DeltaTiles tiles(B, T, H, N);
    return (tiles.states() + tiles.updates() + (Hk != H ? 2 * static_cast<size_t>(B) * T * H * N : 0)) * sizeof(float);
}

int rwkv_delta_forward(void* stream, const rwkv_delta_args* args) {
    using namespace rwkv;
    if (const int rc = check_delta(args, false)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return args->dtype == RWKV_DTYPE_BF16 ? run_fwd<bf16_t>(st, *args) : run_fwd<half_t>(st, *args);
}

int rwkv_delta_backward(void* stream, const rwkv_delta_args* args) {
    using namespace rwkv;
    if (const int rc = check_delta(args, true)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return args->dtype == RWKV_DTYPE_BF16 ? run_bwd<bf16_t>(st, *args) : run_bwd<half_t>(st, *args);
}

}  // extern "C"
