// Gated delta rule (the arguments are explained in rwkv_hip.h):  S = e^g S;  u = beta (v - S^T k);  S += k u^T;  y = scale S^T q.
//
// Token by token: the columns of the state (its value channels) do not depend on each other, so a workgroup keeps 32 of them in registers, a thread
// four columns of every 32nd row.  Both sums over the rows, S^T k and S^T q, are made from the state before the update, y = scale (e^g S^T q + (q.k) u), so that a token
// costs one exchange between the waves.
#include <algorithm>
#include <climits>

#include "delta.h"

namespace rwkv {
namespace {

template <class E, int ROWS>
__global__ __launch_bounds__(256) void delta_steps(const rwkv_delta_args p, float* states) {
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
        if (states && t % DELTA_CHUNK == 0) {
            float* to = states + (head * ((p.T + DELTA_CHUNK - 1) / DELTA_CHUNK) + t / DELTA_CHUNK) * N * N;
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                if (on && r0 + 32 * i < N) *reinterpret_cast<f32x4*>(to + (r0 + 32 * i) * N + c0) = s[i];
        }
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

// The backward, chunk by chunk from the last: a workgroup a head, matrices in memory, sums in fp32.
constexpr int C = DELTA_CHUNK;
template <class A, class B, class O> DEVINL void product(const int M, const int Nn, const int K, A a, B b, O out) {
    for (int x = threadIdx.x; x < M * Nn; x += 256) {
        const int i = x / Nn, j = x % Nn;
        float s = 0.f;
        for (int k = 0; k < K; ++k) s = fmaf(a(i, k), b(k, j), s);
        out(i, j, s);
    }
    __syncthreads();
}
__host__ __device__ inline size_t scratch_floats(int N) { return static_cast<size_t>(N) * N + 8 * C * N + 6 * C * C; }

template <class E>
__global__ __launch_bounds__(256) void delta_back(const rwkv_delta_args p, const float* states, float* scratch, float* dq_of, float* dk_of) {
    const int h = blockIdx.x, b = blockIdx.y, hk = h / (p.H / p.Hk), tid = threadIdx.x, N = p.N, T = p.T, chunks = (T + C - 1) / C;
    const int64_t head = wide(b) * p.H + h;
    float* at = scratch + head * scratch_floats(N);
    const auto take = [&](int n) { float* x = at; at += n; return x; };
    float *dS = take(N * N), *K = take(C * N), *Q = take(C * N), *V = take(C * N), *dY = take(C * N), *U = take(C * N), *dZ = take(C * N), *X = take(C * N), *Z = take(C * N);
    float *A = take(C * C), *P = take(C * C), *I = take(C * C), *KK = take(C * C), *dP = take(C * C), *dA = take(C * C);
    __shared__ float G[C], lo[C], bt[C], enter[C], leave[C], ga[C], gb[C];
    __shared__ int part[C], real[C], cut[C];
    __shared__ float whole, sum[256];
    for (int x = tid; x < N * N; x += 256) dS[x] = p.dsT ? p.dsT[head * N * N + x] : 0.f;
    for (int c = chunks - 1; c >= 0; --c) {
        const float* S = states + (head * chunks + c) * N * N;
        const int t0 = c * C;
        if (tid < C) {
            const DeltaToken token = delta_token(p.doc, wide(b) * T, t0 + tid, T);
            real[tid] = token.real;
            const float lg = token.real ? to_f(static_cast<const E*>(p.g)[b * p.g_sb + (t0 + tid) * p.g_st + h]) : 0.f;
            cut[tid] = token.cut || lg < DELTA_NONE;
            lo[tid] = cut[tid] ? 0.f : lg;
            bt[tid] = token.real ? to_f(static_cast<const E*>(p.beta)[b * p.beta_sb + (t0 + tid) * p.beta_st + h]) : 0.f;
        }
        __syncthreads();
        if (tid == 0) {
            double s = 0;
            double all[C];
            for (int i = 0, n = 0; i < C; ++i) { s += lo[i]; n += cut[i]; all[i] = s; part[i] = n; }
            for (int i = 0; i < C; ++i) {
                G[i] = static_cast<float>(all[i]);
                enter[i] = part[i] == 0 ? expf(G[i]) : 0.f;
                leave[i] = part[i] == part[C - 1] ? expf(static_cast<float>(all[C - 1] - all[i])) : 0.f;
            }
            whole = enter[C - 1];
        }
        for (int x = tid; x < C * N; x += 256) {
            const int i = x / N, n = x % N;
            const int64_t t = t0 + i;
            const bool ok = real[i];
            K[x] = ok ? to_f(static_cast<const E*>(p.k)[b * p.k_sb + t * p.k_st + hk * p.k_sh + n]) : 0.f;
            Q[x] = ok ? to_f(static_cast<const E*>(p.q)[b * p.q_sb + t * p.q_st + hk * p.q_sh + n]) : 0.f;
            V[x] = ok ? to_f(static_cast<const E*>(p.v)[b * p.v_sb + t * p.v_st + h * p.v_sh + n]) : 0.f;
            dY[x] = ok && p.dy ? to_f(static_cast<const E*>(p.dy)[((wide(b) * T + t) * p.H + h) * N + n]) : 0.f;
        }
        __syncthreads();
        const auto decay = [&](int i, int j) { return part[i] == part[j] ? expf(G[i] - G[j]) : 0.f; };
        product(C, C, N, [&](int i, int k) { return K[i * N + k]; }, [&](int k, int j) { return K[j * N + k]; },
                [&](int i, int j, float s) { KK[i * C + j] = s; A[i * C + j] = i > j ? bt[i] * decay(i, j) * s : 0.f; });
        product(C, C, N, [&](int i, int k) { return Q[i * N + k]; }, [&](int k, int j) { return K[j * N + k]; },
                [&](int i, int j, float s) { P[i * C + j] = s; });
        if (tid < C) {                                          // column tid of the inverse of I + A
            for (int i = 0; i < C; ++i) {
                float s = i == tid ? 1.f : 0.f;
                for (int j = tid; j < i; ++j) s = fmaf(-A[i * C + j], I[j * C + tid], s);
                I[i * C + tid] = i < tid ? 0.f : s;
            }
        }
        __syncthreads();
        product(C, N, N, [&](int i, int k) { return K[i * N + k]; }, [&](int k, int j) { return S[k * N + j]; }, [&](int i, int j, float s) { Z[i * N + j] = bt[i] * (V[i * N + j] - enter[i] * s); });
        product(C, N, C, [&](int i, int k) { return I[i * C + k]; }, [&](int k, int j) { return Z[k * N + j]; }, [&](int i, int j, float s) { U[i * N + j] = s; });
        product(C, N, N, [&](int i, int k) { return K[i * N + k]; }, [&](int k, int j) { return dS[k * N + j]; }, [&](int i, int j, float s) { X[i * N + j] = leave[i] * s; });
        product(C, N, C, [&](int j, int i) { return i >= j ? p.scale * decay(i, j) * P[i * C + j] : 0.f; }, [&](int i, int n) { return dY[i * N + n]; }, [&](int j, int n, float s) { X[j * N + n] += s; });
        product(C, N, C, [&](int i, int k) { return I[k * C + i]; }, [&](int k, int j) { return X[k * N + j]; }, [&](int i, int j, float s) { dZ[i * N + j] = s; });
        product(C, C, N, [&](int i, int n) { return dY[i * N + n]; }, [&](int n, int j) { return U[j * N + n]; }, [&](int i, int j, float s) { dP[i * C + j] = i >= j ? p.scale * decay(i, j) * s : 0.f; });
        product(C, C, N, [&](int i, int n) { return dZ[i * N + n]; }, [&](int n, int j) { return U[j * N + n]; }, [&](int i, int j, float s) { dA[i * C + j] = i > j ? -decay(i, j) * s : 0.f; });
        // the parts of dq and dk that go through the states: Z = enter dZ S^T, X = leave U dS^T
        product(C, N, N, [&](int i, int n) { return dZ[i * N + n]; }, [&](int n, int k) { return S[k * N + n]; }, [&](int i, int k, float s) { Z[i * N + k] = enter[i] * s; });
        product(C, N, N, [&](int i, int n) { return U[i * N + n]; }, [&](int n, int k) { return dS[k * N + n]; }, [&](int i, int k, float s) { X[i * N + k] = leave[i] * s; });
        if (tid < C) {
            const int i = tid;
            float db = 0.f, after = 0.f, before = 0.f;
            for (int n = 0; n < N; ++n) {
                db += dZ[i * N + n] * V[i * N + n] - Z[i * N + n] * K[i * N + n];
                after -= bt[i] * Z[i * N + n] * K[i * N + n];
                before += X[i * N + n] * K[i * N + n];
            }
            for (int j = 0; j < C; ++j) {
                db += dA[i * C + j] * KK[i * C + j];
                if (j != i) after += dP[i * C + j] * P[i * C + j] + dA[i * C + j] * bt[i] * KK[i * C + j] - dP[j * C + i] * P[j * C + i] - dA[j * C + i] * bt[j] * KK[j * C + i];
            }
            ga[i] = after;
            gb[i] = before;
            if (real[i]) static_cast<E*>(p.dbeta)[(wide(b) * T + t0 + i) * p.H + h] = from_f<E>(db);
            else if (t0 + i < T) static_cast<E*>(p.dbeta)[(wide(b) * T + t0 + i) * p.H + h] = from_f<E>(0.f);
        }
        float mine = 0.f;
        for (int x = tid; x < N * N; x += 256) mine += dS[x] * S[x];
        sum[tid] = mine;
        __syncthreads();
        // dq: the state's part, with its share of the gates' gradients, then the pairs'
        const auto row = [&](float* to, int i, int n) -> float& { return to[((wide(b) * T + t0 + i) * p.H + h) * N + n]; };
        product(C, N, N, [&](int i, int n) { return dY[i * N + n]; }, [&](int n, int k) { return S[k * N + n]; }, [&](int i, int k, float s) { if (t0 + i < T) row(dq_of, i, k) = p.scale * enter[i] * s; });
        if (tid < C && t0 + tid < T) for (int n = 0; n < N; ++n) ga[tid] += Q[tid * N + n] * row(dq_of, tid, n);
        __syncthreads();
        if (tid == 0) {
            float all = 0.f;
            for (int i = 0; i < 256; ++i) all += sum[i];
            all *= whole;
            float a = 0.f, f = 0.f;
            for (int i = C - 1; i >= 0; --i) { a += ga[i]; ga[i] = a; }
            for (int i = 0; i < C; ++i) { const float x = gb[i]; gb[i] = ga[i] + f + all; f += x; }
        }
        __syncthreads();
        if (tid < C && t0 + tid < T) static_cast<E*>(p.dg)[(wide(b) * T + t0 + tid) * p.H + h] = from_f<E>(real[tid] && !cut[tid] ? gb[tid] : 0.f);
        product(C, N, C, [&](int i, int j) { return dP[i * C + j]; }, [&](int j, int n) { return K[j * N + n]; },
                [&](int i, int n, float s) { if (t0 + i < T) row(dq_of, i, n) = real[i] ? row(dq_of, i, n) + s : 0.f; });
        product(C, N, C, [&](int j, int i) { return dP[i * C + j]; }, [&](int i, int n) { return Q[i * N + n]; }, [&](int i, int n, float s) { X[i * N + n] += s - bt[i] * Z[i * N + n]; });
        product(C, N, C, [&](int i, int j) { return dA[i * C + j] * bt[i] + dA[j * C + i] * bt[j]; }, [&](int j, int n) { return K[j * N + n]; },
                [&](int i, int n, float s) { if (t0 + i < T) row(dk_of, i, n) = real[i] ? X[i * N + n] + s : 0.f; });
        for (int x = tid; x < C * N; x += 256)
            if (t0 + x / N < T) static_cast<E*>(p.dv)[((wide(b) * T + t0 + x / N) * p.H + h) * N + x % N] = from_f<E>(bt[x / N] * dZ[x]);
        product(N, N, C, [&](int k, int i) { return p.scale * enter[i] * Q[i * N + k]; }, [&](int i, int n) { return dY[i * N + n]; }, [&](int k, int n, float s) { dS[k * N + n] = whole * dS[k * N + n] + s; });
        product(N, N, C, [&](int k, int i) { return bt[i] * enter[i] * K[i * N + k]; }, [&](int i, int n) { return dZ[i * N + n]; }, [&](int k, int n, float s) { dS[k * N + n] -= s; });
    }
    if (p.ds0)
        for (int x = tid; x < N * N; x += 256) p.ds0[head * N * N + x] = dS[x];
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

// Few tokens go one by one: a chunk costs the same whatever it holds.
constexpr int FEW = 8;
template <class E> int run_fwd(hipStream_t st, const rwkv_delta_args& p) {
    if (p.saved == nullptr && p.T > FEW) return launch_delta_fwd(st, p);
    const dim3 grid((p.N + 31) / 32, p.H, p.B);
    if (p.N <= 64) hipLaunchKernelGGL((delta_steps<E, 2>), grid, dim3(256), 0, st, p, static_cast<float*>(p.saved));
    else hipLaunchKernelGGL((delta_steps<E, 4>), grid, dim3(256), 0, st, p, static_cast<float*>(p.saved));
    return launch_status();
}
template <class E> int run_bwd(hipStream_t st, const rwkv_delta_args& p) {
    float* ws = static_cast<float*>(p.workspace);
    const size_t n = static_cast<size_t>(p.B) * p.T * p.H * p.N;
    float *dq = ws, *dk = ws + n, *scratch = ws + 2 * n;
    hipLaunchKernelGGL(delta_back<E>, dim3(p.H, p.B), dim3(256), 0, st, p, static_cast<const float*>(p.saved), scratch, dq, dk);
    hipLaunchKernelGGL(delta_sum<E>, dim3(2048), dim3(256), 0, st, p, dq, dk);
    return launch_status();
}

// The sizes that the kernels hold for.
bool delta_sizes(int B, int T, int H, int Hk, int N) {
    return B > 0 && T > 0 && H > 0 && Hk > 0 && H % Hk == 0 && N > 0 && N <= 128 && N % 8 == 0 && B <= 65535 && H <= 65535 && T <= INT_MAX - 65536;
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
    return static_cast<size_t>(B) * H * ((T + DELTA_CHUNK - 1) / DELTA_CHUNK) * N * N * sizeof(float);
}

size_t rwkv_delta_workspace_bytes(int B, int T, int H, int Hk, int N, int backward) {
    using namespace rwkv;
    if (!delta_sizes(B, T, H, Hk, N) || !backward) return 0;
    return (2 * static_cast<size_t>(B) * T * H * N + static_cast<size_t>(B) * H * scratch_floats(N)) * sizeof(float);
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
