// Attention with capped scores, distance bias, documents and prefixes (the arguments are explained in rwkv_hip.h).
// Backward, with p the softmax's weights, dp = dy.v and delta = dy.y:  ds = p (dp - delta) (1 - tanh^2);  dv = p^T dy;  dq = scale ds k;
// dk = scale ds^T q.
#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

constexpr int64_t L(int x) { return x; }

struct Row {                                   // what a query sees
    int pos, doc, prefix;
};
DEVINL Row row_of(const rwkv_attn_args& p, int b, int i) {
    const int pos = p.Tk - p.Tq + i;
    return {pos, p.doc ? p.doc[L(b) * p.Tk + pos] : 0, p.prefix ? p.prefix[b] : 0};
}
DEVINL bool sees(const rwkv_attn_args& p, int b, const Row& r, int j) {
    if (p.causal && j > r.pos && j >= r.prefix) return false;
    if (p.doc && (r.doc < 0 || p.doc[L(b) * p.Tk + j] != r.doc)) return false;
    return true;
}
// the score of a pair and its slope behind the cap
DEVINL float score(const rwkv_attn_args& p, float dot, int h, int pos, int j, float& slope) {
    float s = dot * p.scale;
    slope = 1.f;
    if (p.cap > 0.f) {
        const float t = tanhf(s / p.cap);
        s = p.cap * t;
        slope = 1.f - t * t;
    }
    if (p.slopes) s -= p.slopes[h] * static_cast<float>(abs(pos - j));
    return s;
}
template <class E> DEVINL float dot(const E* a, const E* b, int n) {
    float s = 0.f;
    for (int i = 0; i < n; ++i) s += to_f(a[i]) * to_f(b[i]);
    return s;
}
DEVINL float wave_max(float x) {
    for (int m = 32; m >= 1; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
    return x;
}

// one wave a query; lane = key of a tile of 64, then lane = channel
template <class E, bool BWD> __global__ __launch_bounds__(64) void attn_rows_plain(const rwkv_attn_args p, const float* delta) {
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x, hk = h / (p.H / p.Hk);
    __shared__ float w[64];
    const Row r = row_of(p, b, i);
    const E* q = static_cast<const E*>(p.q) + b * p.q_sb + i * p.q_st + h * p.q_sh;
    const E* k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh;
    const E* v = static_cast<const E*>(p.v) + b * p.v_sb + hk * p.v_sh;
    const int64_t at = ((L(b) * p.Tq + i) * p.H + h) * p.N, st = (L(b) * p.H + h) * p.Tq + i;
    const E* dy = static_cast<const E*>(p.dy) + (BWD ? at : 0);
    float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
    const float lse = BWD ? p.lse[st] : 0.f, dlt = BWD ? delta[st] : 0.f;
    for (int j0 = 0; j0 < p.Tk; j0 += 64) {
        const int j = j0 + lane;
        const bool on = j < p.Tk && sees(p, b, r, j);
        if (__ballot(on) == 0) continue;
        float x = 0.f, slope, s = -INFINITY;
        if (on) s = score(p, dot(q, k + j * p.k_st, p.N), h, r.pos, j, slope);
        float grow = 1.f;
        if constexpr (BWD) {
            if (on) x = __expf(s - lse) * (dot(dy, v + j * p.v_st, p.N) - dlt) * slope * p.scale;
        } else {
            const float top = fmaxf(m, wave_max(s));
            grow = m == -INFINITY ? 0.f : __expf(m - top);
            x = on ? __expf(s - top) : 0.f;
            l = l * grow + group_sum<64>(x);
            m = top;
        }
        w[lane] = x;
        __syncthreads();
        const E* z = BWD ? k : v;
        const int64_t zt = BWD ? p.k_st : p.v_st;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = lane + 64 * e;
            if (d >= p.N) continue;
            acc[e] *= grow;
            for (int n = 0; n < 64 && j0 + n < p.Tk; ++n)
                if (w[n] != 0.f) acc[e] += w[n] * to_f(z[(j0 + n) * zt + d]);
        }
        __syncthreads();
    }
    for (int e = 0; e < 2; ++e) {
        const int d = lane + 64 * e;
        if (d >= p.N) continue;
        if constexpr (BWD) static_cast<E*>(p.dq)[at + d] = from_f<E>(acc[e]);
        else {
            const float y = l == 0.f ? 0.f : acc[e] / l;
            const E r16 = from_f<E>(y);
            static_cast<E*>(p.y)[at + d] = r16;
            if (p.y_rest) static_cast<E*>(p.y_rest)[at + d] = from_f<E>(y - to_f(r16));
        }
    }
    if (!BWD && lane == 0 && p.lse) p.lse[st] = l == 0.f ? -INFINITY : m + __logf(l);
}

// one wave a key; lane = query of a tile of 64, then lane = channel
template <class E> __global__ __launch_bounds__(64) void attn_keys_plain(const rwkv_attn_args p, const float* delta) {
    const int j = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, lane = threadIdx.x, G = p.H / p.Hk;
    __shared__ float w[64], w2[64];
    const E* k = static_cast<const E*>(p.k) + b * p.k_sb + j * p.k_st + hk * p.k_sh;
    const E* v = static_cast<const E*>(p.v) + b * p.v_sb + j * p.v_st + hk * p.v_sh;
    float gk[2] = {0.f, 0.f}, gv[2] = {0.f, 0.f};
    for (int h = hk * G; h < hk * G + G; ++h) {
        const E* q = static_cast<const E*>(p.q) + b * p.q_sb + h * p.q_sh;
        const E* dy = static_cast<const E*>(p.dy) + (L(b) * p.Tq * p.H + h) * p.N;
        for (int i0 = 0; i0 < p.Tq; i0 += 64) {
            const int i = i0 + lane;
            const Row r = i < p.Tq ? row_of(p, b, i) : Row{0, -1, 0};
            const bool on = i < p.Tq && sees(p, b, r, j);
            if (__ballot(on) == 0) continue;
            float x = 0.f, z = 0.f;
            if (on) {
                float slope;
                const int64_t st = (L(b) * p.H + h) * p.Tq + i;
                const float s = score(p, dot(q + i * p.q_st, k, p.N), h, r.pos, j, slope);
                x = __expf(s - p.lse[st]);
                z = x * (dot(dy + L(i) * p.H * p.N, v, p.N) - delta[st]) * slope * p.scale;
            }
            w[lane] = x;
            w2[lane] = z;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = lane + 64 * e;
                if (d >= p.N) continue;
                for (int n = 0; n < 64 && i0 + n < p.Tq; ++n) {
                    if (w[n] != 0.f) gv[e] += w[n] * to_f(dy[L(i0 + n) * p.H * p.N + d]);
                    if (w2[n] != 0.f) gk[e] += w2[n] * to_f(q[(i0 + n) * p.q_st + d]);
                }
            }
            __syncthreads();
        }
    }
    for (int e = 0; e < 2; ++e) {
        const int d = lane + 64 * e;
        if (d >= p.N) continue;
        const int64_t at = ((L(b) * p.Tk + j) * p.Hk + hk) * p.N + d;
        static_cast<E*>(p.dk)[at] = from_f<E>(gk[e]);
        static_cast<E*>(p.dv)[at] = from_f<E>(gv[e]);
    }
}

// delta = sum over the channels of dy y, y to twice its type's accuracy
template <class E> __global__ __launch_bounds__(64) void attn_delta_plain(const rwkv_attn_args p, float* delta) {
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
    const int64_t at = ((L(b) * p.Tq + i) * p.H + h) * p.N;
    float s = 0.f;
    for (int d = lane; d < p.N; d += 64)
        s += to_f(static_cast<const E*>(p.dy)[at + d]) * (to_f(static_cast<const E*>(p.y)[at + d]) + to_f(static_cast<const E*>(p.y_rest)[at + d]));
    s = group_sum<64>(s);
    if (lane == 0) delta[(L(b) * p.H + h) * p.Tq + i] = s;
}

bool multiples_of_8(std::initializer_list<int64_t> xs) {
    for (const int64_t x : xs) if (x % 8 != 0) return false;
    return true;
}
int check_attn(const rwkv_attn_args* p, bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->Tq <= 0 || p->Tk < p->Tq || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 ||
        p->N <= 0 || p->N > 128 || p->N % 8 != 0 || p->B > 65535 || p->H > 65535 || !(p->scale > 0.f) || !(p->cap >= 0.f) || (p->prefix != nullptr && !p->causal)) return RWKV_ERR_SHAPE;
    if (!multiples_of_8({p->q_sb, p->q_st, p->q_sh, p->k_sb, p->k_st, p->k_sh, p->v_sb, p->v_st, p->v_sh})) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k, p->v, p->y})) return rc;
    if (backward) {
        if (const int rc = check_ptrs({p->dy, p->dq, p->dk, p->dv, p->y_rest})) return rc;
        if (p->lse == nullptr) return RWKV_ERR_NULL;
        if (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < rwkv_attn_backward_workspace_bytes(p->B, p->Tq, p->H)) return RWKV_ERR_WORKSPACE;
    } else if (!aligned16(p->y_rest)) return RWKV_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(p->slopes), static_cast<const void*>(p->doc), static_cast<const void*>(p->prefix), static_cast<const void*>(p->lse)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    return RWKV_OK;
}

template <class E> int attn_run(hipStream_t st, const rwkv_attn_args& p, bool backward) {
    const dim3 rows(p.Tq, p.H, p.B), block(64);
    float* delta = static_cast<float*>(p.workspace);
    if (!backward) {
        return launch_attn_fwd(st, p);
    } else {
        hipLaunchKernelGGL((attn_delta_plain<E>), rows, block, 0, st, p, delta);
        hipLaunchKernelGGL((attn_rows_plain<E, true>), rows, block, 0, st, p, delta);
        hipLaunchKernelGGL((attn_keys_plain<E>), dim3(p.Tk, p.Hk, p.B), block, 0, st, p, delta);
    }
    return launch_status();
}
int attn_any(void* stream, const rwkv_attn_args* p, bool backward) {
    if (const int rc = check_attn(p, backward)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return p->dtype == RWKV_DTYPE_BF16 ? attn_run<bf16_t>(st, *p, backward) : attn_run<half_t>(st, *p, backward);
}

}  // namespace
}  // namespace rwkv

extern "C" {

size_t rwkv_attn_backward_workspace_bytes(int B, int Tq, int H) {
    if (B <= 0 || Tq <= 0 || H <= 0) return 0;
    return static_cast<size_t>(B) * Tq * H * sizeof(float);
}
int rwkv_attn_forward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, false); }
int rwkv_attn_backward(void* stream, const rwkv_attn_args* args) { return rwkv::attn_any(stream, args, true); }

}  // extern "C"
