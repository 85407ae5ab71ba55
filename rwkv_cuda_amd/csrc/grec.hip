// Gated linear recurrence, channel by channel: h_t = a_t h_{t-1} + u_t, y_t = h_t (the arguments are explained in rwkv_hip.h).
// Backward, with d_t the gradient of h_t:  d_t = dy_t + a_{t+1} d_{t+1};  da_t = d_t h_{t-1};  du_t = d_t.
#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

constexpr int SEG = 16;

// gate and its complement, both to fp32's accuracy
template <int GATE> DEVINL void gate_of(float w, float& a, float& rest) {
    if constexpr (GATE == RWKV_GATE_SIGMOID) {
        const float e = __expf(-fabsf(w)), s = 1.f / (1.f + e), t = e * s;
        a = w >= 0.f ? s : t;
        rest = w >= 0.f ? t : s;
        if (w != w) a = rest = w;
    } else {
        a = __expf(w);
        rest = -expm1f(w);
    }
}

template <class E, int GATE> __global__ __launch_bounds__(64) void grec_fwd_plain(const rwkv_grec_args p) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= p.C) return;
    const E* w = static_cast<const E*>(p.w) + b * p.w_sb + c;
    const E* x = static_cast<const E*>(p.x) + b * p.x_sb + c;
    E* y = static_cast<E*>(p.y) + static_cast<int64_t>(b) * p.T * p.C + c;
    const int segs = (p.T + SEG - 1) / SEG;
    float h = p.h0 ? p.h0[static_cast<int64_t>(b) * p.C + c] : 0.f;
    int last = 0;
    for (int t = 0; t < p.T; ++t) {
        if (t % SEG == 0 && p.saved) p.saved[(static_cast<int64_t>(b) * segs + t / SEG) * p.C + c] = h;
        const int doc = p.doc ? p.doc[static_cast<int64_t>(b) * p.T + t] : 0;
        if (doc >= 0) {
            float a, rest;
            gate_of<GATE>(to_f(w[t * p.w_st]), a, rest);
            const float xx = to_f(x[t * p.x_st]);
            const float prev = t > 0 && doc != last ? 0.f : h * a;
            h = prev + (p.tied ? rest * xx : xx);
        }
        y[static_cast<int64_t>(t) * p.C] = from_f<E>(doc >= 0 ? h : 0.f);
        last = doc;
    }
    p.hT[static_cast<int64_t>(b) * p.C + c] = h;
}

template <class E, int GATE> __global__ __launch_bounds__(64) void grec_bwd_plain(const rwkv_grec_args p) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= p.C) return;
    const E* w = static_cast<const E*>(p.w) + b * p.w_sb + c;
    const E* x = static_cast<const E*>(p.x) + b * p.x_sb + c;
    const int64_t row = static_cast<int64_t>(b) * p.T;
    const E* dy = static_cast<const E*>(p.dy);
    E *dw = static_cast<E*>(p.dw), *dx = static_cast<E*>(p.dx);
    const int segs = (p.T + SEG - 1) / SEG;
    float d = p.dhT ? p.dhT[static_cast<int64_t>(b) * p.C + c] : 0.f;
    for (int s = segs - 1; s >= 0; --s) {
        float before[SEG];
        float h = p.saved[(static_cast<int64_t>(b) * segs + s) * p.C + c];
#pragma unroll
        for (int i = 0; i < SEG; ++i) {
            const int t = s * SEG + i;
            before[i] = 0.f;
            if (t >= p.T) continue;
            const int doc = p.doc ? p.doc[row + t] : 0;
            if (doc < 0) continue;
            float a, rest;
            gate_of<GATE>(to_f(w[t * p.w_st]), a, rest);
            const float xx = to_f(x[t * p.x_st]);
            before[i] = p.doc && t > 0 && doc != p.doc[row + t - 1] ? 0.f : h;
            h = a * before[i] + (p.tied ? rest * xx : xx);
        }
#pragma unroll
        for (int i = SEG - 1; i >= 0; --i) {
            const int t = s * SEG + i;
            if (t >= p.T) continue;
            const int64_t at = (row + t) * p.C + c;
            const int doc = p.doc ? p.doc[row + t] : 0;
            if (doc < 0) { dw[at] = from_f<E>(0.f); dx[at] = from_f<E>(0.f); continue; }
            float a, rest;
            gate_of<GATE>(to_f(w[t * p.w_st]), a, rest);
            const float xx = to_f(x[t * p.x_st]);
            d += dy ? to_f(dy[at]) : 0.f;
            const float da = d * (p.tied ? before[i] - xx : before[i]);
            dw[at] = from_f<E>(da * a * (GATE == RWKV_GATE_SIGMOID ? rest : 1.f));
            dx[at] = from_f<E>(p.tied ? d * rest : d);
            d = p.doc && t > 0 && doc != p.doc[row + t - 1] ? 0.f : d * a;
        }
    }
    if (p.dh0) p.dh0[static_cast<int64_t>(b) * p.C + c] = d;
}

int check_grec(const rwkv_grec_args* p, bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if (p->dtype < 0 || p->dtype > RWKV_DTYPE_FP32 || p->gate < 0 || p->gate > RWKV_GATE_LOG || p->B <= 0 || p->T <= 0 || p->C <= 0 || p->B > 65535) return RWKV_ERR_SHAPE;
    if (p->w == nullptr || p->x == nullptr) return RWKV_ERR_NULL;
    if (backward ? p->dw == nullptr || p->dx == nullptr || p->saved == nullptr : p->y == nullptr || p->hT == nullptr) return RWKV_ERR_NULL;
    const uintptr_t eb = p->dtype == RWKV_DTYPE_FP32 ? 3 : 1;
    for (const void* q : {p->w, p->x, static_cast<const void*>(p->y), p->dy, static_cast<const void*>(p->dw), static_cast<const void*>(p->dx)})
        if (reinterpret_cast<uintptr_t>(q) & eb) return RWKV_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(p->h0), static_cast<const void*>(p->hT), static_cast<const void*>(p->dhT), static_cast<const void*>(p->dh0), static_cast<const void*>(p->doc)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    if (!aligned16(p->saved)) return RWKV_ERR_ALIGN;
    if (p->saved != nullptr && p->saved_bytes < rwkv_grec_saved_bytes(p->B, p->T, p->C)) return RWKV_ERR_WORKSPACE;
    if (rwkv_grec_workspace_bytes(p->B, p->T, p->C) > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < rwkv_grec_workspace_bytes(p->B, p->T, p->C)))
        return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

template <class E> int grec_run(hipStream_t st, const rwkv_grec_args& p, bool backward) {
    const dim3 grid((p.C + 63) / 64, p.B), block(64);
    const bool s = p.gate == RWKV_GATE_SIGMOID;
    if (!backward) hipLaunchKernelGGL((s ? grec_fwd_plain<E, RWKV_GATE_SIGMOID> : grec_fwd_plain<E, RWKV_GATE_LOG>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((s ? grec_bwd_plain<E, RWKV_GATE_SIGMOID> : grec_bwd_plain<E, RWKV_GATE_LOG>), grid, block, 0, st, p);
    return launch_status();
}
int grec_any(void* stream, const rwkv_grec_args* p, bool backward) {
    if (const int rc = check_grec(p, backward)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (p->dtype) {
        case RWKV_DTYPE_BF16: return grec_run<bf16_t>(st, *p, backward);
        case RWKV_DTYPE_FP16: return grec_run<half_t>(st, *p, backward);
        default: return grec_run<float>(st, *p, backward);
    }
}

}  // namespace
}  // namespace rwkv

extern "C" {

size_t rwkv_grec_saved_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0) return 0;
    return static_cast<size_t>(B) * ((T + rwkv::SEG - 1) / rwkv::SEG) * C * sizeof(float);
}
size_t rwkv_grec_workspace_bytes(int, int, int) { return 0; }
int rwkv_grec_forward(void* stream, const rwkv_grec_args* args) { return rwkv::grec_any(stream, args, false); }
int rwkv_grec_backward(void* stream, const rwkv_grec_args* args) { return rwkv::grec_any(stream, args, true); }

}  // extern "C"
