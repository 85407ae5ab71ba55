// Attention forward on the matrix cores.  A workgroup has 4 waves of 32 QT queries of one head each and walks over the keys that any of
// them sees, 64 at a time: S^T = K Q^T, one pass of the softmax with the running maximum and sum of a lane's query, O^T += V^T P^T.
#include "attn_tile.h"

namespace rwkv {
namespace {

// The maximum that weights are taken relative to follows the running one only when that has grown by 2^GROWTH: sums and weights stay far from fp32's
// and fp16's ends, and the accumulators are rarely scaled.
constexpr float GROWTH = 8.f;

template <class E, int D, int QT, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(256, QT * D > 128 ? 1 : 2) void attn_fwd(const rwkv_attn_args p, const int blocks_q, const int per_xcd) {
    constexpr int QB = 128 * QT;
    __shared__ __align__(16) char smem[4 * Plane<D>::BYTES];
    __shared__ uint8_t kind[WINDOW];
    __shared__ __align__(16) int key_doc[2][TILE];
    __shared__ int docs_lo[4], docs_hi[4];
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    const int64_t all = wide(blocks_q) * p.H * p.B;
    if (id >= all) return;
    const int bh = id / blocks_q, q0 = (blocks_q - 1 - id % blocks_q) * QB, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5;
    const lds_t lds = lds_of(smem);
    constexpr lds_t BUF = 2 * Plane<D>::BYTES;

    const E* kbase = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh;
    const E* vbase = static_cast<const E*>(p.v) + b * p.v_sb + hk * p.v_sh;
    const int* doc = DOC ? p.doc + wide(b) * p.Tk : nullptr;
    const int shift = p.Tk - p.Tq, reach = p.prefix ? min(p.prefix[b], p.Tk) - 1 : -1;

    u32x4 q[QT][D / 16];
    int lim[QT], qdoc[QT];
    float pos[QT];
    int lim_lo = INT_MAX, lim_hi = -1, dlo = INT_MAX, dhi = -1;
#pragma unroll
    for (int z = 0; z < QT; ++z) {
        const int i = q0 + (wave * QT + z) * 32 + (lane & 31);
        const bool on = i < p.Tq;
        load_rows<E, D>(q[z], static_cast<const E*>(p.q) + b * p.q_sb + (on ? i : 0) * p.q_st + h * p.q_sh, on, p.N);
        qdoc[z] = DOC && on ? doc[shift + i] : 0;
        lim[z] = !on || qdoc[z] < 0 ? -1 : (p.causal ? max(shift + i, reach) : p.Tk - 1);
        pos[z] = static_cast<float>(shift + i);
        lim_lo = min(lim_lo, lim[z]);
        lim_hi = max(lim_hi, lim[z]);
        if (on && qdoc[z] >= 0) dlo = min(dlo, qdoc[z]), dhi = max(dhi, qdoc[z]);      // (padding sees nothing: lim is below every key)
    }
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        lim_lo = min(lim_lo, __shfl_xor(lim_lo, m, 64));
        lim_hi = max(lim_hi, __shfl_xor(lim_hi, m, 64));
        dlo = min(dlo, __shfl_xor(dlo, m, 64));
        dhi = max(dhi, __shfl_xor(dhi, m, 64));
    }
    lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
    lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);
    bool uniform = true;
    if constexpr (DOC) {
        if (lane == 0) docs_lo[wave] = dlo, docs_hi[wave] = dhi;
        __syncthreads();
        dlo = min(min(docs_lo[0], docs_lo[1]), min(docs_lo[2], docs_lo[3]));
        dhi = max(max(docs_hi[0], docs_hi[1]), max(docs_hi[2], docs_hi[3]));
        uniform = dlo == dhi;
    }
    // the last key that the block's last query sees
    const int last = p.causal ? max(min(q0 + QB, p.Tq) - 1 + shift, reach) : p.Tk - 1;
    const int tiles = last / TILE + 1;

    const RowReader<D> krow(lane);
    const ColReader<D> vcol(lane);
    Stage<D, 256> ks(tid, p.N), vs(tid, p.N);
    const Scorer sc(p, h);
    const float mul = CAP || BIAS ? 1.f : sc.unit;

    f32x16 o[QT][D / 32];
    float m[QT], l[QT];
#pragma unroll
    for (int z = 0; z < QT; ++z) {
        m[z] = -INFINITY;
        l[z] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[z][d] = f32x16{};
    }

    int next_doc = -1;
    const auto load = [&](const int t) {
        const int j0 = t * TILE, rows = p.Tk - j0;
        ks.load(kbase + j0 * p.k_st, rows, static_cast<int>(p.k_st) * 2, p.N);
        vs.load(vbase + j0 * p.v_st, rows, static_cast<int>(p.v_st) * 2, p.N);
        if constexpr (DOC) next_doc = lane < rows ? doc[j0 + lane] : -1;
    };

    int par = 0;
    for (int w0 = 0; w0 < tiles; w0 += WINDOW) {
        const int w1 = min(tiles, w0 + WINDOW);
        if constexpr (DOC) {
            __syncthreads();
            classify(kind, doc, w0, w1 - w0, p.Tk, dlo, dhi, uniform, 4);
            __syncthreads();
        }
        const auto skip = [&](int t) {
            if constexpr (DOC) return next_tile(kind, t, w0, w1);
            return t;
        };
        int t = skip(w0);
        if (t < w1) load(t);
        while (t < w1) {
            const lds_t kb = lds + par * BUF, vb = kb + Plane<D>::BYTES;
            ks.store(kb);
            if constexpr (DOC) vs.store(vb, __ballot(next_doc >= 0));
            else vs.store(vb);
            if (DOC && tid < TILE) key_doc[par][tid] = next_doc;
            const int now = t, j0 = t * TILE;
            t = skip(t + 1);
            __syncthreads();
            if (t < w1) load(t);
            const int part = DOC ? kind[now - w0] : 2;
            if (j0 <= lim_hi) {
                const bool masked = part != 2 || j0 + TILE - 1 > lim_lo;
                f32x16 s[QT][2];
#pragma unroll
                for (int z = 0; z < QT; ++z) s[z][0] = s[z][1] = f32x16{};
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        const u32x4 kf = krow(kb, e, c);
#pragma unroll
                        for (int z = 0; z < QT; ++z) s[z][e] = mma<E>(kf, q[z][c], s[z][e]);
                    }
                __builtin_amdgcn_sched_barrier(0);
                u32x4 w[QT][4];
#pragma unroll
                for (int z = 0; z < QT; ++z) {
                    if constexpr (CAP || BIAS) {
                        const float dist = pos[z] - static_cast<float>(j0 + 4 * hi);
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[z][e][r] = sc.t<CAP, BIAS>(s[z][e][r], sc.squash<CAP>(s[z][e][r]), dist - (32 * e + 8 * (r >> 2) + (r & 3)));
                    }
                    if (masked) {
                        const int room = lim[z] - j0 - 4 * hi;                  // the keys are j0 + 4 hi + n
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                u32x4 kd;
                                if constexpr (DOC) kd = *reinterpret_cast<const u32x4*>(&key_doc[par][32 * e + 8 * g + 4 * hi]);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    bool on = 32 * e + 8 * g + i <= room;
                                    if constexpr (DOC) on = on && static_cast<int>(kd[i]) == qdoc[z];
                                    s[z][e][4 * g + i] = on ? s[z][e][4 * g + i] : -INFINITY;
                                }
                            }
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[z][e][r]);
                    top = fmaxf(top, other_half(top));
                    const bool grown = (top - m[z]) * mul > GROWTH;              // always at a query's first key, never while it has seen none (-inf and -inf)
                    if (__ballot(grown) != 0ull) {
                        const float to = grown ? top : m[z], f = grown ? __builtin_amdgcn_exp2f((m[z] - to) * mul) : 1.f;
                        m[z] = to;
                        l[z] *= f;
#pragma unroll
                        for (int d = 0; d < D / 32; ++d)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[z][d][r] *= f;
                    }
                    const float base = m[z] == -INFINITY ? 0.f : -m[z] * mul;
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float x = __builtin_amdgcn_exp2f(fmaf(s[z][e][r], mul, base));
                            sum += x;
                            s[z][e][r] = x;
                        }
                        w[z][2 * e] = as_operand<E>(s[z][e], 0);
                        w[z][2 * e + 1] = as_operand<E>(s[z][e], 1);
                    }
                    l[z] += sum;
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) {
                        const u32x4 vf = vcol(vb, c, d);
#pragma unroll
                        for (int z = 0; z < QT; ++z) o[z][d] = mma<E>(vf, w[z][c], o[z][d]);
                    }
            }
            par ^= 1;
        }
    }

#pragma unroll
    for (int z = 0; z < QT; ++z) {
        const int i = q0 + (wave * QT + z) * 32 + (lane & 31);
        const float sum = l[z] + other_half(l[z]), f = sum == 0.f ? 0.f : 1.f / sum;
        const bool on = i < p.Tq;
        const int64_t at = ((wide(b) * p.Tq + (on ? i : 0)) * p.H + h) * p.N;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
            store32<E>(o[z][d], f, static_cast<E*>(p.y) + at, p.y_rest ? static_cast<E*>(p.y_rest) + at : nullptr, 32 * d, p.N, on);
        if (p.lse && on && hi == 0) p.lse[(wide(b) * p.H + h) * p.Tq + i] = sum == 0.f ? -INFINITY : fmaf(m[z], mul, __builtin_amdgcn_logf(sum));
    }
}

template <class E, int D, int QT> int run(hipStream_t st, const rwkv_attn_args& p) {
    const int blocks_q = (p.Tq + 128 * QT - 1) / (128 * QT);
    const int64_t all = wide(blocks_q) * p.H * p.B, per = (all + 7) / 8;
    if (per * 8 > INT_MAX) return RWKV_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(per * 8)), block(256);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, p, blocks_q, static_cast<int>(per)); return launch_status(); };
    const auto masks = [&](auto cap, auto bias) {
        return p.doc ? go(attn_fwd<E, D, QT, decltype(cap)::value, decltype(bias)::value, true>) : go(attn_fwd<E, D, QT, decltype(cap)::value, decltype(bias)::value, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (p.cap > 0.f) return p.slopes ? masks(yes{}, yes{}) : masks(yes{}, no{});
    return p.slopes ? masks(no{}, yes{}) : masks(no{}, no{});
}
template <class E> int run_any(hipStream_t st, const rwkv_attn_args& p) {
    return p.N <= 64 ? run<E, 64, 1>(st, p) : run<E, 128, 1>(st, p);
}

}  // namespace

int launch_attn_fwd(hipStream_t st, const rwkv_attn_args& p) { return p.dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, p) : run_any<half_t>(st, p); }

}  // namespace rwkv
