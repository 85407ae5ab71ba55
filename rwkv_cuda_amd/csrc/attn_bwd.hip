// Attention backward on the matrix cores, without atomics: the weights are made again from the forward's lse, once by the workgroups that own
// queries (dQ: three products a pair) and once by those that own keys (dK, dV: four), each sum in one wave's registers in a fixed order.
#include "attn_tile.h"

namespace rwkv {
namespace {

// fp16 weights as operands are 2^SHIFT times as large: those of thousands of keys would fall below its normal numbers
template <class E> constexpr float SHIFT = std::is_same_v<E, bf16_t> ? 0.f : 8.f;
template <class E> constexpr float UNSHIFT = std::is_same_v<E, bf16_t> ? 1.f : 1.f / 256.f;

// delta = sum over the channels of dy y, y as the forward had it before it was rounded; a row has D / 8 lanes
template <class E, int D> __global__ __launch_bounds__(256) void attn_delta(const rwkv_attn_args p, float* delta) {
    constexpr int LANES = D / 8;
    const int64_t row = (blockIdx.x * wide(256) + threadIdx.x) / LANES, rows = wide(p.B) * p.Tq * p.H;
    const int d = threadIdx.x % LANES * 8;
    float s = 0.f;
    if (row < rows && d < p.N) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.dy) + row * p.N + d), y = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.y) + row * p.N + d),
                    z = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.y_rest) + row * p.N + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s = fmaf(unpack_lo<E>(a[i]), unpack_lo<E>(y[i]) + unpack_lo<E>(z[i]), s);
            s = fmaf(unpack_hi<E>(a[i]), unpack_hi<E>(y[i]) + unpack_hi<E>(z[i]), s);
        }
    }
    s = group_sum<LANES>(s);
    if (row < rows && d == 0) {
        const int h = row % p.H;
        const int64_t bi = row / p.H;
        delta[(bi / p.Tq * p.H + h) * p.Tq + bi % p.Tq] = s;
    }
}

// dQ: 4 waves of 32 queries over the keys that any of them sees; S^T = K Q^T and dP^T = V dY^T, dQ^T += K^T dS^T
template <class E, int D, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(256, 2) void attn_dq(const rwkv_attn_args p, const float* delta, const int blocks_q, const int per_xcd) {
    constexpr int QB = 128;
    __shared__ __align__(16) char smem[4 * Plane<D>::BYTES];
    __shared__ uint8_t kind[WINDOW];
    __shared__ __align__(16) int key_doc[2][TILE];
    __shared__ int docs_lo[4], docs_hi[4];
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (id >= wide(blocks_q) * p.H * p.B) return;
    const int bh = id / blocks_q, q0 = (blocks_q - 1 - id % blocks_q) * QB, b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5;
    const lds_t lds = lds_of(smem);
    constexpr lds_t BUF = 2 * Plane<D>::BYTES;

    const E* kbase = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh;
    const E* vbase = static_cast<const E*>(p.v) + b * p.v_sb + hk * p.v_sh;
    const int* doc = DOC ? p.doc + wide(b) * p.Tk : nullptr;
    const int shift = p.Tk - p.Tq, reach = p.prefix ? min(p.prefix[b], p.Tk) - 1 : -1;

    const int i = q0 + wave * 32 + (lane & 31);
    const bool real = i < p.Tq;
    const int64_t row = ((wide(b) * p.Tq + (real ? i : 0)) * p.H + h) * p.N;
    u32x4 q[D / 16], dy[D / 16];
    load_rows<E, D>(q, static_cast<const E*>(p.q) + b * p.q_sb + (real ? i : 0) * p.q_st + h * p.q_sh, real, p.N);
    load_rows<E, D>(dy, static_cast<const E*>(p.dy) + row, real, p.N);
    const int qdoc = DOC && real ? doc[shift + i] : 0;
    const int lim = !real || qdoc < 0 ? -1 : (p.causal ? max(shift + i, reach) : p.Tk - 1);
    const float pos = static_cast<float>(shift + i);
    const int64_t stat = (wide(b) * p.H + h) * p.Tq + (real ? i : 0);
    const float lse = lim >= 0 ? p.lse[stat] : INFINITY, dlt = lim >= 0 ? delta[stat] : 0.f;
    int lim_lo = lim, lim_hi = lim, dlo = real && qdoc >= 0 ? qdoc : INT_MAX, dhi = real ? qdoc : -1;
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
    const int last = p.causal ? max(min(q0 + QB, p.Tq) - 1 + shift, reach) : p.Tk - 1;
    const int tiles = last / TILE + 1;

    const RowReader<D> rows(lane);
    const ColReader<D> cols(lane);
    Stage<D, 256> ks(tid, p.N), vs(tid, p.N);
    const Scorer sc(p, h);
    const float mul = CAP || BIAS ? 1.f : sc.unit;
    f32x16 g[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) g[d] = f32x16{};

    int next_doc = -1;
    const auto load = [&](const int t) {
        const int j0 = t * TILE, n = p.Tk - j0;
        ks.load(kbase + j0 * p.k_st, n, static_cast<int>(p.k_st) * 2, p.N);
        vs.load(vbase + j0 * p.v_st, n, static_cast<int>(p.v_st) * 2, p.N);
        if constexpr (DOC) next_doc = lane < n ? doc[j0 + lane] : -1;
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
            if constexpr (DOC) ks.store(kb, __ballot(next_doc >= 0));
            else ks.store(kb);
            vs.store(vb);
            if (DOC && tid < TILE) key_doc[par][tid] = next_doc;
            const int now = t, j0 = t * TILE;
            t = skip(t + 1);
            __syncthreads();
            if (t < w1) load(t);
            const int part = DOC ? kind[now - w0] : 2;
            if (j0 <= lim_hi) {
                const bool masked = part != 2 || j0 + TILE - 1 > lim_lo;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) s = mma<E>(rows(kb, e, c), q[c], s);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) dp = mma<E>(rows(vb, e, c), dy[c], dp);
                    __builtin_amdgcn_sched_barrier(0);
                    const float dist = pos - static_cast<float>(j0 + 4 * hi + 32 * e);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float x = s[r], sq = sc.squash<CAP>(x);
                        const float w = __builtin_amdgcn_exp2f(fmaf(sc.t<CAP, BIAS>(x, sq, dist - (8 * (r >> 2) + (r & 3))), mul, -lse));
                        float ds = w * (dp[r] - dlt);
                        if constexpr (CAP) ds *= 4.f * sq * (1.f - sq);
                        s[r] = ds;
                    }
                    if (masked) {
                        const int room = lim - j0 - 4 * hi - 32 * e;
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            u32x4 kd;
                            if constexpr (DOC) kd = *reinterpret_cast<const u32x4*>(&key_doc[par][32 * e + 8 * n + 4 * hi]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                bool on = 8 * n + r <= room;
                                if constexpr (DOC) on = on && static_cast<int>(kd[r]) == qdoc;
                                s[4 * n + r] = on ? s[4 * n + r] : 0.f;
                            }
                        }
                    }
                    const u32x4 w[2] = {as_operand<E>(s, 0), as_operand<E>(s, 1)};
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int d = 0; d < D / 32; ++d) g[d] = mma<E>(cols(kb, 2 * e + c, d), w[c], g[d]);
                }
            }
            par ^= 1;
        }
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store32<E>(g[d], p.scale, static_cast<E*>(p.dq) + row, nullptr, 32 * d, p.N, real);
}

// dK, dV: 4 waves of 32 keys over the queries, of all heads that share them, that see any of them; S = Q K^T and dP = dY V^T,
// dV^T += dY^T P, dK^T += Q^T dS
template <class E, int D, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(256, D == 128 ? 1 : 2) void attn_dkv(const rwkv_attn_args p, const float* delta, const int blocks_k, const int per_xcd) {
    constexpr int KB = 128;
    __shared__ __align__(16) char smem[4 * Plane<D>::BYTES];
    __shared__ uint8_t kind[WINDOW];
    __shared__ __align__(16) int row_doc[2][TILE];
    __shared__ __align__(16) float row_lse[2][TILE], row_delta[2][TILE];
    __shared__ int docs_lo[4], docs_hi[4];
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (id >= wide(blocks_k) * p.Hk * p.B) return;
    const int bh = id / blocks_k, k0 = id % blocks_k * KB, b = bh / p.Hk, hk = bh % p.Hk, G = p.H / p.Hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5;
    const lds_t lds = lds_of(smem);
    constexpr lds_t BUF = 2 * Plane<D>::BYTES;

    const int shift = p.Tk - p.Tq, reach = p.prefix ? min(p.prefix[b], p.Tk) : 0;
    const int* doc = DOC ? p.doc + wide(b) * p.Tk : nullptr;
    const int j = k0 + wave * 32 + (lane & 31);
    const bool real = j < p.Tk;
    u32x4 k[D / 16], v[D / 16];
    load_rows<E, D>(k, static_cast<const E*>(p.k) + b * p.k_sb + (real ? j : 0) * p.k_st + hk * p.k_sh, real, p.N);
    load_rows<E, D>(v, static_cast<const E*>(p.v) + b * p.v_sb + (real ? j : 0) * p.v_st + hk * p.v_sh, real, p.N);
    const int kdoc = DOC && real ? doc[j] : 0;
    const int from = kdoc < 0 ? INT_MAX : (!p.causal || j < reach ? 0 : j);            // the first position that sees the key; none that sees padding
    int from_lo = real ? from : INT_MAX, from_hi = real ? from : 0, dlo = real && kdoc >= 0 ? kdoc : INT_MAX, dhi = real ? kdoc : -1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        from_lo = min(from_lo, __shfl_xor(from_lo, m, 64));
        from_hi = max(from_hi, __shfl_xor(from_hi, m, 64));
        dlo = min(dlo, __shfl_xor(dlo, m, 64));
        dhi = max(dhi, __shfl_xor(dhi, m, 64));
    }
    from_lo = __builtin_amdgcn_readfirstlane(from_lo);
    from_hi = __builtin_amdgcn_readfirstlane(from_hi);
    bool uniform = true;
    if constexpr (DOC) {
        if (lane == 0) docs_lo[wave] = dlo, docs_hi[wave] = dhi;
        __syncthreads();
        dlo = min(min(docs_lo[0], docs_lo[1]), min(docs_lo[2], docs_lo[3]));
        dhi = max(max(docs_hi[0], docs_hi[1]), max(docs_hi[2], docs_hi[3]));
        uniform = dlo == dhi;
    }
    const int first = !p.causal || k0 < reach ? 0 : max(0, k0 - shift) / TILE, tiles = (p.Tq + TILE - 1) / TILE;

    const RowReader<D> rows(lane);
    const ColReader<D> cols(lane);
    Stage<D, 256> qs(tid, p.N), ys(tid, p.N);
    f32x16 gk[D / 32], gv[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) gk[d] = gv[d] = f32x16{};

    int next_doc = -1;
    float next_lse = 0.f, next_delta = 0.f;
    const auto load = [&](const int h, const int t) {
        const int i0 = t * TILE, n = p.Tq - i0;
        qs.load(static_cast<const E*>(p.q) + b * p.q_sb + i0 * p.q_st + h * p.q_sh, n, static_cast<int>(p.q_st) * 2, p.N);
        ys.load(static_cast<const E*>(p.dy) + ((wide(b) * p.Tq + i0) * p.H + h) * p.N, n, p.H * p.N * 2, p.N);
        const bool on = tid < TILE && tid < n;
        if (tid < TILE) {
            const int64_t stat = (wide(b) * p.H + h) * p.Tq + (on ? i0 + tid : 0);
            next_lse = p.lse[stat];
            next_delta = delta[stat] * UNSHIFT<E>;
            if (!on || next_lse == -INFINITY) next_lse = INFINITY, next_delta = 0.f;     // a row that is not there or sees nothing: weights of 0
            next_lse -= SHIFT<E>;
        }
        if constexpr (DOC) next_doc = lane < n ? doc[shift + i0 + lane] : -1;
    };
    int par = 0;
    for (int w0 = first; w0 < tiles; w0 += WINDOW) {
        const int w1 = min(tiles, w0 + WINDOW);
        if constexpr (DOC) {
            __syncthreads();
            classify(kind, doc + shift, w0, w1 - w0, p.Tq, dlo, dhi, uniform, 4);
            __syncthreads();
        }
        const auto skip = [&](int t) {
            if constexpr (DOC) return next_tile(kind, t, w0, w1);
            return t;
        };
        const int begin = skip(w0);
        int t = begin, h = hk * G;
        if (t < w1) load(h, t);
        while (t < w1) {
            const lds_t qb = lds + par * BUF, yb = qb + Plane<D>::BYTES;
            if constexpr (DOC) qs.store(qb, __ballot(next_doc >= 0)), ys.store(yb, __ballot(next_doc >= 0));
            else qs.store(qb), ys.store(yb);
            if (tid < TILE) {
                row_lse[par][tid] = next_lse;
                row_delta[par][tid] = next_delta;
                if (DOC) row_doc[par][tid] = next_doc;
            }
            const int now = t, i0 = t * TILE;
            const Scorer sc(p, h);
            const float mul = CAP || BIAS ? 1.f : sc.unit;
            t = skip(t + 1);
            if (t >= w1 && h + 1 < hk * G + G) t = begin, ++h;
            __syncthreads();
            if (t < w1) load(h, t);
            const int part = DOC ? kind[now - w0] : 2;
            if (shift + i0 + TILE - 1 >= from_lo) {
                const bool masked = part != 2 || shift + i0 < from_hi;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) s = mma<E>(rows(qb, e, c), k[c], s);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) dp = mma<E>(rows(yb, e, c), v[c], dp);
                    __builtin_amdgcn_sched_barrier(0);
                    const float dist = static_cast<float>(shift + i0 + 4 * hi + 32 * e) - static_cast<float>(j);
                    const int need = from - shift - i0 - 4 * hi - 32 * e;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float4 ls = *reinterpret_cast<const float4*>(&row_lse[par][32 * e + 8 * n + 4 * hi]), dl = *reinterpret_cast<const float4*>(&row_delta[par][32 * e + 8 * n + 4 * hi]);
                        const float lse[4] = {ls.x, ls.y, ls.z, ls.w}, dlt[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int at = 4 * n + r;
                            const float x = s[at], sq = sc.squash<CAP>(x);
                            const float w = __builtin_amdgcn_exp2f(fmaf(sc.t<CAP, BIAS>(x, sq, dist + (8 * n + r)), mul, -lse[r]));
                            float ds = w * fmaf(dp[at], UNSHIFT<E>, -dlt[r]);
                            if constexpr (CAP) ds *= 4.f * sq * (1.f - sq);
                            s[at] = w;
                            dp[at] = ds;
                        }
                    }
                    if (masked) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            u32x4 rd;
                            if constexpr (DOC) rd = *reinterpret_cast<const u32x4*>(&row_doc[par][32 * e + 8 * n + 4 * hi]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                bool on = 8 * n + r >= need;
                                if constexpr (DOC) on = on && static_cast<int>(rd[r]) == kdoc;
                                s[4 * n + r] = on ? s[4 * n + r] : 0.f;
                                dp[4 * n + r] = on ? dp[4 * n + r] : 0.f;
                            }
                        }
                    }
                    const u32x4 w[2] = {as_operand<E>(s, 0), as_operand<E>(s, 1)}, ds[2] = {as_operand<E>(dp, 0), as_operand<E>(dp, 1)};
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int d = 0; d < D / 32; ++d) {
                            gv[d] = mma<E>(cols(yb, 2 * e + c, d), w[c], gv[d]);
                            gk[d] = mma<E>(cols(qb, 2 * e + c, d), ds[c], gk[d]);
                        }
                }
            }
            par ^= 1;
        }
    }
    const int64_t row = ((wide(b) * p.Tk + (real ? j : 0)) * p.Hk + hk) * p.N;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        store32<E>(gk[d], p.scale, static_cast<E*>(p.dk) + row, nullptr, 32 * d, p.N, real);
        store32<E>(gv[d], UNSHIFT<E>, static_cast<E*>(p.dv) + row, nullptr, 32 * d, p.N, real);
    }
}

template <class E, int D> int run(hipStream_t st, const rwkv_attn_args& p) {
    float* delta = static_cast<float*>(p.workspace);
    const int64_t rows = wide(p.B) * p.Tq * p.H, row_blocks = (rows * (D / 8) + 255) / 256;
    const int blocks_q = (p.Tq + 127) / 128, blocks_k = (p.Tk + 127) / 128;
    const int64_t per_q = (wide(blocks_q) * p.H * p.B + 7) / 8, per_k = (wide(blocks_k) * p.Hk * p.B + 7) / 8;
    if (row_blocks > INT_MAX || per_q * 8 > INT_MAX || per_k * 8 > INT_MAX) return RWKV_ERR_SHAPE;
    hipLaunchKernelGGL((attn_delta<E, D>), dim3(static_cast<unsigned>(row_blocks)), dim3(256), 0, st, p, delta);
    const auto go = [&](auto dq, auto dkv) {
        hipLaunchKernelGGL(dkv, dim3(static_cast<unsigned>(per_k * 8)), dim3(256), 0, st, p, delta, blocks_k, static_cast<int>(per_k));
        hipLaunchKernelGGL(dq, dim3(static_cast<unsigned>(per_q * 8)), dim3(256), 0, st, p, delta, blocks_q, static_cast<int>(per_q));
        return launch_status();
    };
    const auto masks = [&](auto cap, auto bias) {
        constexpr bool C = decltype(cap)::value, S = decltype(bias)::value;
        return p.doc ? go(attn_dq<E, D, C, S, true>, attn_dkv<E, D, C, S, true>) : go(attn_dq<E, D, C, S, false>, attn_dkv<E, D, C, S, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (p.cap > 0.f) return p.slopes ? masks(yes{}, yes{}) : masks(yes{}, no{});
    return p.slopes ? masks(no{}, yes{}) : masks(no{}, no{});
}
template <class E> int run_any(hipStream_t st, const rwkv_attn_args& p) { return p.N <= 64 ? run<E, 64>(st, p) : run<E, 128>(st, p); }

}  // namespace

int launch_attn_bwd(hipStream_t st, const rwkv_attn_args& p) { return p.dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, p) : run_any<half_t>(st, p); }

}  // namespace rwkv
