// Gated delta rule, whole sequences, the gradients of the inputs (formulas and layouts: delta.h).
//
// A workgroup has a chunk of a head: with the state S that enters it, the gradient dS' of the one that leaves, the updates U and dZ, all of which other kernels left,
//   dP = D o dY U^T (i >= j), dA = -D o dZ U^T (i > j), both once without and once times what they stand beside,
//   dQ = scale e^G dY S^T + scale dP K
//   dK = e^(G_64 - G) U dS'^T - beta e^G dZ S^T + scale dP^T Q + (beta dA) K + (beta dA)^T K
//   dV = beta dZ,   dbeta_i = dZ_i.V_i - e^G_i k_i.(S dZ_i) + sum_j dA_ij k_i.k_j
//   dg_t: all that passes token t, i.e. e^G_64 <dS', S>, the keys' part through dS' of the tokens before, the queries' and keys' parts through S of t and those behind, and the pairs around it.
// The contractions over value channels go 32 at a time: what the state's waves left as four rows a lane goes to LDS as columns and comes back as rows (ds_read_b64_tr_b16).  A wave has 16 of the
// key channels, all tokens, and some of the pairs' blocks.  All sums are in a fixed order.
#include <algorithm>

#include "delta.h"

namespace rwkv {
namespace {

DEVINL float row_sum(float x) {                                 // over 16 lanes
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xf, 0xf, true));
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xf, 0xf, true));
}
DEVINL float group_sum4(const float x) {                        // over the four lanes with the same lane & 15
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
DEVINL float sum4(const f32x4 x) { return (x[0] + x[1]) + (x[2] + x[3]); }

// Inputs as operands: one number of bf16, or two for fp16 (8 and 3 of its 11 bits)
template <class E> struct Input {
    static constexpr int PLANES = std::is_same_v<E, bf16_t> ? 1 : 2;
    u32x4 x[PLANES];
    template <class Read> DEVINL void read(const int plane, const lds_t base, Read r) {
#pragma unroll
        for (int n = 0; n < PLANES; ++n) x[n] = r(base + n * plane);
    }
};
template <class E> DEVINL void planes_of(const u32x4 v, u32x4 (&o)[Input<E>::PLANES]) {
    if constexpr (std::is_same_v<E, bf16_t>) o[0] = v;
    else {
        const Two a = split<bf16_t>(four_of<E>(u32x2{v[0], v[1]})), b = split<bf16_t>(four_of<E>(u32x2{v[2], v[3]}));
        o[0] = join(a.h, b.h);
        o[1] = join(a.l, b.l);
    }
}
template <class E> DEVINL f32x4 mma_in(const Two32& a, const Input<E>& b, f32x4 c) {
    c = mma32<bf16_t>(a.l, b.x[0], c);
    if constexpr (Input<E>::PLANES == 2) c = mma32<bf16_t>(a.h, b.x[1], c);
    return mma32<bf16_t>(a.h, b.x[0], c);
}
template <class E> DEVINL f32x4 mma_in(const Input<E>& a, const Two32& b, f32x4 c) {
    c = mma32<bf16_t>(a.x[0], b.l, c);
    if constexpr (Input<E>::PLANES == 2) c = mma32<bf16_t>(a.x[1], b.h, c);
    return mma32<bf16_t>(a.x[0], b.h, c);
}
template <class E> DEVINL f32x4 mma_in(const Input<E>& a, const Input<E>& b, f32x4 c) {
    if constexpr (Input<E>::PLANES == 2) {
        c = mma32<bf16_t>(a.x[0], b.x[1], c);
        c = mma32<bf16_t>(a.x[1], b.x[0], c);
    }
    return mma32<bf16_t>(a.x[0], b.x[0], c);
}

// 32 value channels by WIDTH tokens or key channels in LDS, two planes
template <int WIDTH> struct Slice {
    static constexpr int PITCH = 2 * WIDTH + 16, PLANE = 32 * PITCH, BYTES = 2 * PLANE;
    static DEVINL void put(const lds_t base, const int lane, const int half, const int tile, const f32x4 x) {
        const Two w = split<bf16_t>(x);
        const lds_t to = base + (16 * half + (lane & 15)) * PITCH + 32 * tile + 8 * (lane >> 4);
        lds_st(to, w.h);
        lds_st(to + PLANE, w.l);
    }
    static DEVINL u32x4 plane(const lds_t base, const int lane, const int tile) {
        typedef v4s __attribute__((address_space(3))) * ptr;
        const int l = lane & 15;
        const lds_t at = base + (4 * (lane >> 4) + (l >> 2)) * PITCH + 32 * tile + 8 * (l & 3);
        const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + 16 * PITCH));
        return join(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b));
    }
    static DEVINL Two32 get(const lds_t base, const int lane, const int tile) { return {plane(base, lane, tile), plane(base + PLANE, lane, tile)}; }
};
// column block j, rows of blocks 2 s and 2 s + 1, of a Lower: the lane's column, the contraction over rows
DEVINL u32x4 lower_column(const lds_t base, const int lane, const int j, const int s) {
    typedef v4s __attribute__((address_space(3))) * ptr;
    const int l = lane & 15;
    const lds_t at = Lower<0>::at(base, 2 * s, 4 * (lane >> 4) + (l >> 2)) + 64 * (j / 2) + 16 * (l & 3) + 8 * (j % 2);
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + 16 * (s ? Lower<0>::LONG : Lower<0>::SHORT)));
    return join(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b));
}
DEVINL Two32 lower_columns(const lds_t base, const int lane, const int j, const int s) { return {lower_column(base, lane, j, s), lower_column(base + Lower<0>::PLANE, lane, j, s)}; }

template <class E, int D> struct Place {
    static constexpr int PLANES = Input<E>::PLANES, WAVES = D / 16;
    static constexpr lds_t K = 0, Q = K + PLANES * Rows<D>::BYTES, SLICES = Q + PLANES * Rows<D>::BYTES, DY = SLICES, V = DY + PLANES * Rows<32>::BYTES, U = V + PLANES * Rows<32>::BYTES, Z = U + Slice<64>::BYTES,
                           S = Z + Slice<64>::BYTES, DS = S + Slice<D>::BYTES, SLICES_END = DS + Slice<D>::BYTES, P = SLICES, A = P + Lower<0>::BYTES, MATRICES_END = A + Lower<0>::BYTES,
                           SCALARS = SLICES_END > MATRICES_END ? SLICES_END : MATRICES_END, ROW = SCALARS + Scalars::BYTES, COLUMN = ROW + 1024, BETA = COLUMN + 1024, VALUES = BETA + 1024, QUERIES = VALUES + 256,
                           KEYS = QUERIES + 256 * WAVES, READS = KEYS + 256 * WAVES, STATES = READS + 256 * WAVES, BYTES = STATES + 64;
    static_assert(BYTES <= 160 * 1024);
};

template <class E, int D>
__global__ __launch_bounds__(4 * D, 2) void delta_grads(const rwkv_delta_args p, const float* dS, const float* dZ, float* dq_of, float* dk_of) {
    using L = Place<E, D>;
    constexpr int WAVES = L::WAVES, LANES = 64 * WAVES, OWN = (10 + WAVES - 1) / WAVES, PARTS = 8 / WAVES, PLANES = Input<E>::PLANES;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
    const int N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int64_t chunk = blockIdx.x;
    const int hb = static_cast<int>(chunk / chunks), t0 = static_cast<int>(chunk % chunks) * DELTA_CHUNK, b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk);
    const DeltaTiles tiles(p);
    const float *states = static_cast<const float*>(p.saved), *updates = states + tiles.states();
    const E *q = static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh, *k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh, *v = static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh;
    const E* dy = p.dy ? static_cast<const E*>(p.dy) + (wide(b) * T * p.H + h) * N : nullptr;

    // lane = token
    const int t = min(t0 + lane, T - 1);
    const float gate = to_f(static_cast<const E*>(p.g)[b * p.g_sb + t * p.g_st + h]), beta_t = to_f(static_cast<const E*>(p.beta)[b * p.beta_sb + t * p.beta_st + h]);
    const DeltaToken token = delta_token(p.doc, wide(b) * T, t0 + lane, T);
    const uint64_t real = __ballot(token.real);
    const lds_t sc = lds + L::SCALARS;
    // the contractions over value channels, 32 at a time
    f32x4 sr[2], dr[2], ur[PARTS], zr[PARTS];
    u32x4 yr[2];                                                 // (of y's gradients and of the values; one of them where there are lanes enough)
    const auto load = [&](const int step) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int ct = 2 * step + e;
            const bool is = ct < tiles.tiles && wave < tiles.tiles;
            sr[e] = is ? *reinterpret_cast<const f32x4*>(states + tiles.state(chunk, ct, wave) + 4 * lane) : zero4();
            dr[e] = is ? *reinterpret_cast<const f32x4*>(dS + tiles.state(chunk, ct, wave) + 4 * lane) : zero4();
        }
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
            const int n = wave + WAVES * m, ct = 2 * step + n / 4;
            ur[m] = ct < tiles.tiles ? *reinterpret_cast<const f32x4*>(updates + tiles.update(chunk, ct, n % 4) + 4 * lane) : zero4();
            zr[m] = ct < tiles.tiles ? *reinterpret_cast<const f32x4*>(dZ + tiles.update(chunk, ct, n % 4) + 4 * lane) : zero4();
        }
#pragma unroll
        for (int m = 0; m < (WAVES == 4 ? 2 : 1); ++m) {
            const int x = tid & 255, row = x / 4, c = 32 * step + 8 * (x % 4);
            const bool values = WAVES == 4 ? m == 1 : tid >= 256, ok = (real >> row & 1) && c < N && (values || dy);
            const E* from = values ? v + wide(t0 + row) * p.v_st + c : dy + wide(t0 + row) * p.H * N + c;
            yr[m] = ok ? *reinterpret_cast<const u32x4*>(from) : u32x4{0, 0, 0, 0};
        }
    };
    const int steps = (tiles.tiles + 1) / 2;
    f32x4 dQ[4], dK[4], R[4], dP[OWN], dA[OWN], vz = zero4();
    float both = 0.f;                                            // of <dS', S>
#pragma unroll
    for (int i = 0; i < 4; ++i) dQ[i] = dK[i] = R[i] = zero4();
#pragma unroll
    for (int m = 0; m < OWN; ++m) dP[m] = dA[m] = zero4();
    // block n of the lower triangle
    const auto row_of = [](const int n) { return n >= 6 ? 3 : (n >= 3 ? 2 : (n >= 1 ? 1 : 0)); };
    const auto column_of = [&](const int n) { return n - row_of(n) * (row_of(n) + 1) / 2; };
    constexpr int PIECES = 64 * D / 8 / LANES;
    u32x4 kr[PIECES], qr[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int x = tid + LANES * i, row = x / (D / 8), c = x % (D / 8);
        const bool ok = (real >> row & 1) && 8 * c < N;
        kr[i] = ok ? *reinterpret_cast<const u32x4*>(k + wide(t0 + row) * p.k_st + 8 * c) : u32x4{0, 0, 0, 0};
        qr[i] = ok ? *reinterpret_cast<const u32x4*>(q + wide(t0 + row) * p.q_st + 8 * c) : u32x4{0, 0, 0, 0};
    }
    load(0);
    if (wave == 0) make_scalars(sc, lane, token, gate, beta_t);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int x = tid + LANES * i, row = x / (D / 8), c = x % (D / 8);
        u32x4 o[PLANES];
        planes_of<E>(kr[i], o);
#pragma unroll
        for (int n = 0; n < PLANES; ++n) Rows<D>::put(lds + L::K + n * Rows<D>::BYTES, row, c, o[n]);
        planes_of<E>(qr[i], o);
#pragma unroll
        for (int n = 0; n < PLANES; ++n) Rows<D>::put(lds + L::Q + n * Rows<D>::BYTES, row, c, o[n]);
    }
    for (int step = 0; step < steps; ++step) {
        __syncthreads();                                         // (the step before has been read)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            Slice<D>::put(lds + L::S, lane, e, wave, sr[e]);
            Slice<D>::put(lds + L::DS, lane, e, wave, dr[e]);
            both += sum4(sr[e] * dr[e]);
        }
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
            const int n = wave + WAVES * m;
            Slice<64>::put(lds + L::U, lane, n / 4, n % 4, ur[m]);
            Slice<64>::put(lds + L::Z, lane, n / 4, n % 4, zr[m]);
        }
#pragma unroll
        for (int m = 0; m < (WAVES == 4 ? 2 : 1); ++m) {
            const int x = tid & 255;
            const bool values = WAVES == 4 ? m == 1 : tid >= 256;
            u32x4 o[PLANES];
            planes_of<E>(yr[m], o);
#pragma unroll
            for (int n = 0; n < PLANES; ++n) Rows<32>::put(lds + (values ? L::V : L::DY) + n * Rows<32>::BYTES, x / 4, x % 4, o[n]);
        }
        __syncthreads();
        if (step + 1 < steps) load(step + 1);
        const Two32 s = Slice<D>::get(lds + L::S, lane, wave), ds = Slice<D>::get(lds + L::DS, lane, wave);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Input<E> y;
            y.read(Rows<32>::BYTES, lds + L::DY, [&](const lds_t at) { return Rows<32>::row(at, lane, i, 0); });
            dQ[i] = mma_in<E>(s, y, dQ[i]);
            dK[i] = mma32(ds, Slice<64>::get(lds + L::U, lane, i), dK[i]);
            R[i] = mma32(s, Slice<64>::get(lds + L::Z, lane, i), R[i]);
        }
#pragma unroll
        for (int m = 0; m < OWN; ++m) {
            const int n = wave + WAVES * m, i = row_of(n), j = column_of(n);
            if (n >= 10) continue;
            const Two32 u = Slice<64>::get(lds + L::U, lane, j);
            Input<E> y;
            y.read(Rows<32>::BYTES, lds + L::DY, [&](const lds_t at) { return Rows<32>::row(at, lane, i, 0); });
            dP[m] = mma_in<E>(u, y, dP[m]);
            dA[m] = mma32(u, Slice<64>::get(lds + L::Z, lane, i), dA[m]);
        }
        if (wave < 4) {                                          // of dZ V^T the diagonal counts
            Input<E> y;
            y.read(Rows<32>::BYTES, lds + L::V, [&](const lds_t at) { return Rows<32>::row(at, lane, wave, 0); });
            vz = mma_in<E>(y, Slice<64>::get(lds + L::Z, lane, wave), vz);
        }
    }
    __syncthreads();

    // the pairs: rows j of a block and its column i in the lanes
    const auto at = [&](const lds_t what, const int n) { return sc + what + 4 * n; };
#pragma unroll
    for (int m = 0; m < OWN; ++m) {
        const int n = wave + WAVES * m, i = row_of(n), j = column_of(n), ti = 16 * i + col, tj = 16 * j + 4 * grp;
        if (n >= 10) continue;
        f32x4 kk = zero4(), qk = zero4();
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            Input<E> kj, ki, qi;
            kj.read(Rows<D>::BYTES, lds + L::K, [&](const lds_t x) { return Rows<D>::row(x, lane, j, s); });
            ki.read(Rows<D>::BYTES, lds + L::K, [&](const lds_t x) { return Rows<D>::row(x, lane, i, s); });
            qi.read(Rows<D>::BYTES, lds + L::Q, [&](const lds_t x) { return Rows<D>::row(x, lane, i, s); });
            kk = mma_in<E>(kj, ki, kk);
            qk = mma_in<E>(kj, qi, qk);
        }
        const float h = lds_ld<float>(at(Scalars::SUM, ti)), l = lds_ld<float>(at(Scalars::REST, ti)), beta = lds_ld<float>(at(Scalars::BETA, ti));
        f32x4 d;
        if (i == j) {
            const f32x4 hj = lds_ld<f32x4>(at(Scalars::SUM, tj)), lj = lds_ld<f32x4>(at(Scalars::REST, tj));
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = ti >= tj + r ? __builtin_amdgcn_exp2f((h - hj[r]) + (l - lj[r])) : 0.f;
        } else {
            const int end = 16 * j + 15;
            d = lds_ld<f32x4>(at(Scalars::TAIL, tj)) * __builtin_amdgcn_exp2f((h - lds_ld<float>(at(Scalars::SUM, end))) + (l - lds_ld<float>(at(Scalars::REST, end))));
        }
        f32x4 dp, ab, pair;
        float db = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool below = ti > tj + r;
            dp[r] = ti >= tj + r ? p.scale * d[r] * dP[m][r] : 0.f;
            const float da = below ? -d[r] * dA[m][r] : 0.f;
            ab[r] = beta * da;
            db = fmaf(da, kk[r], db);
            pair[r] = below ? dp[r] * qk[r] + ab[r] * kk[r] : 0.f;
        }
        Lower<0>::put(lds + L::P, i, col, j, grp, split<bf16_t>(dp));
        Lower<0>::put(lds + L::A, i, col, j, grp, split<bf16_t>(ab));
        const float rows = group_sum4(sum4(pair)), betas = group_sum4(db);
        if (grp == 0) lds_st(lds + L::ROW + 256 * j + 4 * ti, rows), lds_st(lds + L::BETA + 256 * j + 4 * ti, betas);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float columns = row_sum(pair[r]);
            if (col == 0) lds_st(lds + L::COLUMN + 256 * i + 4 * (tj + r), columns);
        }
    }
    if (wave < 2) {                                              // nothing stands above the diagonal
        const Two none = {{0, 0}, {0, 0}};
        Lower<0>::put(lds + L::P, 2 * wave, col, 2 * wave + 1, grp, none);
        Lower<0>::put(lds + L::A, 2 * wave, col, 2 * wave + 1, grp, none);
    }
    if (wave < 4 && col >> 2 == grp) {
        const float x = (col & 3) == 0 ? vz[0] : ((col & 3) == 1 ? vz[1] : ((col & 3) == 2 ? vz[2] : vz[3]));
        lds_st(lds + L::VALUES + 4 * (16 * wave + col), x);
    }
    const float all = group_sum4(row_sum(both));
    if (lane == 0) lds_st(lds + L::STATES + 4 * wave, all);
    __syncthreads();

    // a wave's 16 key channels of dq and dk: a token's in the lanes
    Input<E> kc[2], qc[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        kc[s].read(Rows<D>::BYTES, lds + L::K, [&](const lds_t x) { return Rows<D>::col(x, lane, wave, s); });
        qc[s].read(Rows<D>::BYTES, lds + L::Q, [&](const lds_t x) { return Rows<D>::col(x, lane, wave, s); });
    }
    const auto four = [&](const lds_t base, const int row) {
        f32x4 o = zero4();
#pragma unroll
        for (int n = 0; n < PLANES; ++n) {
            const u32x2 x = Rows<D>::four(base + n * Rows<D>::BYTES, row, wave, grp);
            o += f32x4{bf_lo(x[0]), bf_hi(x[0]), bf_lo(x[1]), bf_hi(x[1])};
        }
        return o;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ti = 16 * i + col;
        const float enter = lds_ld<float>(at(Scalars::ENTER, ti)), leave = lds_ld<float>(at(Scalars::LEAVE, ti)), beta = lds_ld<float>(at(Scalars::BETA, ti));
        const f32x4 q4 = four(lds + L::Q, ti), k4 = four(lds + L::K, ti);
        dQ[i] *= p.scale * enter;
        dK[i] *= leave;
        R[i] *= enter;
        const float queries = group_sum4(sum4(q4 * dQ[i])), keys = group_sum4(sum4(k4 * dK[i])), reads = group_sum4(sum4(k4 * R[i]));
        if (grp == 0) lds_st(lds + L::QUERIES + 256 * wave + 4 * ti, queries), lds_st(lds + L::KEYS + 256 * wave + 4 * ti, keys), lds_st(lds + L::READS + 256 * wave + 4 * ti, reads);
        dK[i] -= beta * R[i];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (i >= 2 * s) {
                dQ[i] = mma_in<E>(kc[s], Lower<0>::two(lds + L::P, lane, i, s), dQ[i]);
                dK[i] = mma_in<E>(kc[s], Lower<0>::two(lds + L::A, lane, i, s), dK[i]);
            }
            if (i < 2 * s + 2) {
                dK[i] = mma_in<E>(qc[s], lower_columns(lds + L::P, lane, i, s), dK[i]);
                dK[i] = mma_in<E>(kc[s], lower_columns(lds + L::A, lane, i, s), dK[i]);
            }
        }
        const int tt = t0 + ti, c = 16 * wave + 4 * grp;
        if (tt >= T || c >= N) continue;
        if (dq_of) {
            const int64_t to = ((wide(b) * T + tt) * p.H + h) * N + c;
            *reinterpret_cast<f32x4*>(dq_of + to) = dQ[i];
            *reinterpret_cast<f32x4*>(dk_of + to) = dK[i];
        } else {
            const int64_t to = ((wide(b) * T + tt) * p.Hk + hk) * N + c;
            *reinterpret_cast<u32x2*>(static_cast<E*>(p.dq) + to) = u32x2{pack2<E>(dQ[i][0], dQ[i][1]), pack2<E>(dQ[i][2], dQ[i][3])};
            *reinterpret_cast<u32x2*>(static_cast<E*>(p.dk) + to) = u32x2{pack2<E>(dK[i][0], dK[i][1]), pack2<E>(dK[i][2], dK[i][3])};
        }
    }
    // dv: 16 value channels a wave, as the updates lie
    for (int ct = wave; ct < tiles.tiles; ct += WAVES)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 z = *reinterpret_cast<const f32x4*>(dZ + tiles.update(chunk, ct, i) + 4 * lane) * lds_ld<f32x4>(at(Scalars::BETA, 16 * i + 4 * grp));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int tt = t0 + 16 * i + 4 * grp + r;
                if (tt < T && 16 * ct + col < N) static_cast<E*>(p.dv)[((wide(b) * T + tt) * p.H + h) * N + 16 * ct + col] = from_f<E>(z[r]);
            }
        }
    __syncthreads();
    if (wave != 0 || t0 + lane >= T) return;
    float after = 0.f, before = 0.f, reads = 0.f, db = lds_ld<float>(lds + L::VALUES + 4 * lane), ends = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        after += lds_ld<float>(lds + L::QUERIES + 256 * w + 4 * lane);
        before += lds_ld<float>(lds + L::KEYS + 256 * w + 4 * lane);
        reads += lds_ld<float>(lds + L::READS + 256 * w + 4 * lane);
        ends += lds_ld<float>(lds + L::STATES + 4 * w);
    }
    const float beta = lds_ld<float>(at(Scalars::BETA, lane));
    after -= beta * reads;
    db -= reads;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        if (n <= lane >> 4) after += lds_ld<float>(lds + L::ROW + 256 * n + 4 * lane), db += lds_ld<float>(lds + L::BETA + 256 * n + 4 * lane);
        if (n >= lane >> 4) after -= lds_ld<float>(lds + L::COLUMN + 256 * n + 4 * lane);
    }
    float suffix = after, prefix = before;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float a = __shfl_down(suffix, x, 64), c = __shfl_up(prefix, x, 64);
        if (lane + x < min(64, T - t0)) suffix += a;
        if (lane >= x) prefix += c;
    }
    const bool counts = token.real && !token.cut && !(gate < DELTA_NONE);
    const int64_t to = (wide(b) * T + t0 + lane) * p.H + h;
    static_cast<E*>(p.dg)[to] = from_f<E>(counts ? suffix + (prefix - before) + ends * lds_ld<float>(at(Scalars::ENTER, 63)) : 0.f);
    static_cast<E*>(p.dbeta)[to] = from_f<E>(db);
}

template <class E, int D> int run(hipStream_t st, const rwkv_delta_args& p, const float* dS, const float* dZ, float* dq, float* dk) {
    const int64_t blocks = DeltaTiles(p).chunks;
    if (blocks > INT_MAX) return RWKV_ERR_SHAPE;
    hipLaunchKernelGGL((delta_grads<E, D>), dim3(static_cast<unsigned>(blocks)), dim3(4 * D), 0, st, p, dS, dZ, dq, dk);
    return launch_status();
}

}  // namespace

int launch_delta_grads(hipStream_t st, const rwkv_delta_args& p, const float* dS, const float* dZ, float* dq, float* dk) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run<bf16_t, 64>(st, p, dS, dZ, dq, dk) : run<bf16_t, 128>(st, p, dS, dZ, dq, dk);
    return p.N <= 64 ? run<half_t, 64>(st, p, dS, dZ, dq, dk) : run<half_t, 128>(st, p, dS, dZ, dq, dk);
}

}  // namespace rwkv
