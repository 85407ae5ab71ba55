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
// Bound by memory: of B8 T4096 H32 N64 bf16 120 KB a chunk and head (64 of them kept by the walks), 2.0 GB in 500 us; two workgroups a CU, whose phases cover each other.
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

// infinities and NaN of bf16 as zeros
DEVINL u32x4 finite_ones(u32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] &= ((x[i] & 0x7f80) == 0x7f80 ? 0u : 0xffffu) | ((x[i] >> 16 & 0x7f80) == 0x7f80 ? 0u : 0xffff0000u);
    return x;
}

// 32 value channels by WIDTH tokens or key channels in LDS, two planes.  Tiles of a row, and their halves, are exchanged with the row's number, so that neither the writes (16 rows, 16 bytes) nor the
// reads (8 rows, 32 bytes) of half a wave meet in a bank.
template <int WIDTH> struct Slice {
    static constexpr int PITCH = 2 * WIDTH, PLANE = 32 * PITCH, BYTES = 2 * PLANE;
    static DEVINL lds_t at(const lds_t base, const int row, const int tile, const int byte) {
        return base + row * PITCH + 32 * (tile ^ (WIDTH == 64 ? row >> 1 & 3 : row & 7)) + (byte ^ (row >> 3 & 1) * 16);
    }
    static DEVINL void put(const lds_t base, const int lane, const int half, const int tile, const u32x4 x) {
        const lds_t to = at(base, lane & 15, tile, 8 * (lane >> 4)) + 16 * half * PITCH;
        lds_st(to, u32x2{x[0], x[1]});
        lds_st(to + PLANE, u32x2{x[2], x[3]});
    }
    static DEVINL Two32 get(const lds_t base, const int lane, const int tile) {
        typedef v4s __attribute__((address_space(3))) * ptr;
        const lds_t from = at(base, 4 * (lane >> 4) + (lane >> 2 & 3), tile, 8 * (lane & 3));
        u32x2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(from + (i & 1) * 16 * PITCH + (i >> 1) * PLANE)));
        return {join(x[0], x[1]), join(x[2], x[3])};
    }
};
// a lane's part of a kept state
DEVINL u32x4 kept_state(const u32x4 x) {
    const Two w = split<bf16_t>(__builtin_bit_cast(f32x4, x));
    return join(w.h, w.l);
}
// the sum of products of two kept tiles' numbers
DEVINL float dot(const uint32_t a, const uint32_t b, const float c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}
DEVINL float dot(const u32x4 a, const u32x4 b, float c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) c = dot(a[i], b[i], dot(a[i], b[i + 2], dot(a[i + 2], b[i], c)));
    return c;
}
// column block j, rows of blocks 2 s and 2 s + 1, of a Lower: the lane's column, the contraction over rows
DEVINL u32x4 lower_column(const lds_t base, const int lane, const int j, const int s) {
    typedef v4s __attribute__((address_space(3))) * ptr;
    const int l = lane & 15;
    const lds_t at = Lower<0>::at(base, 2 * s, 4 * (lane >> 4) + (l >> 2), j / 2, l & 3) + 8 * (j % 2);
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + 16 * (s ? Lower<0>::LONG : Lower<0>::SHORT)));
    return join(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b));
}
DEVINL Two32 lower_columns(const lds_t base, const int lane, const int j, const int s) { return {lower_column(base, lane, j, s), lower_column(base + Lower<0>::PLANE, lane, j, s)}; }

template <class E, int D> struct Place {
    static constexpr int PLANES = Input<E>::PLANES, WAVES = D / 16;
    static constexpr lds_t K = 0, Q = K + PLANES * Rows<D>::BYTES, SLICES = Q + PLANES * Rows<D>::BYTES, DY = SLICES, U = DY + PLANES * Rows<32>::BYTES, Z = U + Slice<64>::BYTES,
                           S = Z + Slice<64>::BYTES, DS = S + Slice<D>::BYTES, SLICES_END = DS + Slice<D>::BYTES, P = SLICES, A = P + Lower<0>::BYTES, MATRICES_END = A + Lower<0>::BYTES,
                           SCALARS = SLICES_END > MATRICES_END ? SLICES_END : MATRICES_END, ROW = SCALARS + Scalars::BYTES, COLUMN = ROW + 1024, BETA = COLUMN + 1024, VALUES = BETA + 1024,
                           QUERIES = VALUES + 64 * WAVES, KEYS = QUERIES + 256 * WAVES, READS = KEYS + 256 * WAVES, STATES = READS + 256 * WAVES, BYTES = STATES + 64;
    static_assert(BYTES <= 160 * 1024);
};

template <class E, int D>
__global__ __launch_bounds__(4 * D, 2) void delta_grads(const rwkv_delta_args p, const float* dS, const float* dZ, float* dq_of, float* dk_of) {
    using L = Place<E, D>;
    constexpr int WAVES = L::WAVES, LANES = 64 * WAVES, OWN = 16 / WAVES, PARTS = 8 / WAVES, PLANES = Input<E>::PLANES;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
    const int N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int t0 = blockIdx.x * DELTA_CHUNK, h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk);
    const int64_t chunk = (wide(b) * p.H + h) * chunks + blockIdx.x;
    const DeltaTiles tiles(p);
    const float *states = static_cast<const float*>(p.saved), *updates = states + tiles.states();

    // lane = token
    const int t = min(t0 + lane, T - 1);
    const float gate = to_f(static_cast<const E*>(p.g)[b * p.g_sb + t * p.g_st + h]), beta_t = to_f(static_cast<const E*>(p.beta)[b * p.beta_sb + t * p.beta_st + h]);
    const DeltaToken token = delta_token(p.doc, wide(b) * T, t0 + lane, T);
    const uint64_t real = __ballot(token.real);
    const auto mask_of = [&](const int row) { return 0u - static_cast<uint32_t>(real >> (row & 63) & 1); };
    const lds_t sc = lds + L::SCALARS;

    // rows of inputs, 16 bytes a lane, BELOW rows from piece to piece; of rows behind the last and channels that are not there others are read, and masked
    constexpr int PIECES = 64 * D / 8 / LANES, BELOW = LANES / (D / 8);
    const int row0 = written_row<D>(written_order<D>(tid)), d0 = 8 * written_piece<D>(tid), most = T - 1 - t0, yrow = written_row<32>(written_order<32>(tid & 255));
    static_assert(BELOW % 8 == 0);
    const bool in = d0 < N;
    u32x4 kr[PIECES], qr[PIECES];
    {
        const E *k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh + wide(t0) * p.k_st + (in ? d0 : 0), *q = static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh + wide(t0) * p.q_st + (in ? d0 : 0);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int row = min(row0 + BELOW * i, most);
            kr[i] = *reinterpret_cast<const u32x4*>(k + row * p.k_st);
            qr[i] = *reinterpret_cast<const u32x4*>(q + row * p.q_st);
        }
    }
    // the contractions over value channels, 32 at a time: a wave brings a tile of 32 of either state, and PARTS tiles of updates and of their gradients
    u32x4 sr[2], dr[2], ur[PARTS], zr[PARTS], yr;
    // ... and has 16 tokens of the values and of their gradients, all 8 or 4 value channels of the 32 in a lane
    constexpr int OWNS = WAVES == 4 ? 2 : 1;
    const int own = 16 * (wave & 3) + col, part = wave >> 2;
    u32x2 vr[OWNS];
    const E* v = static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh + (t0 + min(own, most)) * p.v_st;
    const E* dy = p.dy ? static_cast<const E*>(p.dy) + ((wide(b) * T + t0 + min(yrow, most)) * p.H + h) * N : v;      // (without one the values are read, and not used)
    E* dv = static_cast<E*>(p.dv) + ((wide(b) * T + t0 + own) * p.H + h) * N;
    const auto load = [&](const int step) {
        const int row = min(wave, tiles.tiles - 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int64_t from = tiles.state(chunk, min(2 * step + e, tiles.tiles - 1), row) + 4 * lane;
            sr[e] = *reinterpret_cast<const u32x4*>(states + from);
            dr[e] = *reinterpret_cast<const u32x4*>(dS + from);
        }
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
            const int n = wave + WAVES * m;
            const int64_t from = tiles.update(chunk, min(2 * step + n / 4, tiles.tiles - 1), n % 4) + 4 * lane;
            ur[m] = *reinterpret_cast<const u32x4*>(updates + from);
            zr[m] = *reinterpret_cast<const u32x4*>(dZ + from);
        }
        if (tid < 256) {
            const int c = 32 * step + 8 * (tid % 4);
            yr = *reinterpret_cast<const u32x4*>(dy + (c < N ? c : 0));
        }
#pragma unroll
        for (int e = 0; e < OWNS; ++e) {
            const int c = 32 * step + 16 * (part + e) + 4 * grp;
            vr[e] = *reinterpret_cast<const u32x2*>(v + (c < N ? c : 0));
        }
    };
    load(0);
    // Documents do not see each other, whatever stands in them: pairs across a cut, and states beyond one, are left out (a 0 would not do beside an infinity), and where there is a cut or padding, queries, keys and
    // gates that are no numbers become zeros: their document's states, updates and gradients are no numbers already, and the sums over tokens hold the others' too.
    const uint64_t cuts = __ballot(token.cut || (token.real && gate < DELTA_NONE));                // (not before the loads above are on their way)
    const bool apart = cuts != 0ull || __ballot(t0 + lane < T && !token.real) != 0ull;
    const auto upto = [](const int n) { return (2ull << n) - 1; };                                 // bits 0 .. n
    const auto pairs_of = [&](const int n) {                                                       // tokens up to n that n sees
        const uint64_t here = upto(n), cut = cuts & here;
        return real >> n & 1 ? real & here & (cut ? ~0ull << (63 - __builtin_clzll(cut)) : ~0ull) : 0ull;
    };
    if (wave == 0) make_scalars(sc, lane, token, apart && !finite(gate) && !(gate < DELTA_NONE) ? 0.f : gate, beta_t);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = row0 + BELOW * i;
        const uint32_t mask = in ? mask_of(row) : 0;
        u32x4 o[PLANES];
        planes_of<E>(kr[i] & mask, o);
#pragma unroll
        for (int n = 0; n < PLANES; ++n) Rows<D>::put(lds + L::K + n * Rows<D>::BYTES, row, d0 / 8, o[n]);
        planes_of<E>(qr[i] & mask, o);
#pragma unroll
        for (int n = 0; n < PLANES; ++n) Rows<D>::put(lds + L::Q + n * Rows<D>::BYTES, row, d0 / 8, o[n]);
    }
    const uint32_t y_mask = p.dy ? mask_of(yrow) : 0, v_mask = mask_of(own);
    f32x4 dQ[4], dK[4], R[4], dP[OWN], dA[OWN];
    float both = 0.f, vz = 0.f;                                  // of <dS', S>; of dZ V^T the diagonal
    // The pairs' blocks of row block `pi`: column blocks pj(0), pj(1) .. up to it
    const int pi = wave & 3;
    const auto pj = [&](const int m) { return WAVES == 4 ? m : 2 * m + part; };
#pragma unroll
    for (int step = 0; step < D / 32; ++step) {
        if (32 * step >= N) continue;
        const auto add = [&](const f32x4& c) { return step ? c : zero4(); };
        __syncthreads();                                         // (the step before has been read)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t mask = 2 * step + e < tiles.tiles && wave < tiles.tiles ? ~0u : 0;
            const u32x4 x = kept_state(sr[e] & mask), y = kept_state(dr[e] & mask);
            Slice<D>::put(lds + L::S, lane, e, wave, x);
            Slice<D>::put(lds + L::DS, lane, e, wave, y);
            both = dot(x, y, both);
        }
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
            const int n = wave + WAVES * m;
            const uint32_t mask = 2 * step + n / 4 < tiles.tiles ? ~0u : 0;
            Slice<64>::put(lds + L::U, lane, n / 4, n % 4, ur[m] & mask);
            Slice<64>::put(lds + L::Z, lane, n / 4, n % 4, zr[m] & mask);
        }
        if (tid < 256) {
            u32x4 o[PLANES];
            planes_of<E>(yr & (32 * step + 8 * (tid % 4) < N ? y_mask : 0), o);
#pragma unroll
            for (int n = 0; n < PLANES; ++n) Rows<32>::put(lds + L::DY + n * Rows<32>::BYTES, yrow, tid % 4, o[n]);
        }
        f32x4 values[OWNS];
#pragma unroll
        for (int e = 0; e < OWNS; ++e) values[e] = four_of<E>(vr[e] & (32 * step + 16 * (part + e) + 4 * grp < N ? v_mask : 0));
        __syncthreads();
        if (32 * (step + 1) < N) load(step + 1);
        const Two32 s = Slice<D>::get(lds + L::S, lane, wave), ds = Slice<D>::get(lds + L::DS, lane, wave);
        const auto gradient = [&](const int i) {
            Input<E> y;
            y.read(Rows<32>::BYTES, lds + L::DY, [&](const lds_t at) { return Rows<32>::row(at, lane, i, 0); });
            return y;
        };
        Two32 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = Slice<64>::get(lds + L::U, lane, i);
            dQ[i] = mma_in<E>(s, gradient(i), add(dQ[i]));
            dK[i] = mma32(ds, u[i], add(dK[i]));
            R[i] = mma32(s, Slice<64>::get(lds + L::Z, lane, i), add(R[i]));
        }
        const Input<E> y = gradient(pi);
        const Two32 z = Slice<64>::get(lds + L::Z, lane, pi);
#pragma unroll
        for (int m = 0; m < OWN; ++m) {
            if (pj(m) > pi) continue;
            const Two32 uj = WAVES == 4 ? u[m] : (part ? u[2 * m + 1] : u[2 * m]);
            dP[m] = mma_in<E>(uj, y, add(dP[m]));
            dA[m] = mma32(uj, z, add(dA[m]));
        }
        const float beta = lds_ld<float>(sc + Scalars::BETA + 4 * own);
#pragma unroll
        for (int e = 0; e < OWNS; ++e) {
            const int w = WAVES == 4 ? e : part, c = 32 * step + 16 * w + 4 * grp;
            const u32x2 zh = w ? u32x2{z.h[2], z.h[3]} : u32x2{z.h[0], z.h[1]}, zl = w ? u32x2{z.l[2], z.l[3]} : u32x2{z.l[0], z.l[1]};
            const f32x4 x = four_of<bf16_t>(zh) + four_of<bf16_t>(zl);
            vz += sum4(x * values[e]);
            if (c < N && own <= most) *reinterpret_cast<u32x2*>(dv + c) = u32x2{pack2<E>(beta * x[0], beta * x[1]), pack2<E>(beta * x[2], beta * x[3])};
        }
    }
    __syncthreads();
    if (apart) {
        for (lds_t x = lds + L::K + 16 * tid; x < lds + L::SLICES; x += 16 * LANES) lds_st(x, finite_ones(lds_ld<u32x4>(x)));
        __syncthreads();
    }

    // the pairs: rows j of a block and its column i in the lanes
    const auto at = [&](const lds_t what, const int n) { return sc + what + 4 * n; };
#pragma unroll
    for (int m = 0; m < OWN; ++m) {
        const int i = pi, j = pj(m), ti = 16 * i + col, tj = 16 * j + 4 * grp;
        if (j > i) continue;
        const uint32_t seen = static_cast<uint32_t>(pairs_of(ti) >> tj);                           // bit r: token tj + r
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
            for (int r = 0; r < 4; ++r) d[r] = seen >> r & 1 ? __builtin_amdgcn_exp2f((h - hj[r]) + (l - lj[r])) : 0.f;
        } else {
            const int end = 16 * j + 15;
            d = lds_ld<f32x4>(at(Scalars::TAIL, tj)) * __builtin_amdgcn_exp2f((h - lds_ld<float>(at(Scalars::SUM, end))) + (l - lds_ld<float>(at(Scalars::REST, end))));
        }
        f32x4 dp, ab, pair;
        float db = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool sees = seen >> r & 1, below = sees && ti > tj + r;
            dp[r] = sees ? p.scale * d[r] * dP[m][r] : 0.f;
            const float da = below ? -d[r] * dA[m][r] : 0.f;
            ab[r] = below ? beta * da : 0.f;
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
    vz = group_sum4(vz);
    if (grp == 0) lds_st(lds + L::VALUES + 256 * part + 4 * own, vz);
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
    // where a wave's part of the chunk begins, what 16 tokens take there, and a lane's place: bytes
    const bool own_channels = 16 * wave + 4 * grp < N;
    const int size = dq_of ? 4 : 2, heads = dq_of ? p.H : p.Hk;
    const int64_t to = (((wide(b) * T + t0) * heads + (dq_of ? h : hk)) * N + 16 * wave) * size, step = wide(16) * heads * N * size;
    const uint32_t at_lane = (static_cast<uint32_t>(col) * heads * N + 4 * grp) * size;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ti = 16 * i + col;
        const float enter = lds_ld<float>(at(Scalars::ENTER, ti)), leave = lds_ld<float>(at(Scalars::LEAVE, ti)), beta = lds_ld<float>(at(Scalars::BETA, ti));
        const f32x4 q4 = four(lds + L::Q, ti), k4 = four(lds + L::K, ti);
        const bool is = real >> ti & 1, enters = is && !(cuts & upto(ti)), leaves = is && !(cuts >> ti >> 1);
        dQ[i] = enters ? dQ[i] * (p.scale * enter) : zero4();
        dK[i] = leaves ? dK[i] * leave : zero4();
        R[i] = enters ? R[i] * enter : zero4();
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
        if (t0 + ti >= T || !own_channels) continue;
        if (dq_of) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(dq_of) + to + i * step + at_lane) = dQ[i];
            *reinterpret_cast<f32x4*>(reinterpret_cast<char*>(dk_of) + to + i * step + at_lane) = dK[i];
        } else {
            *reinterpret_cast<u32x2*>(static_cast<char*>(p.dq) + to + i * step + at_lane) = u32x2{pack2<E>(dQ[i][0], dQ[i][1]), pack2<E>(dQ[i][2], dQ[i][3])};
            *reinterpret_cast<u32x2*>(static_cast<char*>(p.dk) + to + i * step + at_lane) = u32x2{pack2<E>(dK[i][0], dK[i][1]), pack2<E>(dK[i][2], dK[i][3])};
        }
    }
    __syncthreads();
    if (wave != 0 || t0 + lane >= T) return;
    float after = 0.f, before = 0.f, reads = 0.f, db = lds_ld<float>(lds + L::VALUES + 4 * lane) + (WAVES == 8 ? lds_ld<float>(lds + L::VALUES + 256 + 4 * lane) : 0.f), ends = 0.f;
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
    // (what passes token t ends at the next cut, and began behind the last: added up across them, others' sums would cancel but to their rounding)
    float suffix = after, prefix = before;
    const int until = cuts >> lane >> 1 ? lane + 1 + __builtin_ctzll(cuts >> lane >> 1) : min(64, T - t0), since = 63 - __builtin_clzll((cuts & (2ull << lane) - 1) | 1);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float a = __shfl_down(suffix, x, 64), c = __shfl_up(prefix, x, 64);
        if (lane + x < until) suffix += a;
        if (lane - x >= since) prefix += c;
    }
    const bool counts = token.real && !(cuts >> lane & 1);
    const int64_t token_at = (wide(b) * T + t0 + lane) * p.H + h;
    static_cast<E*>(p.dg)[token_at] = from_f<E>(counts ? suffix + (prefix - before) + (cuts ? 0.f : ends * lds_ld<float>(at(Scalars::ENTER, 63))) : 0.f);
    static_cast<E*>(p.dbeta)[token_at] = from_f<E>(db);
}

template <class E, int D> int run(hipStream_t st, const rwkv_delta_args& p, const float* dS, const float* dZ, float* dq, float* dk) {
    const int64_t blocks = DeltaTiles(p).chunks;
    if (blocks > INT_MAX) return RWKV_ERR_SHAPE;
    hipLaunchKernelGGL((delta_grads<E, D>), dim3(static_cast<unsigned>(blocks / p.B / p.H), p.H, p.B), dim3(4 * D), 0, st, p, dS, dZ, dq, dk);
    return launch_status();
}

}  // namespace

int launch_delta_grads(hipStream_t st, const rwkv_delta_args& p, const float* dS, const float* dZ, float* dq, float* dk) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run<bf16_t, 64>(st, p, dS, dZ, dq, dk) : run<bf16_t, 128>(st, p, dS, dZ, dq, dk);
    return p.N <= 64 ? run<half_t, 64>(st, p, dS, dZ, dq, dk) : run<half_t, 128>(st, p, dS, dZ, dq, dk);
}

}  // namespace rwkv
