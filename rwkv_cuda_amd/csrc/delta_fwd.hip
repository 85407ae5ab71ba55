// Gated delta rule, whole sequences, forward (formulas and layouts: delta.h).
//
// A workgroup has 16 SW of a head's value channels and walks through the sequence, a chunk of 64 tokens after the other.  SW waves keep 16 columns of the state each and do what
// depends on it; the others bring the next chunk's inputs and make its matrices meanwhile: -A, P and the inverses of the blocks of I + A on the diagonal, with which the triangular system is
// four steps of products.  Two barriers a chunk: before the first the next chunk's rows go to LDS, behind it they are read.
#include <algorithm>

#include "delta.h"

namespace rwkv {
namespace {

template <int D, int SW> struct Place {                          // (scalars are made a chunk earlier than what uses them)
    static constexpr int VPITCH = 32 * SW + 16;
    static constexpr lds_t ROWS = 0, K = 0, Q = Rows<D>::BYTES, STAGE = 2 * Rows<D>::BYTES, V = 2 * STAGE, MATRICES = V + 64 * VPITCH, A = 0, P = Lower<1>::BYTES, INV = P + Lower<0>::BYTES,
                           MATRIX_STAGE = INV + Diagonal::BYTES, SCALARS = MATRICES + 2 * MATRIX_STAGE, BYTES = SCALARS + 3 * Scalars::BYTES;
    static_assert(BYTES <= 160 * 1024);
};

template <class E, int D, int SW, int HELPERS>
__global__ __launch_bounds__(64 * (SW + HELPERS)) void delta_fwd(const rwkv_delta_args p, const int pieces) {
    using L = Place<D, SW>;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    // the pieces of a head are neighbours on one XCD: they read the same keys and queries
    const int slot = blockIdx.x >> 3, piece = slot % pieces, hb = slot / pieces * 8 + (blockIdx.x & 7);
    if (hb >= p.B * p.H) return;
    const int b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk), N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;

    if (wave < SW) {
        const int ct = piece * SW + wave, c0 = 16 * ct;          // its columns
        const DeltaTiles tiles(p);
        float *states = static_cast<float*>(p.saved), *updates = states + tiles.states();
        const bool on = c0 + col < N;
        f32x4 S[D / 16];
        const float* s0 = p.s0 ? p.s0 + wide(hb) * N * N : nullptr;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = s0 && on && 16 * t + 4 * grp + r < N ? s0[(16 * t + 4 * grp + r) * N + c0 + col] : 0.f;
        const lds_t vread = L::V + lds + (4 * grp + (col >> 2)) * L::VPITCH + 32 * wave + 8 * (col & 3);
        E* y = static_cast<E*>(p.y) + (wide(b) * T * p.H + h) * N + c0 + 4 * grp;
        __syncthreads();
        __syncthreads();
        for (int c = 0; c < chunks; ++c) {
            const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE, sc = lds + L::SCALARS + c % 3 * Scalars::BYTES;
            const lds_t K = rows + L::K, Q = rows + L::Q, A = mats + L::A, P = mats + L::P, inv = mats + L::INV;
            typedef v4s __attribute__((address_space(3))) * ptr;
            if (p.saved && c0 < N) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
                    if (t < tiles.tiles) *reinterpret_cast<f32x4*>(states + tiles.state(wide(hb) * chunks + c, ct, t) + 4 * lane) = S[t];
            }
            // what a step reads from LDS is on its way a step earlier
            const Two inv0 = Diagonal::row(inv, lane, 0), a10 = Lower<1>::one(A, lane, 1, 0), inv1 = Diagonal::row(inv, lane, 1);
            f32x4 enter[4], beta[4], Z[4];
            u32x2 v[4];
            Beside<E, D / 16> s;
            u32x4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(vread + 16 * i * L::VPITCH)));
                x[i] = Rows<D>::row(K, lane, i, 0);
            }
            in_order();
            s.take(S);
            __syncthreads();                                     // (the values have been read)
#pragma unroll
            for (int i = 0; i < 4; ++i) Z[i] = mma32<E>(x[i], s.lo(0), zero4());
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                u32x4 next[4];
                if (k + 1 < D / 32)
#pragma unroll
                    for (int i = 0; i < 4; ++i) next[i] = Rows<D>::row(K, lane, i, k + 1);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        enter[i] = lds_ld<f32x4>(sc + Scalars::ENTER + 64 * i + 16 * grp);
                        beta[i] = lds_ld<f32x4>(sc + Scalars::BETA + 64 * i + 16 * grp);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) Z[i] = mma32<E>(x[i], s.hi(k), Z[i]);
                if (k + 1 < D / 32)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = next[i], Z[i] = mma32<E>(x[i], s.lo(k + 1), Z[i]);
                in_order();
            }
            // the triangular system, and beside it the outputs
            f32x4 Y[4], U[4], z[4], leave;
            float enters;
            const float whole = lds_ld<float>(sc + Scalars::ENTER + 4 * 63);
            Two u0, u1, u2, u3;
            const auto queries = [&](const int i) {
#pragma unroll
                for (int k = 0; k < (D == 64 ? 2 : 4); ++k) x[k] = Rows<D>::row(Q, lane, i, k);
                enters = lds_ld<float>(sc + Scalars::ENTER + 4 * (16 * i + col));
            };
            const auto outputs = [&](const int i) {             // of the state that enters
                f32x4 y = mma32<E>(s.lo(0), x[0], zero4());
                y = mma32<E>(s.hi(0), x[0], y);
#pragma unroll
                for (int k = 1; k < D / 32; ++k) {
                    y = mma32<E>(s.lo(k), x[k], y);
                    y = mma32<E>(s.hi(k), x[k], y);
                }
                Y[i] = y * (enters * s.back * p.scale);
            };
            const auto leaves = [&](const int i) { return lds_ld<f32x4>(sc + Scalars::LEAVE + 64 * i + 16 * grp); };
            const auto columns = [&](const int t, const int k) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = Rows<D>::col(K, lane, t + e, k);
            };
            const auto advance = [&](const Beside<E, 2>& u, const int t, const float by) {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = mma32<E>(x[e], u.lo(0), zero4());
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = mma32<E>(x[e], u.hi(0), z[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) S[t + e] = by * S[t + e] + z[e] * u.back;
            };
            queries(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Z[i] = beta[i] * (four_of<E>(v[i]) - enter[i] * s.back * Z[i]);
            }
            U[0] = mma16(inv0, split<bf16_t>(Z[0]), zero4());
            outputs(0);
            in_order();
            queries(1);
            const Two32 a2 = Lower<1>::two(A, lane, 2, 0);
            const Two p00 = Lower<0>::one(P, lane, 0, 0);
            in_order();
            u0 = split<bf16_t>(U[0]);
            Z[1] = mma16(a10, u0, Z[1]);
            outputs(1);
            in_order();
            queries(2);
            const Two32 a3 = Lower<1>::two(A, lane, 3, 0);
            const Two inv2 = Diagonal::row(inv, lane, 2);
            in_order();
            U[1] = mma16(inv1, split<bf16_t>(Z[1]), zero4());
            outputs(2);
            Y[0] = mma16(u0, p00, Y[0]);
            in_order();
            queries(3);
            const f32x4 l0 = leaves(0), l1 = leaves(1);
            const Two32 p1 = Lower<0>::two(P, lane, 1, 0);
            in_order();
            u1 = split<bf16_t>(U[1]);
            const Two32 u01 = join(u0, u1);
            Z[2] = mma32(a2, u01, Z[2]);
            Z[3] = mma32(a3, u01, Z[3]);
            Beside<E, 2> x01, x23;
            x01.take({l0 * U[0], l1 * U[1]});
            in_order();
            const Two a32 = Lower<1>::one(A, lane, 3, 1), inv3 = Diagonal::row(inv, lane, 3);
            in_order();
            U[2] = mma16(inv2, split<bf16_t>(Z[2]), zero4());
            outputs(3);
            columns(0, 0);
            Y[1] = mma32(u01, p1, Y[1]);
            in_order();
            const Two32 p2 = Lower<0>::two(P, lane, 2, 0), p3 = Lower<0>::two(P, lane, 3, 0);
            const f32x4 l2 = leaves(2), l3 = leaves(3);
            u2 = split<bf16_t>(U[2]);
            Z[3] = mma16(a32, u2, Z[3]);
            advance(x01, 0, whole);
            if constexpr (D == 128) columns(4, 0);
            in_order();
            U[3] = mma16(inv3, split<bf16_t>(Z[3]), zero4());
            if constexpr (D == 128) advance(x01, 4, whole);
            columns(0, 1);
            const Two p22 = Lower<0>::one(P, lane, 2, 1);
            Y[2] = mma32(u01, p2, Y[2]);
            Y[3] = mma32(u01, p3, Y[3]);
            in_order();
            x23.take({l2 * U[2], l3 * U[3]});
            advance(x23, 0, 1.f);
            if constexpr (D == 128) columns(4, 1);
            const Two32 p33 = Lower<0>::two(P, lane, 3, 1);
            in_order();
            if constexpr (D == 128) advance(x23, 4, 1.f);
            Y[2] = mma16(u2, p22, Y[2]);
            u3 = split<bf16_t>(U[3]);
            Y[3] = mma32(join(u2, u3), p33, Y[3]);
            if (p.saved && c0 < N) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4*>(updates + tiles.update(wide(hb) * chunks + c, ct, i) + 4 * lane) = U[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = c * DELTA_CHUNK + 16 * i + col;
                if (t < T && c0 + 4 * grp < N) *reinterpret_cast<u32x2*>(y + wide(t) * p.H * N) = u32x2{pack2<E>(Y[i][0], Y[i][1]), pack2<E>(Y[i][2], Y[i][3])};
            }
            __syncthreads();
        }
        if (on)
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * grp + r < N) p.sT[wide(hb) * N * N + (16 * t + 4 * grp + r) * N + c0 + col] = S[t][r];
        return;
    }

    // the helpers
    const int tid = threadIdx.x - 64 * SW, mine = wave - SW;
    constexpr int LANES = 64 * HELPERS, KP = (64 * D / 8 + LANES - 1) / LANES, VP = (64 * 2 * SW + LANES - 1) / LANES;       // pieces of 16 bytes a lane
    const E *q = static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh, *k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh, *v = static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh;
    const E *g = static_cast<const E*>(p.g) + b * p.g_sb + h, *beta = static_cast<const E*>(p.beta) + b * p.beta_sb + h;
    u32x4 kr[KP], qr[KP], vr[VP];
    const auto load = [&](const int c) {
        const int t0 = c * DELTA_CHUNK;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int x = tid + LANES * i, row = x / (D / 8), d = 8 * (x % (D / 8));
            const bool ok = t0 + row < T && d < N;
            kr[i] = ok ? *reinterpret_cast<const u32x4*>(k + wide(t0 + row) * p.k_st + d) : u32x4{0, 0, 0, 0};
            qr[i] = ok ? *reinterpret_cast<const u32x4*>(q + wide(t0 + row) * p.q_st + d) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int x = tid + LANES * i, row = x / (2 * SW), d = 16 * SW * piece + 8 * (x % (2 * SW));
            vr[i] = row < 64 && t0 + row < T && d < N ? *reinterpret_cast<const u32x4*>(v + wide(t0 + row) * p.v_st + d) : u32x4{0, 0, 0, 0};
        }
    };
    E gate, bt;                                                  // (as they come: what is made of them here would wait for them)
    int doc, before;
    const auto load_scalars = [&](const int c) {
        const int t = min(c * DELTA_CHUNK + lane, T - 1);
        gate = g[t * p.g_st];
        bt = beta[t * p.beta_st];
        if (p.doc) doc = p.doc[wide(b) * T + t], before = p.doc[wide(b) * T + max(t - 1, 0)];
    };
    uint64_t real;
    const auto scalars = [&](const int c) {
        const int t = c * DELTA_CHUNK + lane;
        const bool is = t < T && (!p.doc || doc >= 0);
        real = __ballot(is);
        if (mine == HELPERS - 1) make_scalars(lds + L::SCALARS + c % 3 * Scalars::BYTES, lane, {is, is && p.doc && t > 0 && doc != before}, to_f(gate), to_f(bt));   // (the wave with the fewest blocks)
    };
    static_assert(64 * D / 8 % LANES == 0);
    const auto put = [&](const int c) {
        const lds_t rows = lds + (c & 1) * L::STAGE;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int x = tid + LANES * i, row = x / (D / 8), d = x % (D / 8);
            const bool ok = real >> row & 1;
            Rows<D>::put(rows + L::K, row, d, ok ? kr[i] : u32x4{0, 0, 0, 0});
            Rows<D>::put(rows + L::Q, row, d, ok ? qr[i] : u32x4{0, 0, 0, 0});
        }
    };
    const auto put_values = [&] {
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int x = tid + LANES * i, row = x / (2 * SW), d = x % (2 * SW);
            if (row < 64) lds_st(lds + L::V + row * L::VPITCH + 16 * d, real >> row & 1 ? vr[i] : u32x4{0, 0, 0, 0});
        }
    };
    const auto matrices = [&](const int c) {
        const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE;
        make_matrices<E, D, HELPERS, false>(rows + L::K, rows + L::Q, lds + L::SCALARS + c % 3 * Scalars::BYTES, mats + L::A, mats + L::P, mats + L::INV, mine, lane, p.scale);
    };
    load_scalars(0);
    load(0);
    scalars(0);
    if (chunks > 1) load_scalars(1);
    put(0);
    put_values();
    if (chunks > 1) load(1), scalars(1);
    if (chunks > 2) load_scalars(2);
    __syncthreads();
    matrices(0);
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        const bool more = c + 1 < chunks;
        if (more) put(c + 1);
        __syncthreads();
        if (more) {
            put_values();                                        // (the state's waves have read this chunk's)
            if (c + 2 < chunks) load(c + 2);
            matrices(c + 1);
            if (c + 2 < chunks) scalars(c + 2);
            if (c + 3 < chunks) load_scalars(c + 3);
        }
        __syncthreads();
    }
}

template <class E, int D, int SW, int HELPERS> int run(hipStream_t st, const rwkv_delta_args& p) {
    const int pieces = (p.N + 16 * SW - 1) / (16 * SW);
    const int64_t blocks = (static_cast<int64_t>(p.B) * p.H + 7) / 8 * 8 * pieces;
    if (blocks > INT_MAX) return RWKV_ERR_SHAPE;
    hipLaunchKernelGGL((delta_fwd<E, D, SW, HELPERS>), dim3(static_cast<unsigned>(blocks)), dim3(64 * (SW + HELPERS)), 0, st, p, pieces);
    return launch_status();
}
// Columns a workgroup has: as many as leave a workgroup for every CU, so that matrices are made as seldom as may be.
template <class E, int D> int run_any(hipStream_t st, const rwkv_delta_args& p) {
    const int64_t heads = static_cast<int64_t>(p.B) * p.H, tiles = (p.N + 15) / 16;
    const auto enough = [&](int sw) { return heads * ((tiles + sw - 1) / sw) >= 256; };
    constexpr int HELPERS = D == 64 ? 8 : 4;
    if (enough(4)) return run<E, D, 4, HELPERS>(st, p);
    if (enough(2)) return run<E, D, 2, HELPERS>(st, p);
    return run<E, D, 1, HELPERS>(st, p);
}

}  // namespace

int launch_delta_fwd(hipStream_t st, const rwkv_delta_args& p) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run_any<bf16_t, 64>(st, p) : run_any<bf16_t, 128>(st, p);
    return p.N <= 64 ? run_any<half_t, 64>(st, p) : run_any<half_t, 128>(st, p);
}

}  // namespace rwkv
