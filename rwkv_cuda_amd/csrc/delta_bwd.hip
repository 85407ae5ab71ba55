// Gated delta rule, whole sequences, the backward's walk (formulas and layouts: delta.h).
//
// As delta_fwd.hip, from the last chunk to the first: a workgroup has 16 SW value channels of a head's state gradient dS.  Of each chunk it leaves dS as it leaves the chunk and dZ, the gradient
// of the triangular system's right side, in memory; the gradients of the inputs, whose sums run over all value channels, are delta_grads.hip's.
#include <algorithm>

#include "delta.h"

namespace rwkv {
namespace {

// a b + c with b the gradients of four tokens as they came: one number of bf16, or of fp16 made two
template <class E> struct Gradients {
    Two x;
    DEVINL explicit Gradients(const u32x2 v) {
        if constexpr (std::is_same_v<E, bf16_t>) x = {v, v};
        else x = split<bf16_t>(four_of<E>(v));
    }
};
template <class E> DEVINL f32x4 gradients16(const Two& a, const Gradients<E>& b, const f32x4 c) {
    if constexpr (std::is_same_v<E, bf16_t>) return mma32<bf16_t>(join(a.h, a.l), join(b.x.h, b.x.h), c);
    else return mma16(a, b.x, c);
}
template <class E> DEVINL f32x4 gradients32(const Two32& a, const Gradients<E>& b, const Gradients<E>& d, f32x4 c) {
    if constexpr (std::is_same_v<E, bf16_t>) {
        c = mma32<bf16_t>(a.l, join(b.x.h, d.x.h), c);
        return mma32<bf16_t>(a.h, join(b.x.h, d.x.h), c);
    } else return mma32(a, join(b.x, d.x), c);
}

template <class E, int D, int SW, int HELPERS>
__global__ __launch_bounds__(64 * (SW + HELPERS), 1) void delta_bwd(const rwkv_delta_args p, const int pieces, float* states, float* updates) {
    using L = WalkPlace<D, SW, true>;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    const int slot = blockIdx.x >> 3, piece = slot % pieces, hb = slot / pieces * 8 + (blockIdx.x & 7);
    if (hb >= p.B * p.H) return;
    const int b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk), N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;

    if (wave < SW) {
        const int ct = piece * SW + wave, c0 = 16 * ct;
        const bool on = c0 + col < N;
        const DeltaTiles tiles(p);
        f32x4 S[D / 16];                                         // dS
        const float* end = p.dsT ? p.dsT + wide(hb) * N * N : nullptr;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = end && on && 16 * t + 4 * grp + r < N ? end[(16 * t + 4 * grp + r) * N + c0 + col] : 0.f;
        const lds_t vread = L::V + lds + (4 * grp + (col >> 2)) * L::VPITCH + 32 * wave + 8 * (col & 3);
        __syncthreads();
        __syncthreads();
        for (int c = 0; c < chunks; ++c) {
            const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE, sc = lds + L::SCALARS + c % 3 * Scalars::BYTES;
            const lds_t K = rows + L::K, Q = rows + L::Q, A = mats + L::A, P = mats + L::P, inv = mats + L::INV;
            const int64_t chunk = wide(hb) * chunks + chunks - 1 - c;
            typedef v4s __attribute__((address_space(3))) * ptr;
            if (c0 < N) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
                    if (t < tiles.tiles) *reinterpret_cast<f32x4*>(states + tiles.state(chunk, ct, t) + 4 * lane) = S[t];
            }
            u32x2 v[4];
            Beside<E, D / 16> s;
            u32x4 x[4];
            f32x4 X[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(vread + 16 * i * L::VPITCH)));
                x[i] = Rows<D>::row(K, lane, i, 0);
            }
            in_order();
            s.take(S);
            __syncthreads();                                     // (the gradients of y have been read)
#pragma unroll
            for (int i = 0; i < 4; ++i) X[i] = mma32<E>(x[i], s.lo(0), zero4());
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                u32x4 next[4];
                if (k + 1 < D / 32)
#pragma unroll
                    for (int i = 0; i < 4; ++i) next[i] = Rows<D>::row(K, lane, i, k + 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) X[i] = mma32<E>(x[i], s.hi(k), X[i]);
                if (k + 1 < D / 32)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = next[i], X[i] = mma32<E>(x[i], s.lo(k + 1), X[i]);
                in_order();
            }
            const Gradients<E> d0(v[0]), d1(v[1]), d2(v[2]), d3(v[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) X[i] *= lds_ld<f32x4>(sc + Scalars::LEAVE + 64 * i + 16 * grp) * s.back;
            X[3] = gradients16(Upper<0>::one(P, lane, 3, 3), d3, X[3]);
            X[2] = gradients32(Upper<0>::two(P, lane, 2, 1), d2, d3, X[2]);
            // the triangular system; dS: what the queries leave, then what the keys take
            f32x4 z[4];
            const float whole = lds_ld<float>(sc + Scalars::ENTER + 4 * 63);
            const auto factors = [&](const int i) { return lds_ld<f32x4>(sc + Scalars::ENTER + 64 * i + 16 * grp); };
            const auto of_y = [&](const int i) { return four_of<E>(v[i]) * factors(i) * p.scale; };
            const auto of_z = [&](const int i, const f32x4 dz) { return dz * factors(i) * -lds_ld<f32x4>(sc + Scalars::BETA + 64 * i + 16 * grp); };
            const auto advance = [&](const lds_t from, const Beside<E, 2>& u, const int k, const float by) {
#pragma unroll
                for (int t = 0; t < D / 16; t += 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = Rows<D>::col(from, lane, t + e, k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = mma32<E>(x[e], u.lo(0), zero4());
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = mma32<E>(x[e], u.hi(0), z[e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[t + e] = by * S[t + e] + z[e] * u.back;
                }
            };
            const auto leave = [&](const int i, const f32x4 dz) {
                if (c0 < N) *reinterpret_cast<f32x4*>(updates + tiles.update(chunk, ct, i) + 4 * lane) = dz;
            };
            f32x4 Z[4];
            Beside<E, 2> w;
            Z[3] = mma16(Diagonal::row(inv, lane, 3), split<bf16_t>(X[3]), zero4());
            X[1] = gradients16(Upper<0>::one(P, lane, 1, 1), d1, X[1]);
            X[1] = gradients32(Upper<0>::two(P, lane, 1, 1), d2, d3, X[1]);
            w.take({of_y(2), of_y(3)});
            advance(Q, w, 1, whole);
            in_order();
            const Two z3 = split<bf16_t>(Z[3]);
            X[2] = mma16(Upper<1>::one(A, lane, 2, 3), z3, X[2]);
            X[0] = gradients32(Upper<0>::two(P, lane, 0, 0), d0, d1, X[0]);
            X[0] = gradients32(Upper<0>::two(P, lane, 0, 1), d2, d3, X[0]);
            in_order();
            Z[2] = mma16(Diagonal::row(inv, lane, 2), split<bf16_t>(X[2]), zero4());
            w.take({of_y(0), of_y(1)});
            advance(Q, w, 0, 1.f);
            in_order();
            const Two z2 = split<bf16_t>(Z[2]);
            const Two32 z23 = join(z2, z3);
            X[1] = mma32(Upper<1>::two(A, lane, 1, 1), z23, X[1]);
            X[0] = mma32(Upper<1>::two(A, lane, 0, 1), z23, X[0]);
            leave(3, Z[3]);
            in_order();
            Z[1] = mma16(Diagonal::row(inv, lane, 1), split<bf16_t>(X[1]), zero4());
            leave(2, Z[2]);
            w.take({of_z(2, Z[2]), of_z(3, Z[3])});
            advance(K, w, 1, 1.f);
            in_order();
            const Two z1 = split<bf16_t>(Z[1]);
            X[0] = mma16(Upper<1>::one(A, lane, 0, 1), z1, X[0]);
            leave(1, Z[1]);
            in_order();
            Z[0] = mma16(Diagonal::row(inv, lane, 0), split<bf16_t>(X[0]), zero4());
            in_order();
            w.take({of_z(0, Z[0]), of_z(1, Z[1])});
            advance(K, w, 0, 1.f);
            leave(0, Z[0]);
            __syncthreads();
        }
        if (on && p.ds0)
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * grp + r < N) p.ds0[wide(hb) * N * N + (16 * t + 4 * grp + r) * N + c0 + col] = S[t][r];
        return;
    }

    help<E, D, SW, HELPERS, true>(p, lds, b, h, hk, piece, wave - SW, lane);
}

template <class E, int D> int run(hipStream_t st, const rwkv_delta_args& p, float* dS, float* dZ) {
    return walk_width(p, [&](auto sw) {
        constexpr int SW = decltype(sw)::value;
        const int pieces = (p.N + 16 * SW - 1) / (16 * SW);
        const int64_t blocks = (static_cast<int64_t>(p.B) * p.H + 7) / 8 * 8 * pieces;
        if (blocks > INT_MAX) return static_cast<int>(RWKV_ERR_SHAPE);
        hipLaunchKernelGGL((delta_bwd<E, D, SW, 8 - SW>), dim3(static_cast<unsigned>(blocks)), dim3(512), 0, st, p, pieces, dS, dZ);
        return launch_status();
    });
}

}  // namespace

int launch_delta_bwd(hipStream_t st, const rwkv_delta_args& p, float* dS, float* dZ) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run<bf16_t, 64>(st, p, dS, dZ) : run<bf16_t, 128>(st, p, dS, dZ);
    return p.N <= 64 ? run<half_t, 64>(st, p, dS, dZ) : run<half_t, 128>(st, p, dS, dZ);
}

}  // namespace rwkv
