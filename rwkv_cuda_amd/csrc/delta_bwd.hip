// Gated delta rule, whole sequences, the backward's walk (formulas and layouts: delta.h).
//
// As delta_fwd.hip, from the last chunk to the first: a workgroup has 16 SW value channels of a head's state gradient dS.  Of each chunk it leaves dS as it leaves the chunk and dZ, the gradient
// of the triangular system's right side, in memory; the gradients of the inputs, whose sums run over all value channels, are delta_grads.hip's.  Bound as the forward: B8 T4096 H32 N64 bf16 220 to 235 us,
// 3001 tokens of 32 heads of 128 fp16 165 us, 3.5 a chunk, in five documents 108.
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

template <class E, int D, int SW, int HELPERS, bool PARTS>
__global__ __launch_bounds__(64 * (SW + HELPERS), 1) void delta_bwd(const rwkv_delta_args p, const int pieces, float* states, float* updates) {
    using L = WalkPlace<D, SW, true>;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    const int slot = blockIdx.x >> 3, piece = slot % pieces, segment = PARTS ? slot / pieces % 2 : 0, hb = slot / pieces / (PARTS ? 2 : 1) * 8 + (blockIdx.x & 7);
    if (hb >= p.B * p.H) return;
    const int b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk), N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;

    // the chunks of this workgroup, downwards, and whether the first of them is its own
    int start = chunks - 1, count = chunks;
    bool first_own = true;
    if constexpr (PARTS) {
        __shared__ int best;
        const int at = split_at(p.doc + wide(b) * T, T, chunks, &best);
        if (at <= 0) {
            if (segment == 1) return;
        } else if (segment == 1) count = chunks - at;
        else start = at, count = at + 1, first_own = false;
    }

    if (wave < SW) {
        const int ct = piece * SW + wave, c0 = 16 * ct;
        const bool on = c0 + col < N;
        const DeltaTiles tiles(p);
        f32x4 S[D / 16];                                         // dS
        const float* end = p.dsT && first_own ? p.dsT + wide(hb) * N * N : nullptr;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = end && on && 16 * t + 4 * grp + r < N ? no_infinity<E>(end[(16 * t + 4 * grp + r) * N + c0 + col]) : 0.f;
        const lds_t vread = L::V + lds + (4 * grp + (col >> 2)) * L::VPITCH + 32 * wave + 8 * (col & 3);
        __syncthreads();
        __syncthreads();
        for (int c = 0; c < count; ++c) {
            const bool own = !PARTS || first_own || c > 0;
            const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE, sc = lds + L::SCALARS + c % 3 * Scalars::BYTES;
            const lds_t K = rows + L::K, Q = rows + L::Q, A = mats + L::A, P = mats + L::P, inv = mats + L::INV;
            const int64_t chunk = wide(hb) * chunks + start - c;
            typedef v4s __attribute__((address_space(3))) * ptr;
            if (c0 < N && own) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
                    if (t < tiles.tiles) *reinterpret_cast<f32x4*>(states + tiles.state(chunk, ct, t) + 4 * lane) = S[t];
            }
            // what a step reads from LDS is on its way a step earlier
            u32x2 v[4];
            Beside<E, D / 16> s;
            u32x4 kx[D / 32][4], kc[D / 16];
            f32x4 X[4], Z[4], z[4], leave[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(vread + 16 * i * L::VPITCH)));
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) kx[k][i] = Rows<D>::row(K, lane, i, k);
#pragma unroll
            for (int i = 0; i < 4; ++i) leave[i] = lds_ld<f32x4>(sc + Scalars::LEAVE + 64 * i + 16 * grp);
            in_order();
            s.take(S);
            __syncthreads();                                     // (the gradients of y have been read)
            const Two inv3 = Diagonal::row(inv, lane, 3), p33 = Upper<0>::one(P, lane, 3, 3);
            const Two32 p2 = Upper<0>::two(P, lane, 2, 1);
            const float whole = lds_ld<float>(sc + Scalars::ENTER + 4 * 63);
#pragma unroll
            for (int i = 0; i < 4; ++i) X[i] = mma32<E>(kx[0][i], s.lo(0), zero4());
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                if (k > 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i) X[i] = mma32<E>(kx[k][i], s.lo(k), X[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) X[i] = mma32<E>(kx[k][i], s.hi(k), X[i]);
            }
            in_order();
            // the triangular system; dS: what the queries leave, then what the keys take
            const Gradients<E> d0(v[0]), d1(v[1]), d2(v[2]), d3(v[3]);
            const auto factors = [&](const int i) { return lds_ld<f32x4>(sc + Scalars::ENTER + 64 * i + 16 * grp); };
            const auto betas = [&](const int i) { return lds_ld<f32x4>(sc + Scalars::BETA + 64 * i + 16 * grp); };
            const auto columns = [&](const lds_t from, const int k) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) kc[t] = Rows<D>::col(from, lane, t, k);
            };
            constexpr std::integral_constant<int, 1> one;
            const auto advance = [&](const Beside<E, 2>& u, const auto by) {
                if constexpr (std::is_same_v<E, bf16_t>) {
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) S[t] = mma32<E>(kc[t], u.lo(0), std::is_same_v<decltype(by), const std::integral_constant<int, 1>> ? S[t] : S[t] * static_cast<float>(by));
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) S[t] = mma32<E>(kc[t], u.hi(0), S[t]);
                } else
#pragma unroll
                for (int t = 0; t < D / 16; t += 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = mma32<E>(kc[t + e], u.lo(0), zero4());
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = mma32<E>(kc[t + e], u.hi(0), z[e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[t + e] = static_cast<float>(by) * S[t + e] + z[e] * u.back;
                }
            };
            Beside<E, 2> w;
            const Two p11 = Upper<0>::one(P, lane, 1, 1), a23 = Upper<1>::one(A, lane, 2, 3), inv2 = Diagonal::row(inv, lane, 2);
            const Two32 p1 = Upper<0>::two(P, lane, 1, 1);
            f32x4 fa = factors(2), fb = factors(3);
#pragma unroll
            for (int i = 0; i < 4; ++i) X[i] *= leave[i] * s.back;
            X[3] = gradients16(p33, d3, X[3]);
            X[2] = gradients32(p2, d2, d3, X[2]);
            Z[3] = mma16(inv3, split<bf16_t>(X[3]), zero4());
            w.take({no_infinity<E>(four_of<E>(v[2])) * fa * p.scale, no_infinity<E>(four_of<E>(v[3])) * fb * p.scale});
            in_order();
            columns(Q, 1);
            const Two32 a1 = Upper<1>::two(A, lane, 1, 1), a0 = Upper<1>::two(A, lane, 0, 1);
            const Two z3 = split<bf16_t>(Z[3]);
            X[2] = mma16(a23, z3, X[2]);
            X[1] = gradients16(p11, d1, X[1]);
            X[1] = gradients32(p1, d2, d3, X[1]);
            in_order();
            const Two32 p0 = Upper<0>::two(P, lane, 0, 0), p02 = Upper<0>::two(P, lane, 0, 1);
            const Two inv1 = Diagonal::row(inv, lane, 1);
            Z[2] = mma16(inv2, split<bf16_t>(X[2]), zero4());
            advance(w, whole);
            in_order();
            fa = factors(0), fb = factors(1);
            columns(Q, 0);
            const Two z2 = split<bf16_t>(Z[2]);
            const Two32 z23 = join(z2, z3);
            X[1] = mma32(a1, z23, X[1]);
            X[0] = mma32(a0, z23, X[0]);
            X[0] = gradients32(p0, d0, d1, X[0]);
            X[0] = gradients32(p02, d2, d3, X[0]);
            w.take({no_infinity<E>(four_of<E>(v[0])) * fa * p.scale, no_infinity<E>(four_of<E>(v[1])) * fb * p.scale});
            in_order();
            const Two a01 = Upper<1>::one(A, lane, 0, 1), inv0 = Diagonal::row(inv, lane, 0);
            f32x4 ba = betas(2) * factors(2), bb = betas(3) * factors(3);
            Z[1] = mma16(inv1, split<bf16_t>(X[1]), zero4());
            advance(w, one);
            in_order();
            columns(K, 1);
            const Two z1 = split<bf16_t>(Z[1]);
            X[0] = mma16(a01, z1, X[0]);
            w.take({Z[2] * -ba, Z[3] * -bb});
            in_order();
            ba = betas(0) * factors(0), bb = betas(1) * factors(1);
            Z[0] = mma16(inv0, split<bf16_t>(X[0]), zero4());
            advance(w, one);
            in_order();
            columns(K, 0);
            w.take({Z[0] * -ba, Z[1] * -bb});
            advance(w, one);
            if (c0 < N && own) {
                float* to = updates + tiles.update(chunk, ct, 0) + 4 * lane;
                keep(to, split<bf16_t>(Z[0])), keep(to + 256, z1), keep(to + 512, z2), keep(to + 768, z3);
            }
            __syncthreads();
        }
        if (c0 < N && __ballot(!finite(S[0][0])) != 0ull &&         // something that is no number is in all of its column by now
            walk_by_token<E, D, true>((DeltaArguments*)__builtin_amdgcn_kernarg_segment_ptr(), hb, start, count, c0, !PARTS || first_own, states, updates)) return;
        if (on && p.ds0 && start + 1 == count)
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * grp + r < N) p.ds0[wide(hb) * N * N + (16 * t + 4 * grp + r) * N + c0 + col] = S[t][r];
        return;
    }

    help<E, D, SW, HELPERS, true>(p, lds, b, h, hk, piece, wave - SW, lane, start, count);
}

template <class E, int D> int run(hipStream_t st, const rwkv_delta_args& p, float* dS, float* dZ) {
    return walk_width(p, p.dsT, p.ds0, [&](auto sw, auto parts) {
        constexpr int SW = decltype(sw)::value;
        constexpr bool PARTS = decltype(parts)::value;
        const int pieces = (p.N + 16 * SW - 1) / (16 * SW);
        const int64_t blocks = (static_cast<int64_t>(p.B) * p.H + 7) / 8 * 8 * pieces * (PARTS ? 2 : 1);
        if (blocks > INT_MAX) return static_cast<int>(RWKV_ERR_SHAPE);
        hipLaunchKernelGGL((delta_bwd<E, D, SW, 8 - SW, PARTS>), dim3(static_cast<unsigned>(blocks)), dim3(512), 0, st, p, pieces, dS, dZ);
        return launch_status();
    });
}

}  // namespace

int launch_delta_bwd(hipStream_t st, const rwkv_delta_args& p, float* dS, float* dZ) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run<bf16_t, 64>(st, p, dS, dZ) : run<bf16_t, 128>(st, p, dS, dZ);
    return p.N <= 64 ? run<half_t, 64>(st, p, dS, dZ) : run<half_t, 128>(st, p, dS, dZ);
}

}  // namespace rwkv
