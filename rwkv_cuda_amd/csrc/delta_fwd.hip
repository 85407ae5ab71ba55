// Gated delta rule, whole sequences, forward (formulas and layouts: delta.h).
//
// A workgroup has 16 SW of a head's value channels and walks through the sequence, a chunk of 64 tokens after the other.  SW waves keep 16 columns of the state each and do what
// depends on it; the others bring the next chunk's inputs and make its matrices meanwhile: -A, P and the inverses of the blocks of I + A on the diagonal, with which the triangular system is
// four steps of products.  Two barriers a chunk: before the first the next chunk's rows go to LDS, behind it they are read.
// A chunk takes what its walking wave's instructions take, some 560 (heads of 64) or 780 (of 128) at 5 to 6 cycles, 80 to 130 of them products; where a workgroup has four tiles, its SIMDs' issue.  bf16: 32768 tokens
// of 32 heads of 128 1150 us, 2.25 a chunk; B8 T4096 H32 N64 190 to 200 us, with states and updates kept 230 to 245.
#include <algorithm>

#include "delta.h"

namespace rwkv {
namespace {

template <class E, int D, int SW, int HELPERS, bool PARTS>
__global__ __launch_bounds__(64 * (SW + HELPERS), 1) void delta_fwd(const rwkv_delta_args p, const int pieces) {
    using L = WalkPlace<D, SW, false>;
    __shared__ __align__(16) char smem[L::BYTES];
    const lds_t lds = lds_of(smem);
    // the pieces of a head are neighbours on one XCD: they read the same keys and queries
    const int slot = blockIdx.x >> 3, piece = slot % pieces, segment = PARTS ? slot / pieces % 2 : 0, hb = slot / pieces / (PARTS ? 2 : 1) * 8 + (blockIdx.x & 7);
    if (hb >= p.B * p.H) return;
    const int b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk), N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;

    // the chunks of this workgroup, and whether the first of them is its own
    int start = 0, count = chunks;
    bool first_own = true;
    if constexpr (PARTS) {
        __shared__ int best;
        const int at = split_at(p.doc + wide(b) * T, T, chunks, &best);
        if (at < 0 || at == chunks - 1) {
            if (segment == 1) return;
        } else if (segment == 0) count = at + 1;
        else start = at, count = chunks - at, first_own = false;
    }

    if (wave < SW) {
        const int ct = piece * SW + wave, c0 = 16 * ct;          // its columns
        const DeltaTiles tiles(p);
        float *states = static_cast<float*>(p.saved), *updates = states + tiles.states();
        const bool on = c0 + col < N;
        f32x4 S[D / 16];
        const float* s0 = p.s0 && first_own ? p.s0 + wide(hb) * N * N : nullptr;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = s0 && on && 16 * t + 4 * grp + r < N ? no_infinity<E>(s0[(16 * t + 4 * grp + r) * N + c0 + col]) : 0.f;
        const lds_t vread = L::V + lds + (4 * grp + (col >> 2)) * L::VPITCH + 32 * wave + 8 * (col & 3);
        // outputs: a chunk's place, and a lane's in it
        const int row_bytes = p.H * N * 2;
        char* const yc = reinterpret_cast<char*>(static_cast<E*>(p.y) + (wide(b) * T * p.H + h) * N + c0);
        const uint32_t y_lane = static_cast<uint32_t>(col) * row_bytes + 8 * grp;
        __syncthreads();
        __syncthreads();
        for (int c = 0; c < count; ++c) {
            const int at = start + c;
            const bool own = !PARTS || first_own || c > 0;
            const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE, sc = lds + L::SCALARS + c % 3 * Scalars::BYTES;
            const lds_t K = rows + L::K, Q = rows + L::Q, A = mats + L::A, P = mats + L::P, inv = mats + L::INV;
            typedef v4s __attribute__((address_space(3))) * ptr;
            if (p.saved && c0 < N && own) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
                    if (t < tiles.tiles) *reinterpret_cast<f32x4*>(states + tiles.state(wide(hb) * chunks + at, ct, t) + 4 * lane) = S[t];
            }
            // what a step reads from LDS is on its way a step earlier
            const Two inv0 = Diagonal::row(inv, lane, 0), a10 = Lower<1>::one(A, lane, 1, 0), inv1 = Diagonal::row(inv, lane, 1);
            f32x4 enter[4], Z[4];
            u32x2 v[4];
            Beside<E, D / 16> s;
            u32x4 x[4], kx[D / 32][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(vread + 16 * i * L::VPITCH)));
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) kx[k][i] = Rows<D>::row(K, lane, i, k);
#pragma unroll
            for (int i = 0; i < 4; ++i) enter[i] = lds_ld<f32x4>(sc + Scalars::ENTER + 64 * i + 16 * grp);
            in_order();
            s.take(S);
            __syncthreads();                                     // (the values have been read)
#pragma unroll
            for (int i = 0; i < 4; ++i) Z[i] = mma32<E>(kx[0][i], s.lo(0), zero4());
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                if (k > 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i) Z[i] = mma32<E>(kx[k][i], s.lo(k), Z[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) Z[i] = mma32<E>(kx[k][i], s.hi(k), Z[i]);
            }
            in_order();
            // the triangular system, and beside it the outputs
            f32x4 Y[4], U[4], z[4];
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
            u32x4 kc[D / 16];
            const auto columns = [&](const int k) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) kc[t] = Rows<D>::col(K, lane, t, k);
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
            queries(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Z[i] = four_of<E>(v[i]) - enter[i] * s.back * Z[i];
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
            columns(0);
            Y[1] = mma32(u01, p1, Y[1]);
            in_order();
            const Two32 p2 = Lower<0>::two(P, lane, 2, 0), p3 = Lower<0>::two(P, lane, 3, 0);
            const f32x4 l2 = leaves(2), l3 = leaves(3);
            u2 = split<bf16_t>(U[2]);
            Z[3] = mma16(a32, u2, Z[3]);
            advance(x01, whole);
            in_order();
            U[3] = mma16(inv3, split<bf16_t>(Z[3]), zero4());
            columns(1);
            const Two p22 = Lower<0>::one(P, lane, 2, 1);
            Y[2] = mma32(u01, p2, Y[2]);
            Y[3] = mma32(u01, p3, Y[3]);
            in_order();
            x23.take({l2 * U[2], l3 * U[3]});
            advance(x23, one);
            const Two32 p33 = Lower<0>::two(P, lane, 3, 1);
            in_order();
            Y[2] = mma16(u2, p22, Y[2]);
            u3 = split<bf16_t>(U[3]);
            Y[3] = mma32(join(u2, u3), p33, Y[3]);
            if (p.saved && c0 < N && own) {
                float* to = updates + tiles.update(wide(hb) * chunks + at, ct, 0) + 4 * lane;
                keep(to, u0), keep(to + 256, u1), keep(to + 512, u2), keep(to + 768, u3);
            }
            char* const to = yc + wide(at) * DELTA_CHUNK * row_bytes;
            const auto out = [&](const int i) { *reinterpret_cast<u32x2*>(to + wide(16 * i) * row_bytes + y_lane) = u32x2{pack2<E>(Y[i][0], Y[i][1]), pack2<E>(Y[i][2], Y[i][3])}; };
            if (own && (at + 1) * DELTA_CHUNK <= T && c0 + 16 <= N)
#pragma unroll
                for (int i = 0; i < 4; ++i) out(i);
            else if (own)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at * DELTA_CHUNK + 16 * i + col < T && c0 + 4 * grp < N) out(i);
            __syncthreads();
        }
        if (c0 < N && __ballot(!finite(S[0][0])) != 0ull &&         // something that is no number is in all of its column by now
            walk_by_token<E, D, false>((DeltaArguments*)__builtin_amdgcn_kernarg_segment_ptr(), hb, start, count, c0, !PARTS || first_own, static_cast<float*>(p.saved), updates)) return;
        if (on && start + count == chunks)
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * grp + r < N) p.sT[wide(hb) * N * N + (16 * t + 4 * grp + r) * N + c0 + col] = S[t][r];
        return;
    }

    help<E, D, SW, HELPERS, false>(p, lds, b, h, hk, piece, wave - SW, lane, start, count);
}

template <class E, int D> int run(hipStream_t st, const rwkv_delta_args& p) {
    return walk_width(p, p.s0, p.sT, [&](auto sw, auto parts) {
        constexpr int SW = decltype(sw)::value;
        constexpr bool PARTS = decltype(parts)::value;
        const int pieces = (p.N + 16 * SW - 1) / (16 * SW);
        const int64_t blocks = (static_cast<int64_t>(p.B) * p.H + 7) / 8 * 8 * pieces * (PARTS ? 2 : 1);
        if (blocks > INT_MAX) return static_cast<int>(RWKV_ERR_SHAPE);
        hipLaunchKernelGGL((delta_fwd<E, D, SW, 8 - SW, PARTS>), dim3(static_cast<unsigned>(blocks)), dim3(512), 0, st, p, pieces);
        return launch_status();
    });
}

}  // namespace

int launch_delta_fwd(hipStream_t st, const rwkv_delta_args& p) {
    if (p.dtype == RWKV_DTYPE_BF16) return p.N <= 64 ? run<bf16_t, 64>(st, p) : run<bf16_t, 128>(st, p);
    return p.N <= 64 ? run<half_t, 64>(st, p) : run<half_t, 128>(st, p);
}

}  // namespace rwkv
