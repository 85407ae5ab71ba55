// What the attentions over paged caches share (paged.hip, paged8.hip): the way a sequence is cut into pieces, the places of values in LDS, and the kernel that joins the pieces.
#pragma once

#include <algorithm>
#include <climits>

#include "attn_tile.h"

namespace rwkv {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
constexpr int STEP = 32, WAVES = 4, HEADS = 16;

template <class E> DEVINL f32x4_t mma16(const u32x4 a, const u32x4 b, const f32x4_t c) {
    if constexpr (std::is_same_v<E, bf16_t>) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
// Tokens of a sequence, and how many of them a piece has: `pieces` of them hold all, none of less than a round of the waves.
template <class Args> DEVINL int tokens_of(const Args& p, const int b, const int shift) { return static_cast<int>(min(wide(p.lens[b]), wide(p.M) << shift)); }
DEVINL int piece_of(const int n, const int pieces) { return max(1, (n + pieces * STEP * WAVES - 1) / (pieces * STEP * WAVES)) * STEP * WAVES; }

// 32 rows of D values: piece c of row r at place c ^ swap(r), so that 16 rows of two pieces are spread over all banks
template <int D> DEVINL lds_t value_at(const int r, const int c) { return r * 2 * D + ((c ^ (D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3))) << 4); }

// joins the pieces of a head: 256 threads, four channels a thread, the pieces dealt out.  A piece is its maximum, sum and (APART: what the sum's terms are relative to, with the outputs' maximum beside it) output.
template <class Args, class E, int D, bool APART = false> __global__ __launch_bounds__(256) void paged_join(const Args p, const int shift, const int pieces, const float* part) {
    constexpr int LANES = D / 4, SETS = 256 / LANES;
    __shared__ __align__(16) float sums[SETS][D];
    __shared__ float total[SETS], tops[4], refs[4];
    const int h = blockIdx.x, b = blockIdx.y, c = threadIdx.x % LANES, set = threadIdx.x / LANES;
    const int n = tokens_of(p, b, shift), size = piece_of(n, pieces), used = n <= 0 ? 0 : (n + size - 1) / size;
    const int64_t row = wide(b) * p.H + h;
    const float* from = part + row * pieces * (D + 4);
    float top = threadIdx.x < used ? from[wide(threadIdx.x) * (D + 4)] : -INFINITY, ref = APART && threadIdx.x < used ? from[wide(threadIdx.x) * (D + 4) + 2] : -INFINITY;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
        top = fmaxf(top, __shfl_xor(top, x, 64));
        if (APART) ref = fmaxf(ref, __shfl_xor(ref, x, 64));
    }
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top, refs[threadIdx.x >> 6] = ref;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    ref = fmaxf(fmaxf(refs[0], refs[1]), fmaxf(refs[2], refs[3]));
    const float base = top == -INFINITY ? 0.f : top, low = ref == -INFINITY ? 0.f : ref;
    f32x4_t y = f32x4_t{};
    float sum = 0.f;
    for (int i = set; i < used; i += SETS) {
        const float* x = from + wide(i) * (D + 4);
        const float f = __builtin_amdgcn_exp2f(x[0] - base);
        sum = fmaf(x[1], APART ? __builtin_amdgcn_exp2f(x[2] - low) : f, sum);
        if (4 * c < p.N) y += *reinterpret_cast<const f32x4_t*>(x + 4 + 4 * c) * f;
    }
    *reinterpret_cast<f32x4_t*>(&sums[set][4 * c]) = y;
    if (c == 0) total[set] = sum;
    __syncthreads();
    if (set == 0 && 4 * c < p.N) {
        for (int k = 1; k < SETS; ++k) {
            y += *reinterpret_cast<const f32x4_t*>(&sums[k][4 * c]);
            sum += total[k];
        }
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        const float g = APART ? __builtin_amdgcn_exp2f(0.5f * (base - low)) : 1.f;
        if (APART) y = y * f * g * g;
        if (APART) *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + row * p.N + 4 * c) = u32x2{pack2<E>(y[0], y[1]), pack2<E>(y[2], y[3])};
        else *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + row * p.N + 4 * c) = u32x2{pack2<E>(y[0] * f, y[1] * f), pack2<E>(y[2] * f, y[3] * f)};
    }
}

// How many pieces a sequence is cut into (the lengths are on the GPU: by what the table has room for): as many workgroups as keep the card busy, none with less than a
// round of its waves.
constexpr int BUSY = 2048, MAX_PIECES = 256;                     // (as many as paged_join has threads)
inline int chunks_of(int H, int Hk) { return (H / Hk + HEADS - 1) / HEADS; }
inline int pieces_of(int B, int H, int Hk, int page, int M) {
    const int64_t rounds = (static_cast<int64_t>(M) * page + STEP * WAVES - 1) / (STEP * WAVES), blocks = static_cast<int64_t>(B) * Hk * chunks_of(H, Hk);
    return static_cast<int>(std::max<int64_t>(1, std::min({rounds, (BUSY + blocks - 1) / blocks, static_cast<int64_t>(MAX_PIECES)})));
}
inline int width_of(int N) { return N <= 64 ? 64 : 128; }

}  // namespace
}  // namespace rwkv
