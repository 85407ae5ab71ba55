// What the kernels of the gated delta rule share (its arguments are explained in rwkv_hip.h).
//
// 64 tokens at once.  With G the sum of the log decays since the chunk began, D_ij = e^(G_i - G_j), S the state that enters it and U the updates:
//   (I + A) U = beta (V - e^G K S)         A_ij = beta_i D_ij k_i.k_j  (i > j)
//   Y = scale e^G Q S + P U                P_ij = scale D_ij q_i.k_j   (i >= j)
//   S' = e^G_64 S + (e^(G_64 - G) K)^T U
// and backwards, with dS' of the state that leaves:
//   (I + A)^T dZ = P^T dY + e^(G_64 - G) K dS'
//   dS = e^G_64 dS' + scale (e^G Q)^T dY - (beta e^G K)^T dZ,   dV = beta dZ
// The value channels, columns of S, U and Z, do not depend on each other.  A wave keeps 16 of them all along: with them as the lane's index (lane & 15), what a product
// leaves (four rows a lane and tile of 16) is, split in two and packed, the operand of the next, whose contraction runs over those rows; nothing goes through LDS.  The other
// operand comes from there, 32 rows of a contraction in the order that this gives: 4 g .. 4 g + 3 and 16 + 4 g .. for the 16 lanes of group g.
//
// Operands that are inputs are bf16 or fp16 as they stand.  All others are two numbers of 16 bits, hi + lo: bf16 where both are such (three products, lo lo is left out: 2^-18 of
// the product at most), or, beside an fp16 input, fp16 times a power of two that brings the wave's largest to 2^9 .. 2^10.  The states' errors stay near 2^-17 so; with single
// bf16 operands they were 2^-9, as large as an output's own rounding, and an fp32 state that is passed on would lose 15 of its 24 bits.
#pragma once

#include "attn_tile.h"

namespace rwkv {

constexpr int DELTA_CHUNK = 64;                                 // tokens of a chunk
// A log decay below this is a decay of 0: e^-104 lies below half of fp32's least number.
constexpr float DELTA_NONE = -104.f;

// What becomes of a token: padding leaves the state as it is; a cut lets nothing of it through.
struct DeltaToken { bool real, cut; };
DEVINL DeltaToken delta_token(const int* doc, const int64_t row, const int t, const int T) {
    if (t >= T) return {false, false};
    if (doc == nullptr) return {true, false};
    const int d = doc[row + t];
    return {d >= 0, d >= 0 && t > 0 && doc[row + t - 1] != d};
}

// What the forward keeps for the backward, and the backward for its last kernel, of each head and chunk: the state that enters (whose gradient leaves) and the updates (their gradients), fp32, as
// the waves hold them: tiles of 16 by 16, four neighbouring rows of a column a lane, 16 bytes.  States: [column tile][row tile], updates [column tile][token tile].
struct DeltaTiles {
    int tiles;                                                  // of 16 channels
    int64_t chunks;                                             // all of them
    __host__ __device__ explicit DeltaTiles(const rwkv_delta_args& p) : DeltaTiles(p.B, p.T, p.H, p.N) {}
    __host__ __device__ DeltaTiles(int B, int T, int H, int N) : tiles((N + 15) / 16), chunks(static_cast<int64_t>(B) * H * ((T + DELTA_CHUNK - 1) / DELTA_CHUNK)) {}
    __host__ __device__ size_t states() const { return static_cast<size_t>(chunks) * tiles * tiles * 256; }       // floats
    __host__ __device__ size_t updates() const { return static_cast<size_t>(chunks) * tiles * 4 * 256; }
    __host__ __device__ int64_t state(const int64_t chunk, const int column, const int row) const { return ((chunk * tiles + column) * tiles + row) * 256; }
    __host__ __device__ int64_t update(const int64_t chunk, const int column, const int token) const { return ((chunk * tiles + column) * 4 + token) * 256; }
};
// delta_fwd.hip, delta_bwd.hip, delta_grads.hip (arguments checked)
int launch_delta_fwd(hipStream_t st, const rwkv_delta_args& p);
int launch_delta_bwd(hipStream_t st, const rwkv_delta_args& p, float* dS, float* dZ);
int launch_delta_grads(hipStream_t st, const rwkv_delta_args& p, const float* dS, const float* dZ, float* dq, float* dk);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

DEVINL f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
// v_mfma_f32_16x16x32: [row lane & 15 of a][column lane & 15 of b], four rows 4 (lane >> 4) .. a lane.  (Not 16x16x16 beside it: accumulators that both add to came out wrong now and
// then in a workgroup whose other waves used the matrix unit too.)
template <class E> DEVINL f32x4 mma32(const u32x4 a, const u32x4 b, const f32x4 c) {
    if constexpr (std::is_same_v<E, bf16_t>) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
DEVINL u32x4 join(const u32x2 a, const u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }

// What stands before it is issued before what stands behind: the steps of the triangular system wait for each other, and the products between them are there to fill that time.
DEVINL void in_order() { __builtin_amdgcn_sched_barrier(0); }

// four values of a tile as two numbers of 16 bits each
struct Two { u32x2 h, l; };
struct Two32 { u32x4 h, l; };
DEVINL Two32 join(const Two& a, const Two& b) { return {join(a.h, b.h), join(a.l, b.l)}; }
template <class E> DEVINL Two split(const f32x4 x) {
    Two o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h = pack2<E>(x[2 * i], x[2 * i + 1]);
        asm("" : "+v"(h));                                      // (or the compiler rounds each value once more to take it apart)
        o.h[i] = h;
        o.l[i] = pack2<E>(x[2 * i] - unpack_lo<E>(h), x[2 * i + 1] - unpack_hi<E>(h));
    }
    return o;
}
template <class E> DEVINL f32x4 four_of(const u32x2 v) { return f32x4{unpack_lo<E>(v[0]), unpack_hi<E>(v[0]), unpack_lo<E>(v[1]), unpack_hi<E>(v[1])}; }
// a b + c of two such operands, bf16, over a single tile: both small products in one instruction, the large one beside zeros
DEVINL f32x4 mma16(const Two& a, const Two& b, f32x4 c) {
    c = mma32<bf16_t>(join(a.h, a.l), join(b.l, b.h), c);
    return mma32<bf16_t>(join(u32x2{0, 0}, a.h), join(b.l, b.h), c);
}
DEVINL f32x4 mma32(const Two32& a, const Two32& b, f32x4 c) {
    c = mma32<bf16_t>(a.h, b.l, c);
    c = mma32<bf16_t>(a.l, b.h, c);
    return mma32<bf16_t>(a.h, b.h, c);
}
// the largest of a wave, in all lanes
DEVINL float wave_max(float x) {
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true)));   // row_ror 8, 4, 2, 1
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, true)));
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xf, 0xf, true)));
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xf, 0xf, true)));
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
// Tiles as operands beside an input of type E: bf16 as they are, fp16 times a power of two, whose inverse is what the product is to be multiplied with.
template <class E, int TILES> struct Beside {
    Two x[TILES];
    float back;
    DEVINL void take(const f32x4 (&v)[TILES]) {
        if constexpr (std::is_same_v<E, bf16_t>) {
            back = 1.f;
#pragma unroll
            for (int i = 0; i < TILES; ++i) x[i] = split<bf16_t>(v[i]);
        } else {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(v[i][r]));
            const int e = min(max(static_cast<int>(__float_as_uint(wave_max(top)) >> 23) - 127, -100), 120);
            const float by = __uint_as_float(static_cast<uint32_t>(127 + 9 - e) << 23);
            back = __uint_as_float(static_cast<uint32_t>(127 - 9 + e) << 23);
#pragma unroll
            for (int i = 0; i < TILES; ++i) x[i] = split<half_t>(v[i] * by);
        }
    }
    DEVINL u32x4 hi(const int s) const { return join(x[2 * s].h, x[2 * s + 1].h); }
    DEVINL u32x4 lo(const int s) const { return join(x[2 * s].l, x[2 * s + 1].l); }
};

// The scalars of a chunk's 64 tokens, by token, fp32.  Log decays are summed in 64 bits, to base 2, and their sums kept as two numbers: differences count.  A cut, or a decay of nothing, is one
// by 2^-(2^20): what crosses it is 0, and the others' differences stay exact to 2^-21.
struct Scalars {
    static constexpr lds_t SUM = 0, REST = 256, BETA = 512, ENTER = 768, LEAVE = 1024, TAIL = 1280, BYTES = 1536;      // TAIL: the decay up to the end of a token's block of 16, or (HEAD) since it began
};
constexpr double CUT = -0x1p20;

// 64 rows of D inputs in LDS, 16 bytes more than their size apart (16 rows at one place touch all banks).  Of every 32 channels number 16 e + 4 g + r is at place 8 g + 4 e + r: 16 bytes
// are what a lane of group g needs.
template <int D> struct Rows {
    static constexpr int PITCH = 2 * D + 16, BYTES = 64 * PITCH;
    // channels 8 c .. 8 c + 7 of a row
    static DEVINL void put(const lds_t base, const int row, const int c, const u32x4 x) {
        const lds_t to = base + row * PITCH + 64 * (c / 4) + 32 * (c % 2) + 8 * (c / 2 % 2);
        lds_st(to, u32x2{x[0], x[1]});
        lds_st(to + 16, u32x2{x[2], x[3]});
    }
    // four of a row's channels, 16 t + 4 g ..
    static DEVINL u32x2 four(const lds_t base, const int row, const int t, const int g) { return lds_ld<u32x2>(base + row * PITCH + 64 * (t / 2) + 16 * g + 8 * (t % 2)); }
    // row 16 i + (lane & 15), channels of the 32 s-th: the contraction runs over channels
    static DEVINL u32x4 row(const lds_t base, const int lane, const int i, const int s) { return lds_ld<u32x4>(base + (16 * i + (lane & 15)) * PITCH + 64 * s + 16 * (lane >> 4)); }
    // channel 16 t + (lane & 15), rows of the 32 s-th: the contraction runs over rows
    static DEVINL u32x4 col(const lds_t base, const int lane, const int t, const int s) {
        typedef v4s __attribute__((address_space(3))) * ptr;
        const int l = lane & 15;
        const lds_t at = base + (32 * s + 4 * (lane >> 4) + (l >> 2)) * PITCH + 64 * (t / 2) + 16 * (l & 3) + 8 * (t % 2);
        const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + 16 * PITCH));
        return join(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b));
    }
};

// A lower triangle of 64 by 64, by blocks of 16, as two planes of bf16, columns in the order of Rows: P, or (FIRST = 1) A without the blocks of its diagonal, whose first row block is 1.
template <int FIRST> struct Lower {
    static constexpr int SHORT = 80, LONG = 144, PLANE = (16 * (2 * SHORT + (2 - FIRST) * LONG) + 511) / 512 * 512, BYTES = 2 * PLANE;
    static DEVINL lds_t at(const lds_t base, const int i, const int r) { return base + (i - FIRST < 2 ? (16 * (i - FIRST) + r) * SHORT : 32 * SHORT + (16 * (i - FIRST - 2) + r) * LONG); }
    // rows 16 i + r; columns 16 j + 4 g ..
    static DEVINL void put(const lds_t base, const int i, const int r, const int j, const int g, const Two& x) {
        const lds_t to = at(base, i, r) + 64 * (j / 2) + 16 * g + 8 * (j % 2);
        lds_st(to, x.h);
        lds_st(to + PLANE, x.l);
    }
    // the lane's row of row block i: block 2 s of its columns, or blocks 2 s and 2 s + 1
    static DEVINL Two one(const lds_t base, const int lane, const int i, const int s) {
        const lds_t from = at(base, i, lane & 15) + 64 * s + 16 * (lane >> 4);
        return {lds_ld<u32x2>(from), lds_ld<u32x2>(from + PLANE)};
    }
    static DEVINL Two32 two(const lds_t base, const int lane, const int i, const int s) {
        const lds_t from = at(base, i, lane & 15) + 64 * s + 16 * (lane >> 4);
        return {lds_ld<u32x4>(from), lds_ld<u32x4>(from + PLANE)};
    }
};
// Their transposes: rows 16 j + r, columns from block j (P) or j + 1 (A) on.
template <int FIRST> struct Upper {
    static constexpr int SHORT = 80, LONG = 144, PLANE = (16 * (2 * LONG + (2 - FIRST) * SHORT) + 511) / 512 * 512, BYTES = 2 * PLANE;
    static DEVINL lds_t at(const lds_t base, const int j, const int r) { return base + (j < 2 ? (16 * j + r) * LONG : 32 * LONG + (16 * (j - 2) + r) * SHORT - 64); }
    static DEVINL void put(const lds_t base, const int j, const int r, const int i, const int g, const Two& x) {
        const lds_t to = at(base, j, r) + 64 * (i / 2) + 16 * g + 8 * (i % 2);
        lds_st(to, x.h);
        lds_st(to + PLANE, x.l);
    }
    // the lane's row of row block j: column block i, or blocks 2 s and 2 s + 1
    static DEVINL Two one(const lds_t base, const int lane, const int j, const int i) {
        const lds_t from = at(base, j, lane & 15) + 64 * (i / 2) + 16 * (lane >> 4) + 8 * (i % 2);
        return {lds_ld<u32x2>(from), lds_ld<u32x2>(from + PLANE)};
    }
    static DEVINL Two32 two(const lds_t base, const int lane, const int j, const int s) {
        const lds_t from = at(base, j, lane & 15) + 64 * s + 16 * (lane >> 4);
        return {lds_ld<u32x4>(from), lds_ld<u32x4>(from + PLANE)};
    }
};
// The inverses of the diagonal blocks of I + A, two planes each, rows of 32 bytes.
struct Diagonal {
    static constexpr int PLANE = 512, BLOCK = 2 * PLANE, BYTES = 4 * BLOCK;
    static DEVINL Two row(const lds_t base, const int lane, const int i) {
        const lds_t from = base + i * BLOCK + (lane & 15) * 32 + 8 * (lane >> 4);
        return {lds_ld<u32x2>(from), lds_ld<u32x2>(from + PLANE)};
    }
};

// lane - n's value within rows of 16 lanes (row_shr), or the last lane's of the row or the rows before (row_bcast); 0 where there is none
template <int HOW, int ROWS> DEVINL double from_lane(const double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), HOW, ROWS, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), HOW, ROWS, 0xf, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
DEVINL double at_lane(const double x, const int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Scalars of a chunk (lane = token), by one wave.
template <bool HEAD = false> DEVINL void make_scalars(const lds_t to, const int lane, const DeltaToken token, const float gate, const float beta) {
    double sum = token.cut || (token.real && gate < DELTA_NONE) ? CUT : (token.real ? static_cast<double>(gate) * 1.4426950408889634 : 0.0);
    sum += from_lane<0x111, 0xf>(sum);                          // row_shr 1, 2, 4, 8
    sum += from_lane<0x112, 0xf>(sum);
    sum += from_lane<0x114, 0xf>(sum);
    sum += from_lane<0x118, 0xf>(sum);
    sum += from_lane<0x142, 0xa>(sum);                          // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    sum += from_lane<0x143, 0xc>(sum);
    const double a = at_lane(sum, 15), b = at_lane(sum, 31), c = at_lane(sum, 47), d = at_lane(sum, 63), end = lane < 16 ? a : (lane < 32 ? b : (lane < 48 ? c : d));
    const float h = static_cast<float>(sum);
    lds_st(to + Scalars::SUM + 4 * lane, h);
    lds_st(to + Scalars::REST + 4 * lane, static_cast<float>(sum - h));
    lds_st(to + Scalars::BETA + 4 * lane, token.real ? beta : 0.f);
    lds_st(to + Scalars::ENTER + 4 * lane, __builtin_amdgcn_exp2f(h));
    lds_st(to + Scalars::LEAVE + 4 * lane, __builtin_amdgcn_exp2f(static_cast<float>(d - sum)));
    const double begin = lane < 16 ? 0.0 : (lane < 32 ? a : (lane < 48 ? b : c));
    lds_st(to + Scalars::TAIL + 4 * lane, __builtin_amdgcn_exp2f(static_cast<float>(HEAD ? sum - begin : end - sum)));
}

// What HELPERS waves make of a chunk whose rows and scalars are there: -A, P and the inverses of the diagonal blocks.  Four have a block of 16 tokens on the diagonal each, four (the same, where there are no
// more) the six blocks below, of A and P together: there D_ij = e^(G_i - G_end) e^(G_end - G_j) with `end` the last token of j's block, neither above 1 where no log decay is.
// BACK: their transposes, and D_ij = e^(G_i - G_begin) e^(G_begin - G_j) with `begin` the token before i's block.
template <class E, int D, int HELPERS, bool BACK> DEVINL void make_matrices(const lds_t K, const lds_t Q, const lds_t sc, const lds_t A, const lds_t P, const lds_t inv, const int wave, const int lane,
                                                                 const float scale) {
    const int col = lane & 15, grp = lane >> 4;
    if (HELPERS == 4 || wave >= 4) {
#pragma unroll 1
        for (int n = wave & 3; n < 6; n += 4) {
            const int i = n >= 3 ? 3 : (n >= 1 ? 2 : 1), j = n - i * (i - 1) / 2, token = 16 * (BACK ? j : i) + col;
            f32x4 x = zero4(), y = zero4();
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const u32x4 k = Rows<D>::row(K, lane, j, s), ki = Rows<D>::row(K, lane, i, s), qi = Rows<D>::row(Q, lane, i, s);
                x = BACK ? mma32<E>(ki, k, x) : mma32<E>(k, ki, x);
                y = BACK ? mma32<E>(qi, k, y) : mma32<E>(k, qi, y);
            }
            const lds_t at = sc + 4 * token, ref = sc + 4 * (BACK ? 16 * i - 1 : 16 * j + 15);
            const float up = (lds_ld<float>(at + Scalars::SUM) - lds_ld<float>(ref + Scalars::SUM)) + (lds_ld<float>(at + Scalars::REST) - lds_ld<float>(ref + Scalars::REST));
            const float d = __builtin_amdgcn_exp2f(BACK ? -up : up);
            const f32x4 tail = lds_ld<f32x4>(sc + Scalars::TAIL + 64 * (BACK ? i : j) + 16 * grp);
            if constexpr (BACK) {
                const f32x4 beta = lds_ld<f32x4>(sc + Scalars::BETA + 64 * i + 16 * grp);
                Upper<1>::put(A, j, col, i, grp, split<bf16_t>(x * -d * tail * beta));
                Upper<0>::put(P, j, col, i, grp, split<bf16_t>(y * (scale * d) * tail));
            } else {
                const float beta = lds_ld<float>(at + Scalars::BETA);
                Lower<1>::put(A, i, col, j, grp, split<bf16_t>(x * (-beta * d) * tail));
                Lower<0>::put(P, i, col, j, grp, split<bf16_t>(y * (scale * d) * tail));
            }
        }
    }
    if (HELPERS == 4 || wave < 4) {
        // A: rows 4 grp .. of the block, column lane & 15 (k_i.k_j is symmetric); P: row lane & 15, columns 4 grp ..; BACK: rows and columns the other way round
        f32x4 x = zero4(), y = zero4();
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const u32x4 k = Rows<D>::row(K, lane, wave, s), q = Rows<D>::row(Q, lane, wave, s);
            x = mma32<E>(k, k, x);
            y = BACK ? mma32<E>(q, k, y) : mma32<E>(k, q, y);
        }
        const int token = 16 * wave + col;
        const float h = lds_ld<float>(sc + Scalars::SUM + 4 * token), l = lds_ld<float>(sc + Scalars::REST + 4 * token);
        const lds_t four = sc + 64 * wave + 16 * grp;
        const f32x4 hj = lds_ld<f32x4>(four + Scalars::SUM) - h, lj = lds_ld<f32x4>(four + Scalars::REST) - l;
        const f32x4 rows = lds_ld<f32x4>(four + Scalars::BETA);
        const float row = lds_ld<float>(sc + Scalars::BETA + 4 * token);
        float m[16], z[16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float down = __builtin_amdgcn_exp2f(hj[r] + lj[r]), up = __builtin_amdgcn_exp2f(-hj[r] - lj[r]);      // (one of them is used where it does not exceed 1)
            const float a = BACK ? (col > 4 * grp + r ? -row * up * x[r] : 0.f) : (col < 4 * grp + r ? -rows[r] * down * x[r] : 0.f);
            y[r] = BACK ? (col <= 4 * grp + r ? scale * down * y[r] : 0.f) : (col >= 4 * grp + r ? scale * up * y[r] : 0.f);
            // every group's rows to all groups
            const uint32_t u = __float_as_uint(a);
            const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
            const auto even = __builtin_amdgcn_permlane32_swap(s[0], s[0], false, false), odd = __builtin_amdgcn_permlane32_swap(s[1], s[1], false, false);
            z[r] = __uint_as_float(even[0]), z[8 + r] = __uint_as_float(even[1]), z[4 + r] = __uint_as_float(odd[0]), z[12 + r] = __uint_as_float(odd[1]);
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) m[t] = t == col ? 1.f : 0.f;
        solve_bc<!BACK>(m, z);                                  // row lane & 15 of the inverse: m_s = -sum over t > s of m_t A_ts; BACK: the column, m_s = -sum over t < s of A_st m_t
        if constexpr (BACK) Upper<0>::put(P, wave, col, wave, grp, split<bf16_t>(y));
        else Lower<0>::put(P, wave, col, wave, grp, split<bf16_t>(y));
        f32x4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = grp == 0 ? m[r] : (grp == 1 ? m[4 + r] : (grp == 2 ? m[8 + r] : m[12 + r]));
        const Two w = split<bf16_t>(o);
        lds_st(inv + wave * Diagonal::BLOCK + col * 32 + 8 * grp, w.h);
        lds_st(inv + wave * Diagonal::BLOCK + Diagonal::PLANE + col * 32 + 8 * grp, w.l);
    }
}

}  // namespace
}  // namespace rwkv
