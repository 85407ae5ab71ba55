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

#include <climits>

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

// What the forward keeps for the backward, and the backward for its last kernel, of each head and chunk, as the waves hold them: tiles of 16 by 16, four neighbouring rows of a column a lane, 16
// bytes.  The state that enters (whose gradient leaves), fp32, [column tile][row tile], stored at a chunk's start, where its wave waits; and the updates (their gradients), [column tile][token tile],
// as the two numbers that they were operands as, four first ones, then four second ones.  (fp16 alone, 11 bits, would halve the traffic, but states and updates cancel within a chunk wherever new
// values replace old ones, and where these are the larger its error would be seen.)
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
DEVINL float sum4(const f32x4 x) { return (x[0] + x[1]) + (x[2] + x[3]); }
DEVINL float group_sum4(const float x) {                        // over the four lanes with the same lane & 15
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
DEVINL bool finite(const float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

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
DEVINL void keep(float* to, const Two& x) { *reinterpret_cast<u32x4*>(to) = join(x.h, x.l); }
// one token's part of what keep() leaves of a chunk's four tiles
DEVINL void keep_token(float* updates, const int token, const int col, const float x) {
    uint16_t* const to = reinterpret_cast<uint16_t*>(updates + 256 * (token >> 4) + 4 * (16 * (token >> 2 & 3) + col)) + (token & 3);
    const bf16_t h = from_f<bf16_t>(x);
    to[0] = __builtin_bit_cast(uint16_t, h), to[4] = __builtin_bit_cast(uint16_t, from_f<bf16_t>(x - to_f(h)));
}
// Tiles as operands beside an input of type E: bf16 as they are, fp16 times a power of two, whose inverse is what the product is to be multiplied with.  (A value 2^-k of the wave's
// largest keeps 35 - k bits, 22 at most.  NaN do not count as large; infinities would, so that what comes from outside is made no_infinity: a column with one is NaN after its first product in any case.)
template <class E, class V> DEVINL V no_infinity(const V x) {
    if constexpr (std::is_same_v<E, bf16_t>) return x;
    else return __builtin_elementwise_fma(x, V(0.f), x);
}
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

// LDS is read 256 bytes a cycle: of 16 bytes a lane by lanes 0-3, 12-15 and 20-27, then 4-11, 16-19 and 28-31, and likewise from 32 on; of 8 by half a wave; it is written 128 bytes a cycle, by 8 or
// 16 neighbours.  (Found with the counters of conflicts.)  A row of 64 bytes or more is cut into blocks of 64, these into pieces of 16, and rows exchange both among themselves, so that 16 rows'
// pieces, one a row, fall on all banks once in each of those groups; where columns are read, 8 bytes of a piece, two rows meet.
DEVINL int piece_swap(const int row) { return -(row >> 2) & 3; }
template <int BYTES> DEVINL int block_swap(const int row) { return BYTES == 256 ? row & 3 : (BYTES == 128 ? row >> 1 & 1 : 0); }
template <int BYTES> DEVINL lds_t place(const int row, const int block, const int piece) { return row * BYTES + 64 * (block ^ block_swap<BYTES>(row)) + 16 * (piece ^ piece_swap(row)); }

// Which of eight rows the lanes' n-th is where rows are written, and which 16 bytes of it a lane has: 16 neighbours have 128 bytes (64) of two rows (four), which then meet nowhere.
template <int D> DEVINL int written_row(const int n) { return D == 32 ? (n & ~7) | (n & 1) | (n << 1 & 4) | (n >> 1 & 2) : (n & ~7) | (n << 2 & 4) | (n >> 1 & 3); }
template <int D> DEVINL int written_order(const int lane) { return D == 128 ? (lane >> 4 & ~1) | (lane >> 3 & 1) : lane / (D / 8); }
template <int D> DEVINL int written_piece(const int lane) { return D == 128 ? (lane & 7) | (lane >> 1 & 8) : lane % (D / 8); }
// 64 rows of D inputs in LDS.  Of every 32 channels number 16 e + 4 g + r is at place 8 g + 4 e + r: 16 bytes
// are what a lane of group g needs.
template <int D> struct Rows {
    static constexpr int PITCH = 2 * D, BYTES = 64 * PITCH;
    // channels 8 c .. 8 c + 7 of a row
    static DEVINL void put(const lds_t base, const int row, const int c, const u32x4 x) {
        const lds_t to = place<PITCH>(row, c / 4, 2 * (c % 2)) + 8 * (c / 2 % 2);
        lds_st(base + to, u32x2{x[0], x[1]});
        lds_st(base + (to ^ 16), u32x2{x[2], x[3]});
    }
    // four of a row's channels, 16 t + 4 g ..
    static DEVINL u32x2 four(const lds_t base, const int row, const int t, const int g) { return lds_ld<u32x2>(base + place<PITCH>(row, t / 2, g) + 8 * (t % 2)); }
    // row 16 i + (lane & 15), channels of the 32 s-th: the contraction runs over channels
    static DEVINL u32x4 row(const lds_t base, const int lane, const int i, const int s) { return lds_ld<u32x4>(base + 16 * i * PITCH + place<PITCH>(lane & 15, s, lane >> 4)); }
    // channel 16 t + (lane & 15), rows of the 32 s-th: the contraction runs over rows
    static DEVINL u32x4 col(const lds_t base, const int lane, const int t, const int s) {
        typedef v4s __attribute__((address_space(3))) * ptr;
        const int l = lane & 15;
        const lds_t at = base + 32 * s * PITCH + place<PITCH>(4 * (lane >> 4) + (l >> 2), t / 2, l & 3) + 8 * (t % 2);
        const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + 16 * PITCH));
        return join(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b));
    }
};

// A lower triangle of 64 by 64, by blocks of 16, as two planes of bf16, columns in the order of Rows: P, or (FIRST = 1) A without the blocks of its diagonal, whose first row block is 1.
template <int FIRST> struct Lower {
    static constexpr int SHORT = 64, LONG = 128, PLANE = 16 * (2 * SHORT + (2 - FIRST) * LONG), BYTES = 2 * PLANE;
    // a piece of row 16 i + r: columns 16 (2 s) + 4 g .. and 16 (2 s + 1) + 4 g ..
    static DEVINL lds_t at(const lds_t base, const int i, const int r, const int s, const int g) {
        return base + (i - FIRST < 2 ? 16 * (i - FIRST) * SHORT + place<SHORT>(r, s, g) : 32 * SHORT + 16 * (i - FIRST - 2) * LONG + place<LONG>(r, s, g));
    }
    // rows 16 i + r; columns 16 j + 4 g ..
    static DEVINL void put(const lds_t base, const int i, const int r, const int j, const int g, const Two& x) {
        const lds_t to = at(base, i, r, j / 2, g) + 8 * (j % 2);
        lds_st(to, x.h);
        lds_st(to + PLANE, x.l);
    }
    // the lane's row of row block i: block 2 s of its columns, or blocks 2 s and 2 s + 1
    static DEVINL Two one(const lds_t base, const int lane, const int i, const int s) {
        const Two32 x = two(base, lane, i, s);                  // (half a piece would take as long)
        return {u32x2{x.h[0], x.h[1]}, u32x2{x.l[0], x.l[1]}};
    }
    static DEVINL Two32 two(const lds_t base, const int lane, const int i, const int s) {
        const lds_t from = at(base, i, lane & 15, s, lane >> 4);
        return {lds_ld<u32x4>(from), lds_ld<u32x4>(from + PLANE)};
    }
};
// Their transposes: rows 16 j + r, columns from block j (P) or j + 1 (A) on.
template <int FIRST> struct Upper {
    static constexpr int SHORT = 64, LONG = 128, PLANE = 16 * (2 * LONG + (2 - FIRST) * SHORT), BYTES = 2 * PLANE;
    static DEVINL lds_t at(const lds_t base, const int j, const int r, const int s, const int g) {
        return base + (j < 2 ? 16 * j * LONG + place<LONG>(r, s, g) : 32 * LONG + 16 * (j - 2) * SHORT + place<SHORT>(r, s - 1, g));
    }
    static DEVINL void put(const lds_t base, const int j, const int r, const int i, const int g, const Two& x) {
        const lds_t to = at(base, j, r, i / 2, g) + 8 * (i % 2);
        lds_st(to, x.h);
        lds_st(to + PLANE, x.l);
    }
    // the lane's row of row block j: column block i, or blocks 2 s and 2 s + 1
    static DEVINL Two one(const lds_t base, const int lane, const int j, const int i) {
        const Two32 x = two(base, lane, j, i / 2);
        return i % 2 ? Two{u32x2{x.h[2], x.h[3]}, u32x2{x.l[2], x.l[3]}} : Two{u32x2{x.h[0], x.h[1]}, u32x2{x.l[0], x.l[1]}};
    }
    static DEVINL Two32 two(const lds_t base, const int lane, const int j, const int s) {
        const lds_t from = at(base, j, lane & 15, s, lane >> 4);
        return {lds_ld<u32x4>(from), lds_ld<u32x4>(from + PLANE)};
    }
};
// The inverses of the diagonal blocks of I + A, two planes each, rows of 32 bytes, whose halves the second eight rows exchange.
struct Diagonal {
    static constexpr int PLANE = 512, BLOCK = 2 * PLANE, BYTES = 4 * BLOCK;
    static DEVINL Two row(const lds_t base, const int lane, const int i) {
        const lds_t from = base + i * BLOCK + (lane & 15) * 32 + (8 * (lane >> 4) ^ 2 * (lane & 8));
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

// Which of a chunk's matrices a helping wave makes, a rule on how many there are (8 waves a workgroup, of which 4, 2 or 1 walk: those come first, and the helpers with the least to do share their
// SIMDs).  Bits 0 .. 5: the blocks below the diagonal, of A and P together, (1,0), (2,0), (2,1), (3,0), (3,1), (3,2); 6 .. 9: P's blocks on the diagonal; 10, 11: the inverses of blocks 0 and 1, of
// 2 and 3; 12: the scalars.
template <int HELPERS> DEVINL uint32_t tasks_of(const int wave) {
    constexpr uint32_t INV0 = 1 << 10, INV1 = 1 << 11, SCALARS = 1 << 12;
    if constexpr (HELPERS == 4) return wave == 0 ? INV0 | 0xc0 : (wave == 1 ? INV1 | 0x300 : (wave == 2 ? 0x07 | SCALARS : 0x38));
    else if constexpr (HELPERS == 6) return wave == 0 ? INV0 : (wave == 1 ? INV1 : (wave == 2 ? 0x03 : (wave == 3 ? 0x04 | SCALARS : (wave == 4 ? 0x08 | 0xc0 : 0x30 | 0x300))));
    else return wave == 0 ? INV0 : (wave == 1 ? INV1 : (wave == 2 ? 0x03 : (wave == 3 ? SCALARS : (wave == 4 ? 0x0c : (wave == 5 ? 0x10 | 0xc0 : 0x20 | 0x300)))));
}

// Those of a chunk whose rows and scalars are there.  Blocks below the diagonal: D_ij = e^(G_i - G_end) e^(G_end - G_j) with `end` the last token of j's block, neither above 1 where no log decay is.  Forward:
// A without beta, and the inverses times beta (of their columns), so that the right side is V - e^G K S alone.  BACK: the transposes, and `end` is the token before i's block.
template <class E, int D, bool BACK> DEVINL void make_matrices(const lds_t K, const lds_t Q, const lds_t sc, const lds_t A, const lds_t P, const lds_t inv, const uint32_t tasks, const int lane, const float scale) {
    const int col = lane & 15, grp = lane >> 4;
    const auto at = [&](const lds_t what, const int n) { return sc + what + 4 * n; };
#pragma unroll 1
    for (uint32_t left = tasks & 0x3f; left != 0; left &= left - 1) {
        const int n = __builtin_ctz(left), i = n >= 3 ? 3 : (n >= 1 ? 2 : 1), j = n - i * (i - 1) / 2, token = 16 * (BACK ? j : i) + col;
        f32x4 x = zero4(), y = zero4();
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const u32x4 k = Rows<D>::row(K, lane, j, s), ki = Rows<D>::row(K, lane, i, s), qi = Rows<D>::row(Q, lane, i, s);
            x = BACK ? mma32<E>(ki, k, x) : mma32<E>(k, ki, x);
            y = BACK ? mma32<E>(qi, k, y) : mma32<E>(k, qi, y);
        }
        const int ref = BACK ? 16 * i - 1 : 16 * j + 15;
        const float up = (lds_ld<float>(at(Scalars::SUM, token)) - lds_ld<float>(at(Scalars::SUM, ref))) + (lds_ld<float>(at(Scalars::REST, token)) - lds_ld<float>(at(Scalars::REST, ref)));
        const float d = __builtin_amdgcn_exp2f(BACK ? -up : up);
        const f32x4 tail = lds_ld<f32x4>(at(Scalars::TAIL, 16 * (BACK ? i : j) + 4 * grp)) * d;
        if constexpr (BACK) {
            Upper<1>::put(A, j, col, i, grp, split<bf16_t>(x * -tail * lds_ld<f32x4>(at(Scalars::BETA, 16 * i + 4 * grp))));
            Upper<0>::put(P, j, col, i, grp, split<bf16_t>(y * scale * tail));
        } else {
            Lower<1>::put(A, i, col, j, grp, split<bf16_t>(x * -tail));
            Lower<0>::put(P, i, col, j, grp, split<bf16_t>(y * scale * tail));
        }
    }
#pragma unroll 1
    for (uint32_t left = tasks >> 6 & 0xf; left != 0; left &= left - 1) {
        const int w = __builtin_ctz(left);
        f32x4 y = zero4();                                      // row lane & 15, columns 4 grp ..; BACK: the transpose's
        u32x4 k[D / 32], q[D / 32];
#pragma unroll
        for (int s = 0; s < D / 32; ++s) k[s] = Rows<D>::row(K, lane, w, s), q[s] = Rows<D>::row(Q, lane, w, s);
        in_order();                                             // (or the compiler may wait for each)
#pragma unroll
        for (int s = 0; s < D / 32; ++s) y = BACK ? mma32<E>(q[s], k[s], y) : mma32<E>(k[s], q[s], y);
        const float h = lds_ld<float>(at(Scalars::SUM, 16 * w + col)), l = lds_ld<float>(at(Scalars::REST, 16 * w + col));
        const f32x4 hj = lds_ld<f32x4>(at(Scalars::SUM, 16 * w + 4 * grp)) - h, lj = lds_ld<f32x4>(at(Scalars::REST, 16 * w + 4 * grp)) - l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float d = __builtin_amdgcn_exp2f(BACK ? hj[r] + lj[r] : -hj[r] - lj[r]);
            y[r] = (BACK ? col <= 4 * grp + r : col >= 4 * grp + r) ? scale * d * y[r] : 0.f;
        }
        if constexpr (BACK) Upper<0>::put(P, w, col, w, grp, split<bf16_t>(y));
        else Lower<0>::put(P, w, col, w, grp, split<bf16_t>(y));
    }
    if (tasks >> 10 & 3) {                                       // blocks w and w + 1: at last one in the lanes' first half, one in the second
        const int w = tasks >> 10 & 1 ? 0 : 2;
        f32x4 a[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            f32x4 x = zero4();                                  // rows 4 grp .., column lane & 15 (k_i.k_j is symmetric); BACK: the other way round
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const u32x4 k = Rows<D>::row(K, lane, w + e, s);
                x = mma32<E>(k, k, x);
            }
            const int token = 16 * (w + e) + col, four = 16 * (w + e) + 4 * grp;
            const float h = lds_ld<float>(at(Scalars::SUM, token)), l = lds_ld<float>(at(Scalars::REST, token));
            const f32x4 hj = lds_ld<f32x4>(at(Scalars::SUM, four)) - h, lj = lds_ld<f32x4>(at(Scalars::REST, four)) - l, rows = lds_ld<f32x4>(at(Scalars::BETA, four));
            const float row = lds_ld<float>(at(Scalars::BETA, token));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float d = __builtin_amdgcn_exp2f(BACK ? -hj[r] - lj[r] : hj[r] + lj[r]);
                a[e][r] = (BACK ? col > 4 * grp + r : col < 4 * grp + r) ? -(BACK ? row : rows[r]) * d * x[r] : 0.f;
            }
        }
        float m[16], z[16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {                            // every group's rows to both groups of their block's half
            const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a[0][r]), __float_as_uint(a[1][r]), false, false);
            const auto low = __builtin_amdgcn_permlane16_swap(s[0], s[0], false, false), high = __builtin_amdgcn_permlane16_swap(s[1], s[1], false, false);
            z[r] = __uint_as_float(low[0]), z[4 + r] = __uint_as_float(low[1]), z[8 + r] = __uint_as_float(high[0]), z[12 + r] = __uint_as_float(high[1]);
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) m[t] = t == col ? 1.f : 0.f;
        solve_bc<!BACK>(m, z);                                  // row lane & 15 of the inverse: m_s = -sum over t > s of m_t A_ts; BACK: the column, m_s = -sum over t < s of A_st m_t
        const int block = w + (lane >> 5), half = grp & 1;       // of a row: the first or the last eight
        const lds_t to = inv + block * Diagonal::BLOCK + col * 32 + (16 * half ^ 2 * (col & 8));
        Two o[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = half ? m[8 + 4 * e + r] : m[4 * e + r];
            if constexpr (!BACK) x *= lds_ld<f32x4>(at(Scalars::BETA, 16 * block + 8 * half + 4 * e));
            o[e] = split<bf16_t>(x);
        }
        lds_st(to, join(o[0].h, o[1].h));
        lds_st(to + Diagonal::PLANE, join(o[0].l, o[1].l));
    }
}

// A walk once more, token by token, by one walking wave for its 16 columns, where its state came to be no number in a row with documents, padding or decays of nothing: products by 0 carry that across a cut and
// into all that stands behind (BACK: before), up to the end, while here what must not count is not looked at.  False where there is no such thing in the row.  The arguments are read once more, so
// that little of this takes registers of the loops that do the work.  It takes some 2 us a token (a row of 8192 tokens, 32 heads of 128, 15 ms instead of 0.22).
typedef const rwkv_delta_args __attribute__((address_space(4))) DeltaArguments;
template <class E, int D, bool BACK> DEVINL bool walk_by_token(DeltaArguments* arguments, const int hb, const int start, const int count, const int c0, const bool first_own, float* states, float* updates) {
    asm volatile("" : "+s"(arguments));
    DeltaArguments& p = *arguments;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, N = p.N, T = p.T, chunks = (T + DELTA_CHUNK - 1) / DELTA_CHUNK, column = c0 + col;
    const int b = hb / p.H, h = hb % p.H, hk = h / (p.H / p.Hk);
    const E *g = static_cast<const E*>(p.g) + b * p.g_sb + h, *beta = static_cast<const E*>(p.beta) + b * p.beta_sb + h;
    const auto token_of = [&](const int t) { return delta_token(p.doc, wide(b) * T, t, T); };
    bool apart = false;
    for (int t = lane; t < T; t += 64) {
        const DeltaToken is = token_of(t);
        apart |= !is.real || is.cut || to_f(g[t * p.g_st]) < DELTA_NONE;
    }
    if (__ballot(apart) == 0ull) return false;
    const DeltaTiles tiles(p.B, T, p.H, N);
    const bool on = column < N;
    const E *q = static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh, *k = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh, *v = static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh;
    const int64_t dense = (wide(b) * T * p.H + h) * N + column, step = wide(p.H) * N, square = wide(hb) * N * N;
    const auto four = [&](const E* row, const int t) {          // a lane's four key channels of tile t
        const int d = 16 * t + 4 * grp;
        return d < N ? four_of<E>(*reinterpret_cast<const u32x2*>(row + d)) : zero4();
    };
    const float* const first = !first_own ? nullptr : (BACK ? p.dsT : p.s0);
    f32x4 S[D / 16];
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] = first && on && 16 * t + 4 * grp + r < N ? first[square + (16 * t + 4 * grp + r) * N + column] : 0.f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // what is stored again is stored behind what was
    for (int c = 0; c < count; ++c) {
        const int chunk = BACK ? start - c : start + c, t0 = chunk * DELTA_CHUNK, n = min(DELTA_CHUNK, T - t0);
        const int64_t kept = wide(hb) * chunks + chunk;
        const bool own = first_own || c > 0;
        if (states && own)
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
                if (t < tiles.tiles) *reinterpret_cast<f32x4*>(states + tiles.state(kept, c0 / 16, t) + 4 * lane) = S[t];
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int token = BACK ? n - 1 - i : i, t = t0 + token;
            const DeltaToken is = token_of(t);
            float u = 0.f, y = 0.f;
            if (is.real) {
                const float lg = to_f(g[t * p.g_st]), a = is.cut || lg < DELTA_NONE ? 0.f : expf(lg), bt = to_f(beta[t * p.beta_st]);
                const E *qt = q + t * p.q_st, *kt = k + t * p.k_st;
                float x = 0.f;
                if constexpr (BACK) {
                    const float dy = on && p.dy ? p.scale * to_f(static_cast<const E*>(p.dy)[dense + t * step]) : 0.f;
#pragma unroll
                    for (int r = 0; r < D / 16; ++r) {
                        S[r] += four(qt, r) * dy;
                        x += sum4(four(kt, r) * S[r]);
                    }
                    u = group_sum4(x);
#pragma unroll
                    for (int r = 0; r < D / 16; ++r) {
                        S[r] -= four(kt, r) * (bt * u);
                        S[r] = a == 0.f ? zero4() : S[r] * a;
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < D / 16; ++r) {
                        S[r] = a == 0.f ? zero4() : S[r] * a;
                        x += sum4(four(kt, r) * S[r]);
                    }
                    u = bt * ((on ? to_f(v[t * p.v_st + column]) : 0.f) - group_sum4(x));
#pragma unroll
                    for (int r = 0; r < D / 16; ++r) {
                        S[r] += four(kt, r) * u;
                        y += sum4(four(qt, r) * S[r]);
                    }
                    y = p.scale * group_sum4(y);
                }
            }
            if (!own || grp != 0) continue;
            if (!BACK && on) static_cast<E*>(p.y)[dense + t * step] = from_f<E>(y);
            if (states) keep_token(updates + tiles.update(kept, c0 / 16, 0), token, col, on ? u : 0.f);
        }
    }
    float* const last = BACK ? (start + 1 == count ? p.ds0 : nullptr) : (start + count == chunks ? p.sT : nullptr);
    if (last && on)
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * t + 4 * grp + r < N) last[square + (16 * t + 4 * grp + r) * N + column] = S[t][r];
    return true;
}

// Where things are in a walking workgroup's LDS.  (Scalars are made a chunk earlier than what uses them.)
template <int D, int SW, bool BACK> struct WalkPlace {
    static constexpr int VPITCH = 32 * SW + 16;
    static constexpr lds_t K = 0, Q = Rows<D>::BYTES, STAGE = 2 * Rows<D>::BYTES, V = 2 * STAGE, MATRICES = V + 64 * VPITCH, A = 0, P = BACK ? Upper<1>::BYTES : Lower<1>::BYTES,
                           INV = P + (BACK ? Upper<0>::BYTES : Lower<0>::BYTES), MATRIX_STAGE = INV + Diagonal::BYTES, SCALARS = MATRICES + 2 * MATRIX_STAGE, BYTES = SCALARS + 3 * Scalars::BYTES;
    static_assert(BYTES <= 160 * 1024);
};

// The helping waves of a walk over `chunks` chunks from `start` on: forward, with the values beside queries and keys; BACK, downwards, with the gradients of y.  Before the walkers' first barrier
// a chunk's rows go to LDS, between it and the second the next chunk's matrices are made.
template <class E, int D, int SW, int HELPERS, bool BACK> DEVINL void help(const rwkv_delta_args& p, const lds_t lds, const int b, const int h, const int hk, const int piece, const int mine, const int lane, const int start,
                                                                                      const int chunks) {
    using L = WalkPlace<D, SW, BACK>;
    constexpr int LANES = 64 * HELPERS, RP = D / 8, KP = (64 * RP + LANES - 1) / LANES, VP = (64 * 2 * SW + LANES - 1) / LANES, KSTEP = LANES / RP, VSTEP = LANES / (2 * SW);       // 16 bytes a lane: pieces, rows between them
    static_assert(LANES % RP == 0 && LANES % (2 * SW) == 0);
    const int N = p.N, T = p.T, tid = 64 * mine + lane;
    const uint32_t tasks = tasks_of<HELPERS>(mine);
    const int krow = written_order<D>(tid), kd = 8 * written_piece<D>(tid), vrow = tid / (2 * SW), vd = 16 * SW * piece + 8 * (tid % (2 * SW));
    const bool kin = kd < N, vin = vd < N && (!BACK || p.dy);
    const int64_t v_st = BACK ? wide(p.H) * N : p.v_st;
    const auto first = [&](const int c) { return (BACK ? start - c : start + c) * DELTA_CHUNK; };
    const char *k = reinterpret_cast<const char*>(static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh), *q = reinterpret_cast<const char*>(static_cast<const E*>(p.q) + b * p.q_sb + hk * p.q_sh);
    const char* v = reinterpret_cast<const char*>(BACK ? static_cast<const E*>(p.dy) + (wide(b) * T * p.H + h) * N : static_cast<const E*>(p.v) + b * p.v_sb + h * p.v_sh);
    if (BACK && !p.dy) v = q;                                    // (read, not used)
    const int64_t ks = 2 * p.k_st, qs = 2 * p.q_st, vs = BACK && !p.dy ? 0 : 2 * v_st;
    u32x4 kr[KP], qr[KP], vr[VP];
    // A lane's places in a chunk, bytes; rows behind the last are read as it.  Heads of 64 keep them from chunk to chunk (32768 tokens of 32 heads: 945 us instead, with them 884), with heads of 128 loads that
    // follow each other at once cost more than the instructions between them (1148 us, and 1200).
    constexpr bool KEPT = D == 64;
    const int kc0 = 2 * (kin ? kd : 0), vc0 = 2 * (vin ? vd : 0);
    int64_t ko[KP], qo[KP], vo[VP];
    int rows = -1;
    const auto load = [&](const int c) {
        const int t0 = first(c), last = min(T - 1 - t0, 63);
        const char *kc = k + t0 * ks, *qc = q + t0 * qs, *vc = v + t0 * vs;
        if constexpr (KEPT) {
            if (last != rows) {
                rows = last;
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const int row = min(written_row<D>(krow + KSTEP * i), last);
                    ko[i] = row * ks + kc0, qo[i] = row * qs + kc0;
                }
#pragma unroll
                for (int i = 0; i < VP; ++i) vo[i] = min(vrow + VSTEP * i, last) * vs + vc0;
            }
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                kr[i] = *reinterpret_cast<const u32x4*>(kc + ko[i]);
                qr[i] = *reinterpret_cast<const u32x4*>(qc + qo[i]);
            }
#pragma unroll
            for (int i = 0; i < VP; ++i) vr[i] = *reinterpret_cast<const u32x4*>(vc + vo[i]);
        } else {
            kc += kc0, qc += kc0, vc += vc0;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const int row = min(written_row<D>(krow + KSTEP * i), last);
                kr[i] = *reinterpret_cast<const u32x4*>(kc + row * ks);
                qr[i] = *reinterpret_cast<const u32x4*>(qc + row * qs);
            }
#pragma unroll
            for (int i = 0; i < VP; ++i) vr[i] = *reinterpret_cast<const u32x4*>(vc + min(vrow + VSTEP * i, last) * vs);
        }
    };
    const E *g = static_cast<const E*>(p.g) + b * p.g_sb + h, *beta = static_cast<const E*>(p.beta) + b * p.beta_sb + h;
    E gate, bt;                                                  // (as they come: what is made of them here would wait for them)
    int doc = 0, before = 0;
    const auto load_scalars = [&](const int c) {
        const int t = min(first(c) + lane, T - 1);
        if (tasks >> 12) gate = g[t * p.g_st], bt = beta[t * p.beta_st];
        if (p.doc) doc = p.doc[wide(b) * T + t], before = p.doc[wide(b) * T + max(t - 1, 0)];
    };
    uint64_t real;
    const auto scalars = [&](const int c) {
        const int t = first(c) + lane;
        const bool is = t < T && doc >= 0;
        real = __ballot(is);
        if (tasks >> 12) make_scalars<BACK>(lds + L::SCALARS + c % 3 * Scalars::BYTES, lane, {is, is && t > 0 && doc != before}, to_f(gate), to_f(bt));
    };
    const auto mask_of = [&](const int row) { return 0u - static_cast<uint32_t>(real >> (row & 63) & 1); };      // all bits of a real token's, none of others
    // (with a whole chunk of real tokens and all channels there is nothing to mask)
    const auto put_rows = [&](const int c, auto whole) {
        const lds_t to = lds + (c & 1) * L::STAGE;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int row = written_row<D>(krow + KSTEP * i);
            if (64 * RP % LANES != 0 && i == KP - 1 && row >= 64) continue;
            if constexpr (decltype(whole)::value) {
                Rows<D>::put(to + L::K, row, kd / 8, kr[i]);
                Rows<D>::put(to + L::Q, row, kd / 8, qr[i]);
            } else {
                const uint32_t keep = kin ? mask_of(row) : 0;
                Rows<D>::put(to + L::K, row, kd / 8, kr[i] & keep);
                Rows<D>::put(to + L::Q, row, kd / 8, qr[i] & keep);
            }
        }
    };
    const auto put = [&](const int c) {
        if (real == ~0ull && N == D) put_rows(c, std::true_type());
        else put_rows(c, std::false_type());
    };
    const auto put_values = [&] {
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int row = vrow + VSTEP * i;
            if (64 * 2 * SW % LANES != 0 && i == VP - 1 && row >= 64) continue;
            lds_st(lds + L::V + row * L::VPITCH + 16 * (tid % (2 * SW)), vr[i] & (vin ? mask_of(row) : 0));
        }
    };
    const auto matrices = [&](const int c) {
        const lds_t rows = lds + (c & 1) * L::STAGE, mats = lds + L::MATRICES + (c & 1) * L::MATRIX_STAGE;
        make_matrices<E, D, BACK>(rows + L::K, rows + L::Q, lds + L::SCALARS + c % 3 * Scalars::BYTES, mats + L::A, mats + L::P, mats + L::INV, tasks, lane, p.scale);
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
            put_values();                                        // (the walkers have read this chunk's)
            if (c + 2 < chunks) load(c + 2);
            matrices(c + 1);
            if (c + 2 < chunks) scalars(c + 2);
            if (c + 3 < chunks) load_scalars(c + 3);
        }
        __syncthreads();
    }
}
// Where a row of documents is walked by two workgroups.  Behind a cut nothing counts of what stood before, so that the second of them may begin with a chunk that has one, from a state of zero: what it has at
// that chunk's end is right, while the chunk itself is the first one's.  (Backward the other way round: the first part's gradient begins with that chunk, which is the second one's.)  The chunk with a cut
// that is nearest the middle; -1 without one.  By all threads.
DEVINL int split_at(const int* doc, const int T, const int chunks, int* best) {
    if (threadIdx.x == 0) *best = INT_MAX;
    __syncthreads();
    for (int t = 1 + threadIdx.x; t < T; t += blockDim.x) {
        const int d = doc[t];
        if (d < 0 || doc[t - 1] == d) continue;
        const int off = 2 * (t / DELTA_CHUNK) + 1 - chunks;
        atomicMin(best, off < 0 ? -2 * off : 2 * off + 1);
    }
    __syncthreads();
    const int key = *best;
    return key == INT_MAX ? -1 : (chunks - 1 + (key & 1 ? key >> 1 : -(key >> 1))) / 2;
}
// Columns a walking workgroup has, in tiles of 16.  A CU holds one workgroup, and one with more tiles takes longer, by the costs below, but makes its matrices for more of them: the width whose rounds
// over 256 CUs take the least.  us of the forward, 2048 tokens, bf16, with one, two and four tiles:  heads of 64: 64 of them 65 73 89;  128: 124 76 90;  256: 250 143 98;   heads of 128: 32 of them
// 81 88 115;  64: 155 94 116;  128: 309 176 131;  256: 619 350 256
// With documents two workgroups may share a row: a walk of three quarters of it is reckoned with, and taken where it costs less.  us of the forward, bf16, a row of 3001 tokens, 32 heads of 128, no documents,
// one, two halves, five: 122 135 76 86;  32 heads of 64 95 100 58 66;  8192 tokens of 8 heads of 64 246 257 135 160;  4 rows of 2048, 16 heads of 64, 69 77 46 53
// `in`, `out`: the states that a walk reads first and writes last; where they share memory a row stays with one workgroup, as two do not wait for each other.
template <class Run> int walk_width(const rwkv_delta_args& p, const float* in, const float* out, Run run) {
    using std::integral_constant;
    const int64_t heads = static_cast<int64_t>(p.B) * p.H, tiles = (p.N + 15) / 16, chunks = (p.T + DELTA_CHUNK - 1) / DELTA_CHUNK;
    const auto cost = [&](const int sw, const int segments) {
        return (heads * segments * ((tiles + sw - 1) / sw) + 255) / 256 * (sw == 1 ? 8 : (sw == 2 ? 9 : 12)) * (segments == 1 ? 4 * chunks : 3 * chunks + 4);
    };
    const uintptr_t from = reinterpret_cast<uintptr_t>(in), to = reinterpret_cast<uintptr_t>(out), size = static_cast<uintptr_t>(heads) * p.N * p.N * sizeof(float);
    const bool parts = p.doc && chunks >= 8 && !(in && out && from < to + size && to < from + size);
    int best = 1, segments = 1;
    for (const int n : {1, 2})
        for (const int sw : {1, 2, 4})                           // (four tiles and two workgroups a row never win: two tiles and one take no more rounds, of 9 times 4 chunks against 12 times 3 and more)
            if ((n == 1 || (parts && sw < 4)) && cost(sw, n) < cost(best, segments)) best = sw, segments = n;
    using std::true_type, std::false_type;
    if (segments == 2) return best == 1 ? run(integral_constant<int, 1>{}, true_type()) : run(integral_constant<int, 2>{}, true_type());
    if (best == 1) return run(integral_constant<int, 1>{}, false_type());
    return best == 2 ? run(integral_constant<int, 2>{}, false_type()) : run(integral_constant<int, 4>{}, false_type());
}

}  // namespace
}  // namespace rwkv
