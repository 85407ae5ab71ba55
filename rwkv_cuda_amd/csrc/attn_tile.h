// Tiles of attention on the matrix cores (v_mfma_f32_32x32x16, bf16 and fp16): what the forward and the backward kernels share.
//
// Every product is written so that one index of its result, the lane's, is the one whose running sums stay put: an accumulator holds
// [row][column] with column = lane & 31 and row = 8 (r >> 2) + 4 (lane >> 5) + (r & 3) in register r.  Scores are made as K Q^T, a lane
// holding one query's scores, so that maxima and sums of a row are a lane's own (and its partner's, lane ^ 32).  Rounded and packed
// in pairs, eight of these registers are, as they stand, the second operand of the next product, whose contraction runs over
// the keys in that order; its first operand, V^T, is read from LDS in the same order (ds_read_b64_tr_b16: four rows and a
// column a lane).
#pragma once

#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t lds_t;                                         // a byte address in the workgroup's LDS
typedef __amdgpu_buffer_rsrc_t buf_t;

constexpr int TILE = 64;                                        // keys (queries) of a tile in LDS
constexpr float LOG2E = 1.4426950408889634f;

__host__ __device__ __forceinline__ int64_t wide(int x) { return x; }
template <class T> DEVINL T lds_ld(const lds_t a) { return *(const __attribute__((address_space(3))) T*)(a); }
template <class T> DEVINL void lds_st(const lds_t a, const T v) { *(__attribute__((address_space(3))) T*)(a) = v; }
DEVINL lds_t lds_of(const void* p) { return static_cast<lds_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p)); }

template <class E> DEVINL f32x16 mma(const u32x4 a, const u32x4 b, const f32x16 c) {
    if constexpr (std::is_same_v<E, bf16_t>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
// two values of the type, rounded to nearest even
template <class E> DEVINL uint32_t pack2(const float lo, const float hi) {
    if constexpr (std::is_same_v<E, bf16_t>) return pack_bf2(lo, hi);
    else {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        const f16x2_t h = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
        return __builtin_bit_cast(uint32_t, h);
    }
}
template <class E> DEVINL float unpack_lo(const uint32_t x) {
    if constexpr (std::is_same_v<E, bf16_t>) return bf_lo(x);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x)));
}
template <class E> DEVINL float unpack_hi(const uint32_t x) {
    if constexpr (std::is_same_v<E, bf16_t>) return bf_hi(x);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x >> 16)));
}
// registers 8 s .. 8 s + 7 of an accumulator as the operand of a contraction over its rows 16 s .. 16 s + 15
template <class E> DEVINL u32x4 as_operand(const f32x16& x, const int s) {
    return u32x4{pack2<E>(x[8 * s], x[8 * s + 1]), pack2<E>(x[8 * s + 2], x[8 * s + 3]), pack2<E>(x[8 * s + 4], x[8 * s + 5]), pack2<E>(x[8 * s + 6], x[8 * s + 7])};
}
DEVINL float other_half(const float x) {                        // lane ^ 32's
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}

// A matrix in LDS: `rows` rows of D values in 16-byte pieces, piece c of row r at place c ^ swap(r).  16 lanes that read one piece of 16
// rows, and 16 lanes that read four pieces of four rows, both touch every bank once.
template <int D> struct Plane {
    static constexpr int ROW = 2 * D, PIECES = D / 8, BYTES = TILE * ROW;
    static DEVINL int swap(const int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }
    static DEVINL lds_t at(const int r, const int c) { return r * ROW + ((c ^ swap(r)) << 4); }
};
// rows of a Plane as the first operand with the channels along the contraction: lane = row, `a` the addresses for row lane & 31
template <int D> struct RowReader {
    lds_t a[D / 16];
    DEVINL RowReader(const int lane) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) a[s] = Plane<D>::at(lane & 31, 2 * s + (lane >> 5));
    }
    DEVINL u32x4 operator()(const lds_t base, const int rows32, const int s) const { return lds_ld<u32x4>(a[s] + base + rows32 * 32 * Plane<D>::ROW); }
};
// ... with the rows along the contraction, in accumulator order: lane = channel of a block of 32
template <int D> struct ColReader {
    lds_t a[D / 32][2];
    DEVINL ColReader(const int lane) {
        const int l = lane & 15, r = 4 * (lane >> 5) + (l >> 2);
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) a[d][e] = Plane<D>::at(r + 8 * e, 4 * d + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) + 8 * (l & 1);
    }
    DEVINL u32x4 operator()(const lds_t base, const int rows16, const int d) const {
        typedef v4s __attribute__((address_space(3))) * ptr;
        const lds_t o = base + rows16 * 16 * Plane<D>::ROW;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(a[d][0] + o)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(a[d][1] + o));
        const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
        return u32x4{x[0], x[1], y[0], y[1]};
    }
};

// The way of a tile of 64 rows from memory to LDS: a piece of 16 bytes a thread and step, zeros behind the last row and the last channel
// (the buffer's bounds), and for rows that are to count as zeros.
template <int D, int THREADS> struct Stage {
    static constexpr int STEPS = TILE * D / 8 / THREADS, STEP_ROWS = THREADS / (D / 8);
    u32x4 x[STEPS];
    int row, off;                                               // the thread's first row, and its bytes within a row (beyond all bounds: no such channel)
    lds_t to;
    DEVINL Stage(const int tid, const int N) {
        row = tid / (D / 8);
        const int c = tid % (D / 8);
        off = 8 * c < N ? 16 * c : 0x7ffffff0;
        to = Plane<D>::at(row, c);
    }
    // rows from `first` on, `rows` of them there, `step` bytes apart
    DEVINL void load(const void* first, const int rows, const int step, const int N) {
        const buf_t b = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(first), 0, rows > 0 ? (rows - 1) * step + 2 * N : 0, 0x00027000);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int r = row + i * STEP_ROWS;
            x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, off == 0x7ffffff0 || r >= rows ? 0x7ffffff0 : r * step + off, 0, 0));
        }
    }
    DEVINL void store(const lds_t base) const {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) lds_st(base + to + i * STEP_ROWS * Plane<D>::ROW, x[i]);
    }
    // only the rows whose bit is set: those of padding may hold anything and count as zeros
    DEVINL void store(const lds_t base, const uint64_t rows) const {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const bool on = rows >> (row + i * STEP_ROWS) & 1;
            u32x4 z = x[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = on ? z[e] : 0u;
            lds_st(base + to + i * STEP_ROWS * Plane<D>::ROW, z);
        }
    }
};

// An accumulator [channel][row of the output] times `f`, rounded, to 32 channels of the lane's row (and what the rounding lost to `rest`).
// Lanes l and l + 32 exchange halves so that each has eight consecutive channels to store.
template <class E> DEVINL void store32(const f32x16& o, const float f, E* y, E* rest, const int d0, const int N, const bool on) {
    const int hi = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        uint32_t w[2][2], z[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = o[4 * (g + e) + 2 * i] * f, b = o[4 * (g + e) + 2 * i + 1] * f;
                w[e][i] = pack2<E>(a, b);
                if (rest) z[e][i] = pack2<E>(a - unpack_lo<E>(w[e][i]), b - unpack_hi<E>(w[e][i]));
            }
        const int d = d0 + 8 * (g + hi);
        const auto s0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false), s1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        if (on && d < N) *reinterpret_cast<u32x4*>(y + d) = u32x4{s0[0], s1[0], s0[1], s1[1]};
        if (rest) {
            const auto t0 = __builtin_amdgcn_permlane32_swap(z[0][0], z[1][0], false, false), t1 = __builtin_amdgcn_permlane32_swap(z[0][1], z[1][1], false, false);
            if (on && d < N) *reinterpret_cast<u32x4*>(rest + d) = u32x4{t0[0], t1[0], t0[1], t1[1]};
        }
    }
}
// 32 rows of a tensor as the second operand of products over the channels: lane = row
template <class E, int D> DEVINL void load_rows(u32x4 (&x)[D / 16], const E* row, const bool on, const int N) {
    const int hi = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const int d = 16 * s + 8 * hi;
        x[s] = on && d < N ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
    }
}

// Scores.  In units of ln 2: t = x scale log2(e), or capped and biased; without cap and bias x itself, `unit` being scale log2(e).
struct Scorer {
    float unit, in, out, slope;                                 // tanh's argument is x in / 2 (in: times log2(e)); the cap and the slope in units of ln 2
    DEVINL Scorer(const rwkv_attn_args& p, const int h) {
        unit = p.scale * LOG2E;
        in = p.cap > 0.f ? 2.f * unit / p.cap : 0.f;
        out = p.cap * LOG2E;
        slope = p.slopes ? p.slopes[h] * LOG2E : 0.f;
    }
    // r: 1 / (1 + e^(2 z)), z the tanh's argument: tanh z = 1 - 2 r, its slope 4 r (1 - r)
    template <bool CAP> DEVINL float squash(const float x) const { return CAP ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * in)) : 0.f; }
    template <bool CAP, bool BIAS> DEVINL float t(const float x, const float r, const float dist) const {
        if constexpr (!CAP && !BIAS) return x;
        float t = CAP ? fmaf(r, -2.f * out, out) : x * unit;
        if constexpr (BIAS) t = fmaf(fabsf(dist), -slope, t);
        return t;
    }
};

// Which tiles of 64 positions a block whose rows have documents lo .. hi has to look at: 0 none of its tokens, 1 some, 2 all of them and of its rows
// one document.  Written for a window of tiles to LDS.
constexpr int WINDOW = 1024;
DEVINL void classify(uint8_t* kind, const int* doc, const int first_tile, const int tiles, const int T, const int lo, const int hi, const bool uniform, const int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int AHEAD = 8;
    for (int i0 = wave * AHEAD; i0 < tiles; i0 += waves * AHEAD) {
        int d[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int64_t j = wide(first_tile + i0 + e) * TILE + lane;
            d[e] = i0 + e < tiles && j < T ? doc[j] : -1;
        }
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const bool any = __ballot(d[e] >= 0 && d[e] >= lo && d[e] <= hi) != 0ull, all = __ballot(d[e] == lo) == ~0ull;
            if (lane == 0 && i0 + e < tiles) kind[i0 + e] = !any ? 0 : (all && uniform ? 2 : 1);
        }
    }
}

// the first tile from `t` on (below `end`) that is looked at; `kind` begins with tile w0
DEVINL int next_tile(const uint8_t* kind, int t, const int w0, const int end) {
    const int lane = threadIdx.x & 63;
    for (; t < end; t += 64) {
        const uint64_t some = __ballot(t + lane < end && kind[t + lane - w0] != 0);
        if (some) return __builtin_amdgcn_readfirstlane(t + __builtin_ctzll(some));
    }
    return end;
}

}  // namespace
}  // namespace rwkv
