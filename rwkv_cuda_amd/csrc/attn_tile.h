// Tiles of attention on the matrix cores (v_mfma_f32_32x32x16, bf16 and fp16): what the forward and the backward kernels share.
//
// Every product is written so that one index of its result, the lane's, is the one whose running sums stay put: an accumulator holds
// [row][column] with column = lane & 31 and row = 8 (r >> 2) + 4 (lane >> 5) + (r & 3) in register r.  Scores are made as K Q^T, a lane
// holding one query's scores, so that maxima and sums of a row are a lane's own (and its partner's, lane ^ 32).  Rounded and packed
// in pairs, eight of these registers are, as they stand, the second operand of the next product, whose contraction runs over
// the keys in that order; its first operand, V^T, is read from LDS in the same order (ds_read_b64_tr_b16: four rows and a
// column a lane).
#pragma once

#include <climits>

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

// A matrix of 64 rows of D values in LDS.  A kilobyte (4 rows of 128 values, 8 of 64) is what a wave brings at once; kilobytes lie 16 or 32 bytes further apart
// than their size, and piece c (16 bytes) of a row is at place c ^ swap(row).  So 16 lanes that read one piece of 16 rows, and 16 lanes that read four pieces of
// four rows, touch every bank once, and most of an address is a constant: a lane keeps one for every bit of the piece's number that is swapped.
template <int D> struct Plane {
    static constexpr int ROW = 2 * D, ROWS = 512 / D, STEP = D == 128 ? 1040 : 1056, BYTES = TILE / ROWS * STEP;
    static DEVINL int swap(const int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2 | ((r >> 2) & 1); }
    static DEVINL lds_t at(const int r, const int c) { return r / ROWS * STEP + r % ROWS * ROW + ((c ^ swap(r)) << 4); }
};
// rows of a Plane as the first operand with the channels along the contraction: lane = row, `a` the addresses for row lane & 31 and channels 32 n
template <int D> struct RowReader {
    lds_t a[D / 32];
    DEVINL RowReader(const int lane) {
#pragma unroll
        for (int n = 0; n < D / 32; ++n) a[n] = Plane<D>::at(lane & 31, 4 * n + (lane >> 5));
    }
    DEVINL u32x4 operator()(const lds_t base, const int rows32, const int s) const { return lds_ld<u32x4>(a[s / 2] + base + rows32 * (32 / Plane<D>::ROWS) * Plane<D>::STEP + s % 2 * 32); }
    DEVINL void move(const int by) {
#pragma unroll
        for (int n = 0; n < D / 32; ++n) a[n] += by;
    }
};
// ... with the rows along the contraction, in accumulator order: lane = channel of a block of 32
template <int D> struct ColReader {
    lds_t a[D / 32];
    DEVINL ColReader(const int lane) {
        const int l = lane & 15, r = 4 * (lane >> 5) + (l >> 2);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) a[d] = Plane<D>::at(r, 4 * d + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) + 8 * (l & 1);
    }
    DEVINL u32x4 operator()(const lds_t base, const int rows16, const int d) const {
        typedef v4s __attribute__((address_space(3))) * ptr;
        constexpr int EIGHT = 8 / Plane<D>::ROWS * Plane<D>::STEP;  // eight rows
        const lds_t o = a[d] + base + rows16 * 2 * EIGHT;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(o)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(o + EIGHT));
        const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
        return u32x4{x[0], x[1], y[0], y[1]};
    }
    DEVINL void move(const int by) {
#pragma unroll
        for (int d = 0; d < D / 32; ++d) a[d] += by;
    }
};
// keeps an operand where the program has it made: left to itself the compiler moves it to its use, behind the products that it should run beside
DEVINL void here(u32x4& x) { asm volatile("" : "+v"(x)); }
DEVINL void here(float& x) { asm volatile("" : "+v"(x)); }

// The way of a tile of 64 rows from memory straight to LDS: 16 bytes a lane, a wave's 1024 bytes in the order of its lanes, so that each lane fetches the piece whose
// place it is.  Rows behind the last and channels behind N come as zeros (the buffer's bounds).  The compiler does not count these loads: arrived() before the barrier behind which they are read.  Of the waves of a
// workgroup each brings every WAVES-th kilobyte.
// The bounds are those of the tile's own rows, of all that are left: 31 bits hold no more than a tile.
constexpr uint32_t NOWHERE = 0x7ffffff0u;                       // an offset beyond all bounds: such lanes bring zeros
__host__ __device__ __forceinline__ constexpr uint32_t tile_bytes(const int rows, const int step, const int N) { return rows > 0 ? ((rows < TILE ? rows : TILE) - 1) * step + 2 * N : 0; }
static_assert(tile_bytes(INT_MAX, 2 * (MAX_TOKEN_STRIDE - 1), 128) <= NOWHERE && tile_bytes(INT_MAX, 2 * (MAX_TOKEN_STRIDE - 1), 128) == 63u * 2 * (MAX_TOKEN_STRIDE - 1) + 256, "a tile in 31 bits");
static_assert(tile_bytes(TILE, 256, 128) == TILE * 256 && tile_bytes(TILE + 1, 256, 128) == TILE * 256 && tile_bytes(TILE - 1, 256, 128) == (TILE - 1) * 256, "a tile's rows");
static_assert(tile_bytes(1, 2 * (MAX_TOKEN_STRIDE - 1), 8) == 16 && tile_bytes(0, 256, 128) == 0 && tile_bytes(-1, 256, 128) == 0, "the last rows, and none");
template <int D, int WAVES> struct Fetch {
    static constexpr int LANES = D / 8, ROWS = Plane<D>::ROWS, STEPS = TILE / (ROWS * WAVES);
    uint32_t row, off;
    DEVINL Fetch(const int tid, const int N) {
        const int lane = tid & 63;
        row = (tid >> 6) * ROWS + lane / LANES;
        const int piece = (lane % LANES) ^ Plane<D>::swap(row);
        off = 8 * piece < N ? 16 * piece : NOWHERE;
    }
    // the rows from `first` on, of which `rows` are left, `step` bytes apart, to the plane at `to`; of those only the ones whose bit is set
    template <bool SOME> DEVINL void operator()(const lds_t to, const void* first, const int rows, const int step, const int N, const uint64_t which) const {
        const buf_t b = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(first), 0, tile_bytes(rows, step, N), 0x00027000);
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        uint32_t first_off = off;
        asm volatile("" : "+v"(first_off));                     // (offsets are made anew: kept, they would be spilled, and a reload waits for all that is under way)
        const bool on = first_off != NOWHERE;
        first_off += on ? row * step : 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            uint32_t o = first_off + (on ? i * ROWS * WAVES * step : 0);
            if (SOME) o = which >> (row + i * ROWS * WAVES) & 1 ? o : NOWHERE;
            // (M0 is read one wait state after it is written)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(to + (i * WAVES + wave) * Plane<D>::STEP), "v"(o), "s"(b) : "memory", "m0");
        }
    }
};
// Rows of padding may hold anything, and count as zeros where rows are summed.  Called by all of a workgroup's threads; the barrier behind it is here.
template <int D, int WAVES = 4> DEVINL void clear_padding(const lds_t plane, const int* docs) {
    constexpr int SHARE = WAVES;                                // threads of a row
    const int r = threadIdx.x / SHARE;
    if (docs[r] < 0)
        for (int c = threadIdx.x % SHARE; c < D / 8; c += SHARE) lds_st(plane + Plane<D>::at(r, c), u32x4{0, 0, 0, 0});
    __syncthreads();
}
// The order of what stands before it: a product, and its part of the LDS reads and of the other instructions.
template <int PRODUCTS, int READS, int VALUS, int TRANS> DEVINL void beside() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int c = 0; c < PRODUCTS; ++c) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, (READS + PRODUCTS - 1) / PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (VALUS + PRODUCTS - 1) / PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, (TRANS + PRODUCTS - 1) / PRODUCTS, 0);
    }
}
DEVINL void arrived() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

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

// how many of the first keys are seen from everywhere; a prefix lies on the GPU and may be any number
DEVINL int reach_of(const rwkv_attn_args& p, const int b) { return p.prefix ? max(0, min(p.prefix[b], p.Tk)) : 0; }
// head (or group) c of n of an item whose blocks follow each other: neighbours to one XCD where that comes out even
DEVINL int dealt(const int c, const int n) { return n % 8 == 0 ? (c & 7) * (n >> 3) + (c >> 3) : c; }
__host__ __device__ __forceinline__ int64_t tiles_of(const int T) { return (wide(T) + TILE - 1) / TILE; }
// The tiles first .. end - 1 that hold tokens of documents lo .. hi, from the first on or, BACK, from the last, and whether each is whole and all of the one document
// lo (= hi).  Without documents: all.
template <bool DOC, bool BACK> struct Walk {
    const Range* ranges;
    int lo, hi, first, count, base;                             // steps 0 .. count - 1; those from base on are in the masks
    uint64_t some, full;
    int u, t;                                                   // the step, and its tile
    bool whole;
    DEVINL Walk(const Range* ranges, const int lo, const int hi, const int first, const int end)
        : ranges(ranges), lo(lo), hi(hi), first(first), count(max(0, end - first)), base(0), some(0), full(0), u(0), t(0), whole(true) {
        if (DOC && count > 0) look();
        settle();
    }
    DEVINL bool more() const { return u < count; }
    DEVINL int tile(const int step) const { return BACK ? first + count - 1 - step : first + step; }
    DEVINL void look() {
        const int i = base + static_cast<int>(threadIdx.x & 63);
        Range r = {INT_MAX, -1, 0, 0};
        if (i < count) r = ranges[tile(i)];
        some = __ballot(r.lo <= hi && r.hi >= lo);
        full = __ballot(r.whole && r.lo == lo && r.hi == lo && lo == hi);
    }
    DEVINL void settle() {                                      // to the first step from u on whose tile is looked at
        if constexpr (DOC)
            while (u < count) {
                if (u - base >= 64) { base = u; look(); }
                const uint64_t left = some >> (u - base);
                if (left) {
                    u += __builtin_ctzll(left);
                    whole = full >> (u - base) & 1;
                    break;
                }
                u = base + 64;
            }
        t = tile(u);
    }
    DEVINL void next() {
        ++u;
        if constexpr (!DOC) asm volatile("" : "+s"(u));         // (no sums of the tile's number kept from one to the next: they cost registers)
        settle();
    }
};

}  // namespace

}  // namespace rwkv
