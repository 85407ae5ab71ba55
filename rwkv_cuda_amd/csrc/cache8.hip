// A paged cache in 8 bits: writing it (the arguments are explained in rwkv_hip.h).
//
// A scale belongs to a page and head, so the tokens that go into one page are one wave's, for one head and for keys or values: a pass for the
// largest magnitude, the scale, a pass that rounds (the first HOLD rows of the wave stay in registers and are on their way at once, others are read again), and, where the page held tokens and its scale grew, those once more.  Scales are powers
// of two: a token's own rounding is all that is lost until its page's scale grows, and a second one is the first one's number where no bits fall off.
#include <climits>

#include "mixers.h"

namespace rwkv {
namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int WAVES = 4, LEAST = -100;                          // the least scale's exponent
DEVINL bool finite_bits(const uint32_t x) { return (x & 0x7f800000u) != 0x7f800000u; }
template <class E> DEVINL void values8(const u32x4 x, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<E, bf16_t>) f[2 * i] = bf_lo(x[i]), f[2 * i + 1] = bf_hi(x[i]);
        else {
            f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x[i])));
            f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x[i] >> 16)));
        }
    }
}
// Magnitudes of 16-bit numbers are ordered as their bits without the sign.
DEVINL uint32_t larger(const uint32_t a, const uint32_t b) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <class E> DEVINL uint32_t largest(const u32x4 x, const uint32_t than) {
    return larger(larger(than, x[0] & 0x7fff7fffu), larger(larger(x[1] & 0x7fff7fffu, x[2] & 0x7fff7fffu), x[3] & 0x7fff7fffu));
}
// ... infinities and NaN as zeros
template <class E> DEVINL u32x4 finite_ones(u32x4 x) {
    constexpr uint32_t TOP = std::is_same_v<E, bf16_t> ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] &= ((x[i] & TOP) == TOP ? 0u : 0xffffu) | ((x[i] >> 16 & TOP) == TOP ? 0u : 0xffff0000u);
    return x;
}
// four values as codes, to nearest even; none is above 448
DEVINL uint32_t codes4(const float a, const float b, const float c, const float d) {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    x = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, x, true);
    return static_cast<uint32_t>(x);
}
DEVINL uint32_t refit4(const uint32_t x, const float by) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
    return codes4(a[0] * by, a[1] * by, b[0] * by, b[1] * by);
}
// the exponent of the least power of two by which values up to `top` stay within 448 = 1.75 2^8
DEVINL int exponent_for(const float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, LEAST);
}
DEVINL float power(const int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }     // -126 .. 127

template <class E, int HOLD>
__global__ __launch_bounds__(64 * WAVES) void cache8_write(const rwkv_cache8_args p, const int shift, const int window, const int windows) {
    const int lane = threadIdx.x & 63, pieces = p.N / 8;        // of 8 values; a lane has one of them, in every 64 / width-th token
    const int width = p.N <= 64 ? 8 : 16, piece = lane & (width - 1), row = lane / width, rows = 64 / width;
    const bool on = piece < pieces;
    const int64_t work = static_cast<int64_t>(blockIdx.x) * WAVES + (threadIdx.x >> 6);
    const int head = static_cast<int>(work % p.Hk), kv = static_cast<int>(work / p.Hk % 2);
    const int64_t at = work / p.Hk / 2;
    if (at >= windows) return;
    const int w0 = static_cast<int>(at) * window;
    const E* x = static_cast<const E*>(kv ? p.v : p.k) + head * (kv ? p.v_sh : p.k_sh) + (on ? 8 * piece : 0);
    const int64_t xt = kv ? p.v_st : p.k_st, sp = kv ? p.vp_sp : p.kp_sp, st = kv ? p.vp_st : p.kp_st;
    uint8_t* pages = static_cast<uint8_t*>(kv ? p.v_pages : p.k_pages) + head * (kv ? p.vp_sh : p.kp_sh) + 8 * piece;
    float* scales = (kv ? p.v_scales : p.k_scales) + head;
    const int mask = p.page - 1;
    const auto page_of = [&](int i) {                           // -1: outside the cache
        const int s = i >= 0 && i < p.n ? p.slots[i] : -1;
        return s < 0 || (s >> shift) >= p.P ? -1 : s >> shift;
    };
    const int mine = lane < window ? page_of(w0 + lane) : -1, before = __shfl_up(mine, 1, 64), left = lane == 0 ? page_of(w0 - 1) : before;
    uint64_t starts = __ballot(mine >= 0 && mine != left);
    while (starts != 0ull) {
        const int s = __builtin_ctzll(starts);
        starts &= starts - 1;
        const int begin = w0 + s, page = __shfl(mine, s, 64);
        // up to the next token of another page, and the first place that is written
        int end = begin + 1, first = INT_MAX, place = 0;        // place: of token begin + lane
        for (int i = begin;; i += 64) {
            const bool same = page_of(i + lane) == page;
            const uint64_t other = ~__ballot(same);
            const int n = other == 0ull ? 64 : __builtin_ctzll(other);
            if (lane < n) {
                const int z = p.slots[i + lane] & mask;
                first = min(first, z), place = i == begin ? z : place;
            }
            end = i + n;
            if (n < 64) break;
        }
        u32x4 held[HOLD];
#pragma unroll
        for (int u = 0; u < HOLD; ++u)
            if (begin + rows * u < end) held[u] = *reinterpret_cast<const u32x4*>(x + min(begin + row + rows * u, end - 1) * xt);
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) first = min(first, __shfl_xor(first, m, 64));
        const float old = scales[static_cast<int64_t>(page) * p.Hk];
        const auto top_of = [&](auto only) {                    // (where rows end inside of the last access it is the last token's once more)
            uint32_t top = 0;
            const auto take = [&](const u32x4 v) { top = largest<E>(only ? finite_ones<E>(v) : v, top); };
#pragma unroll
            for (int u = 0; u < HOLD; ++u)
                if (begin + rows * u < end) take(held[u]);
            for (int i = begin + row + rows * HOLD; i < end; i += rows) take(*reinterpret_cast<const u32x4*>(x + i * xt));
            top = on ? max(top & 0xffff, top >> 16) : 0;
#pragma unroll
            for (int m = 32; m >= 1; m >>= 1) top = max(top, __shfl_xor(top, m, 64));
            return top;
        };
        uint32_t top = top_of(std::false_type());
        const bool odd = top >= (std::is_same_v<E, bf16_t> ? 0x7f80 : 0x7c00);      // infinities or NaN: a second look, without them
        if (odd) top = top_of(std::true_type());
        const float need = power(exponent_for(to_f(__builtin_bit_cast(E, static_cast<uint16_t>(top))))), scale = first > 0 ? fmaxf(need, old) : need;
        const float by = 1.f / scale;
        uint8_t* to = pages + page * sp;
        const auto put = [&](const u32x4 v, const int z) {
            float f[8];
            values8<E>(v, f);
            if (odd)
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = finite_bits(__float_as_uint(f[e])) ? f[e] : NAN;
            *reinterpret_cast<u32x2*>(to + z * st) = u32x2{codes4(f[0] * by, f[1] * by, f[2] * by, f[3] * by), codes4(f[4] * by, f[5] * by, f[6] * by, f[7] * by)};
        };
#pragma unroll
        for (int u = 0; u < HOLD; ++u)
            if (begin + rows * u < end) {
                const int n = row + rows * u, z = n < 64 ? __shfl(place, n & 63, 64) : p.slots[min(begin + n, end - 1)] & mask;
                if (on && begin + n < end) put(held[u], z);
            }
        for (int i = begin + row + rows * HOLD; i < end; i += rows)
            if (on) put(*reinterpret_cast<const u32x4*>(x + i * xt), p.slots[i] & mask);
        if (first > 0 && scale > old) {
            const float fit = old / scale;
            for (int i = row; i < first; i += rows) {
                if (!on) continue;
                u32x2* z = reinterpret_cast<u32x2*>(to + i * st);
                const u32x2 c = *z;
                *z = u32x2{refit4(c[0], fit), refit4(c[1], fit)};
            }
        }
        if (lane == 0 && scale != old) scales[static_cast<int64_t>(page) * p.Hk] = scale;
    }
}

// How many tokens a wave looks through for pages that begin: one while waves are few (a token of each of many sequences: a page each), more as there are more of them (a
// prompt's tokens fill pages, and most begin none), up to a page or the lanes of a wave.  And how many rows it keeps: 16 where it looks through more than 8 tokens, 4 below, where most runs are of
// one token and the longer code and the registers only cost.  us, 8 heads of 128, with 4096, 8192, 32768 waves (4 rows up to 4 tokens), and 8192 waves with 4 rows up to 8:
//   64 sequences of one token 4.5 4.2 4.5 4.7;   1024 of one 9.4 10.0 11.6 10.1;   4096 of one 72 59 30 27;   256 of 8 8.9 8.4 22 8.3;   one prompt of 1000 11.4 12.7 12.8 12.7;   4 of 1000
//   (pages of 16) 10.0 10.2 25 7.7;   4 of 2000 13.9 14.3 35 14.4;   16 of 2000 41.6 41.6 39.2 41.7, which is 202 MB at 4.8 TB/s
constexpr int BUSY = 8192;
int window_of(const rwkv_cache8_args& p) {
    const int64_t waves = 2ll * p.n * p.Hk;
    int w = 1;
    while (w < 64 && w < p.page && waves / w > BUSY) w *= 2;
    return w;
}
template <class E> int run(hipStream_t st, const rwkv_cache8_args& p) {
    const int window = window_of(p), windows = static_cast<int>((static_cast<int64_t>(p.n) + window - 1) / window);
    const int64_t blocks = (2ll * windows * p.Hk + WAVES - 1) / WAVES;
    if (blocks > INT_MAX) return RWKV_ERR_SHAPE;
    const auto kernel = window > 8 ? cache8_write<E, 16> : cache8_write<E, 4>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * WAVES), 0, st, p, __builtin_ctz(p.page), window, windows);
    return launch_status();
}

int check_write(const rwkv_cache8_args* p) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->n <= 0 || p->n > INT_MAX - 65536 || p->Hk <= 0 || p->Hk > 65535 || p->N <= 0 || p->N > 128 || p->N % 16 != 0 ||
        p->P <= 0 || p->page <= 0 || (p->page & (p->page - 1)) != 0) return RWKV_ERR_SHAPE;
    for (const int64_t s : {p->k_st, p->k_sh, p->v_st, p->v_sh}) if (s % 8 != 0) return RWKV_ERR_ALIGN;
    for (const int64_t s : {p->kp_sp, p->kp_st, p->kp_sh, p->vp_sp, p->vp_st, p->vp_sh}) if (s % 16 != 0) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->k, p->v, p->k_pages, p->v_pages})) return rc;
    for (const void* x : {static_cast<const void*>(p->k_scales), static_cast<const void*>(p->v_scales), static_cast<const void*>(p->slots)}) {
        if (x == nullptr) return RWKV_ERR_NULL;
        if (reinterpret_cast<uintptr_t>(x) & 3) return RWKV_ERR_ALIGN;
    }
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" int rwkv_cache8_write(void* stream, const rwkv_cache8_args* args) {
    using namespace rwkv;
    if (const int rc = check_write(args)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return args->dtype == RWKV_DTYPE_BF16 ? run<bf16_t>(st, *args) : run<half_t>(st, *args);
}
