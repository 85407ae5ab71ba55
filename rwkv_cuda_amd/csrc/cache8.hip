// A paged cache in 8 bits: writing it (the arguments are explained in rwkv_hip.h).
//
// A scale belongs to a page and head, so the tokens that go into one page are one wave's, for one head and for keys or values: a pass for the
// largest magnitude, the scale, a pass that rounds (its reads hit the cache), and, where the page held tokens and its scale grew, those once more.  Scales are powers
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

template <class E>
__global__ __launch_bounds__(64 * WAVES) void cache8_write(const rwkv_cache8_args p, const int shift, const int window, const int windows) {
    const int lane = threadIdx.x & 63, pieces = p.N / 8;        // of 8 values; a lane has one of them, in every 64 / width-th token
    const int width = p.N <= 64 ? 8 : 16, piece = lane & (width - 1), row = lane / width, rows = 64 / width;
    const bool on = piece < pieces;
    const int64_t work = static_cast<int64_t>(blockIdx.x) * WAVES + (threadIdx.x >> 6);
    const int head = static_cast<int>(work % p.Hk), kv = static_cast<int>(work / p.Hk % 2);
    const int64_t at = work / p.Hk / 2;
    if (at >= windows) return;
    const int w0 = static_cast<int>(at) * window;
    const E* x = static_cast<const E*>(kv ? p.v : p.k) + head * (kv ? p.v_sh : p.k_sh) + 8 * piece;
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
        int end = begin + 1, first = INT_MAX;
        for (int i = begin;; i += 64) {
            const bool same = page_of(i + lane) == page;
            const uint64_t other = ~__ballot(same);
            const int n = other == 0ull ? 64 : __builtin_ctzll(other);
            if (lane < n) first = min(first, p.slots[i + lane] & mask);
            end = i + n;
            if (n < 64) break;
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) first = min(first, __shfl_xor(first, m, 64));
        float top = 0.f;
        for (int i = begin + row; i < end; i += rows) {
            if (!on) continue;
            float f[8];
            values8<E>(*reinterpret_cast<const u32x4*>(x + i * xt), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_bits(__float_as_uint(f[e])) ? fabsf(f[e]) : 0.f);
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
        const float need = power(exponent_for(top)), old = scales[static_cast<int64_t>(page) * p.Hk], scale = first > 0 ? fmaxf(need, old) : need;
        const float by = 1.f / scale;
        uint8_t* to = pages + page * sp;
        for (int i = begin + row; i < end; i += rows) {
            if (!on) continue;
            float f[8];
            values8<E>(*reinterpret_cast<const u32x4*>(x + i * xt), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = finite_bits(__float_as_uint(f[e])) ? f[e] * by : NAN;
            *reinterpret_cast<u32x2*>(to + (p.slots[i] & mask) * st) = u32x2{codes4(f[0], f[1], f[2], f[3]), codes4(f[4], f[5], f[6], f[7])};
        }
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
// prompt's tokens fill pages, and most begin none), up to a page or the lanes of a wave.
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
    hipLaunchKernelGGL(cache8_write<E>, dim3(static_cast<unsigned>(blocks)), dim3(64 * WAVES), 0, st, p, __builtin_ctz(p.page), window, windows);
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
