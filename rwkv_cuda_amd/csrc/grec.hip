// Gated linear recurrence, channel by channel: h_t = a_t h_{t-1} + u_t, y_t = h_t (the arguments are explained in rwkv_hip.h).
// Backward, with d_t the gradient of h_t:  d_t = dy_t + a_{t+1} d_{t+1};  da_t = d_t h_{t-1};  du_t = d_t.
#include <climits>

#include "common.h"
#include "mixers.h"

namespace rwkv {
namespace {
// The map of a run of tokens on the state before it is h -> A h + B, and two such maps one after the other are one again; so is the way
// back of the gradient, with the same A.  A thread holds S tokens of two channels in registers and makes their map, a workgroup (32 threads
// side by side: 64 channels, a 128-byte row; G groups of S tokens) joins the groups' maps in LDS, and so it has the states of a tile of 8 G
// tokens.  Over the whole length, with columns of 64 channels enough for every CU a workgroup goes through its column tile by tile (the
// forward with the next one's inputs under way); with fewer a workgroup has one tile: it publishes its map, looks back over the maps of the
// tiles before it to one whose end state is known, and publishes its own end state.  Every input is read once and every output written once.
// Progress of the latter: a column's tiles are numbered by a ticket that a workgroup takes when it runs, a tile publishes its map before it
// waits, and it waits for lower tickets of its column only: the lowest unfinished one waits for nothing.  (A counter a column: with one for
// all a T3001 C1536 fp16 forward took 25 us instead of 17.)
// Bound by memory.  bf16 B8 T4096 C4096: forward 0.195 ms (805 MB, 4.1 TB/s; a copy reaches 6.0), backward 0.29 ms (1342 MB, 4.6 TB/s).
constexpr int S = 8, MAX_GROUPS = 16;

inline int groups_of(int T) { const int g = (T + S - 1) / S; return g >= MAX_GROUPS ? MAX_GROUPS : (g + 1) / 2 * 2; }
inline int tiles_of(int T) { return (T + S * groups_of(T) - 1) / (S * groups_of(T)); }

// e^x to about two roundings (x log2(e) in two parts); infinities are exact and a NaN stays one
DEVINL float exp_of(const float x, const float most) {
    const float raw = x * 1.4426950408889634f, low = fmaf(x, 1.9259629911266175e-8f, fmaf(x, 1.4426950408889634f, -raw));
    const float z = raw > most ? most : raw, e = __builtin_amdgcn_exp2f(z);
    return fmaf(e, fabsf(raw) < 115.f ? low * 0.6931471805599453f : 0.f, e);
}
// Two workgroups a CU and more: each goes through its column.  Fewer: the tiles are workgroups of their own.  Forward + backward in us, going through / chained, T 4096:
// bf16 512 columns 187 + 301 / 198 + 352, 384 columns 165 + 247 / 152 + 262, 256 columns 103 + 185 / 102 + 173, 64 columns 91 + 121 / 28 + 42; fp32 512 columns
// 325 + 571 / 320 + 536, 256 columns 234 + 279 / 158 + 269; T 512: bf16 512 columns 22 + 37 / 26 + 42, 2048 columns 92 + 149 / 97 + 170.
inline bool chained(int B, int T, int C) { return tiles_of(T) > 1 && static_cast<int64_t>((C + 63) / 64) * B < 512; }

// gate and its complement, both to fp32's accuracy
template <int GATE> DEVINL void gate_of(const float w, float& a, float& rest) {
    if constexpr (GATE == RWKV_GATE_SIGMOID) {
        const float e = exp_of(-w, 115.f);                       // below w = -80 the gate is 2^-115
        a = __builtin_amdgcn_rcpf(1.f + e);
        rest = e * a;
    } else {
        a = exp_of(w, INFINITY);
        rest = -expm1f(w);
    }
}

// A of a run in which a document starts: what was before does not count, not even an infinity
constexpr uint32_t CUT = 0x80000000u;
DEVINL bool is_cut(const float a) { return __float_as_uint(a) == CUT; }
struct Map { float a, b; };
// GROWS: a run's A, a product of gates, may be an infinity where no gate is (log gates above 0): of a state of zero nothing comes all the same.  (Only there: with it
// everywhere the bf16 layer's forward took 198 us, not 195.)
template <bool DOC, bool GROWS = false> DEVINL float apply(const Map m, const float h) { return DOC && is_cut(m.a) ? m.b : fmaf(GROWS && h == 0.f ? 0.f : m.a, h, m.b); }
template <bool DOC, bool GROWS = false> DEVINL Map after(const Map second, const Map first) {
    if (DOC && is_cut(second.a)) return second;
    return {DOC && is_cut(first.a) ? first.a : second.a * first.a, apply<false, GROWS>(second, first.b)};
}

template <class E> struct Two;
template <> struct Two<bf16_t> { typedef uint32_t raw; static DEVINL float lo(raw x) { return bf_lo(x); } static DEVINL float hi(raw x) { return bf_hi(x); } static DEVINL raw make(float a, float b) { return pack_bf2(a, b); } };
template <> struct Two<half_t> {
    typedef uint32_t raw;
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    static DEVINL float lo(raw x) { return static_cast<float>(__builtin_bit_cast(h2, x)[0]); }
    static DEVINL float hi(raw x) { return static_cast<float>(__builtin_bit_cast(h2, x)[1]); }
    static DEVINL raw make(float a, float b) { const h2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)}; return __builtin_bit_cast(raw, h); }
};
template <> struct Two<float> { typedef float2 raw; static DEVINL float lo(raw x) { return x.x; } static DEVINL float hi(raw x) { return x.y; } static DEVINL raw make(float a, float b) { return {a, b}; } };
// two neighbouring channels, of which `n` are there; VEC: both, and on a boundary of two
template <class E, bool VEC> DEVINL typename Two<E>::raw load2(const E* p, const int n) {
    if constexpr (VEC) return *reinterpret_cast<const typename Two<E>::raw*>(p);
    else return Two<E>::make(n > 0 ? to_f(p[0]) : 0.f, n > 1 ? to_f(p[1]) : 0.f);
}
template <class E, bool VEC> DEVINL void store2(E* p, const int n, float a, float b) {
    asm("" : "+v"(a), "+v"(b));                                 // (no fp16 multiply-add that rounds once: what is stored does not depend on how)
    if constexpr (VEC) *reinterpret_cast<typename Two<E>::raw*>(p) = Two<E>::make(a, b);
    else { if (n > 0) p[0] = from_f<E>(a); if (n > 1) p[1] = from_f<E>(b); }
}

// ----------------------------------------------------------------------------- the chain of tiles
// What a tile publishes is its own sign of being there: memory is filled with ones before, and no value is stored as that NaN.
typedef unsigned long long u64;
DEVINL float no_ones(const float x) { return __float_as_uint(x) == 0xffffffffu ? __uint_as_float(0x7fc00000u) : x; }
struct Chain {
    u64* maps;                                                  // [tiles][columns of 64][64]
    uint32_t* ends;
    int64_t step;                                               // values of a tile
    DEVINL Chain(void* ws, const int64_t columns, const int tiles) {
        maps = reinterpret_cast<u64*>(static_cast<char*>(ws) + 64 * columns);      // (behind the tickets, a cache line each)
        ends = reinterpret_cast<uint32_t*>(maps + columns * 64 * tiles);
        step = columns * 64;
    }
    DEVINL void publish(const int64_t at, const Map m) const {
        __hip_atomic_store(maps + at, static_cast<u64>(__float_as_uint(no_ones(m.b))) << 32 | __float_as_uint(m.a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    DEVINL void publish(const int64_t at, const float h) const { __hip_atomic_store(ends + at, __float_as_uint(no_ones(h)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
    // the state before the tile whose values begin at `at`, `n` tiles (at least one) before it in the order of the tickets: the nearest known end state
    // through the maps of the tiles between, one by one, so that its bits do not depend on which that is
    template <bool DOC, bool GROWS> DEVINL float look_back(const int64_t at, const int n) const {
        constexpr int BACK = 4;
        for (int polls = 0; polls < 1 << 22; ++polls) {          // (bounded, so that no mistake can hang the GPU: it would end as a NaN)
            u64 m[BACK];
            uint32_t e[BACK];
#pragma unroll
            for (int i = 0; i < BACK; ++i) {
                const int64_t o = at - (i < n ? i + 1 : n) * step;
                e[i] = __hip_atomic_load(ends + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                m[i] = __hip_atomic_load(maps + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            bool known = false;
            float h = 0.f;
#pragma unroll
            for (int i = BACK - 1; i >= 0; --i) {
                if (e[i] != 0xffffffffu) h = __uint_as_float(e[i]), known = true;
                else if (m[i] == ~0ull) known = false;
                else h = apply<DOC, GROWS>({__uint_as_float(static_cast<uint32_t>(m[i])), __uint_as_float(static_cast<uint32_t>(m[i] >> 32))}, h);
            }
            if (known) return h;
            __builtin_amdgcn_s_sleep(1);
        }
        return __uint_as_float(0x7fc00000u);
    }
};
__global__ __launch_bounds__(256) void grec_clear(uint4* p, const int64_t n) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// where a workgroup works
struct Place {
    int tile, b, c, n, t0, groups;                              // c: the thread's first channel, n: how many of its two are there, t0: its first token
    int first;                                                  // the workgroup's first token
    int64_t value;                                              // of channel 0 of the tile in [tile][column][64]
    // `order`: how many of the column's tiles come before this one
    DEVINL Place(const rwkv_grec_args& p, const int tiles, const int64_t col, const int order, const bool reverse) {
        const int cols = (p.C + 63) / 64;
        value = (order * static_cast<int64_t>(cols) * p.B + col) * 64;
        tile = reverse ? tiles - 1 - order : order;
        b = static_cast<int>(col / cols);
        c = static_cast<int>(col % cols) * 64 + 2 * (threadIdx.x & 31);
        n = p.C - c;
        groups = blockDim.x >> 5;
        go(tile);
    }
    DEVINL void go(const int to) {
        tile = to;
        first = to * groups * S;
        t0 = first + (threadIdx.x >> 5) * S;
    }
    DEVINL int there(const rwkv_grec_args& p) const { return n <= 0 ? 0 : p.T - t0 < S ? p.T - t0 : S; }      // the thread's tokens that there are (may be below zero)
};
// a thread's S tokens of [B,T,C]: the token's address is the same for the whole workgroup and the thread's part 32 bits, so that 24 accesses take one register of
// addresses each array (with 64 bits a thread, and pairs kept unpacked below, the backward
// spilled 28 registers and took 0.64 ms instead of 0.35 at B8 T4096 C4096, chained).  VEC promises that 32 bits do.
template <class E, bool VEC> struct Rows {
    char* base;
    int64_t step;
    std::conditional_t<VEC, uint32_t, int64_t> part;
    DEVINL Rows(const void* p, const Place& at, const int64_t sb, const int64_t st) {
        base = static_cast<char*>(const_cast<void*>(p)) + (at.b * sb + at.first * st) * static_cast<int64_t>(sizeof(E));
        step = st * static_cast<int64_t>(sizeof(E));
        part = static_cast<decltype(part)>(((threadIdx.x >> 5) * S * st + at.c) * static_cast<int64_t>(sizeof(E)));
    }
    DEVINL E* at(const int i) const { return reinterpret_cast<E*>(base + i * step + part); }
};
// the next tile of a column
DEVINL int take_ticket(void* ws, const int64_t col) {
    __shared__ uint32_t ticket;
    if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(static_cast<uint32_t*>(ws) + 16 * col, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(ticket);
}
// which of a thread's tokens are real, and which of them start a document
DEVINL void marks(const rwkv_grec_args& p, const Place& at, uint32_t& real, uint32_t& first) {
    const int* doc = p.doc + static_cast<int64_t>(at.b) * p.T;
    real = first = 0;
    int before = at.t0 > 0 && at.t0 <= p.T ? doc[at.t0 - 1] : 0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int t = at.t0 + i, d = t < p.T ? doc[t] : -1;
        if (d >= 0) real |= 1u << i;
        if (d >= 0 && t > 0 && d != before) first |= 1u << i;
        before = d;
    }
}

template <class E, int GATE, bool TIED, bool DOC, bool VEC, bool CHAIN>
__global__ __launch_bounds__(512, 4) void grec_fwd(const rwkv_grec_args p, const int tiles) {
    constexpr bool GROWS = GATE == RWKV_GATE_LOG;
    __shared__ float map_a[MAX_GROUPS][64], map_b[MAX_GROUPS][64], before[64];
    const int64_t columns = static_cast<int64_t>((p.C + 63) / 64) * p.B, col = blockIdx.x % columns;
    Place at(p, tiles, col, CHAIN ? take_ticket(p.workspace, col) : 0, false);
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = at.c - 2 * lane + (threadIdx.x & 63);
    const bool there = c < p.C;                                  // of the first wave: the channel it joins the groups of
    const int64_t row = static_cast<int64_t>(at.b) * p.C + c;
    typename Two<E>::raw wr[S], xr[S];
    const auto load = [&](const Place& at) {
        const Rows<E, VEC> w(p.w, at, p.w_sb, p.w_st), x(p.x, at, p.x_sb, p.x_st);
        const int there = at.there(p);
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i < there) {
                wr[i] = load2<E, VEC>(w.at(i), at.n);
                xr[i] = load2<E, VEC>(x.at(i), at.n);
            }
    };
    load(at);
    float state = p.h0 && there ? p.h0[row] : 0.f;               // of the first wave, before the tile
    for (;;) {
        const int n = at.there(p);
        uint32_t real = 0, first = 0;
        if constexpr (DOC) marks(p, at, real, first);
        float a[S][2], u[S][2];
        Map m[2] = {{1.f, 0.f}, {1.f, 0.f}};
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool on = i < n && (!DOC || (real >> i & 1));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[i][e] = 1.f;
                u[i][e] = 0.f;
                if (on) {
                    float rest;
                    gate_of<GATE>(e ? Two<E>::hi(wr[i]) : Two<E>::lo(wr[i]), a[i][e], rest);
                    const float z = e ? Two<E>::hi(xr[i]) : Two<E>::lo(xr[i]);
                    u[i][e] = TIED ? rest * z : z;
                    if (DOC && (first >> i & 1)) a[i][e] = __uint_as_float(CUT);
                }
                m[e] = after<DOC>({a[i][e], u[i][e]}, m[e]);
            }
        }
        const bool more = !CHAIN && at.tile + 1 < tiles;
        Place next = at;
        next.go(at.tile + 1);
        if (more) load(next);
#pragma unroll
        for (int e = 0; e < 2; ++e) map_a[g][2 * lane + e] = m[e].a, map_b[g][2 * lane + e] = m[e].b;
        __syncthreads();
        if (threadIdx.x < 64) {
            const int64_t value = at.value + threadIdx.x;
            Map all = {1.f, 0.f};
#pragma unroll 4
            for (int k = 0; k < at.groups; ++k) {                // what is before each group, within the tile
                const Map own = {map_a[k][threadIdx.x], map_b[k][threadIdx.x]};
                map_a[k][threadIdx.x] = all.a;
                map_b[k][threadIdx.x] = all.b;
                all = after<DOC, GROWS>(own, all);
            }
            if constexpr (CHAIN) {
                const Chain chain(p.workspace, columns, tiles);
                if (at.tile > 0) {
                    if (at.tile + 1 < tiles) chain.publish(value, all);
                    state = chain.look_back<DOC, GROWS>(value, at.tile);
                }
                if (at.tile + 1 < tiles) chain.publish(value, apply<DOC, GROWS>(all, state));
            }
            before[threadIdx.x] = state;
            if (there && p.saved) p.saved[(static_cast<int64_t>(at.b) * tiles + at.tile) * p.C + c] = state;
            state = apply<DOC, GROWS>(all, state);
            if (there && at.tile + 1 == tiles) p.hT[row] = state;
        }
        __syncthreads();
        if (at.n > 0) {
            float h[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) h[e] = apply<DOC, GROWS>({map_a[g][2 * lane + e], map_b[g][2 * lane + e]}, before[2 * lane + e]);
            const Rows<E, VEC> y(p.y, at, static_cast<int64_t>(p.T) * p.C, p.C);
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (i >= n) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) h[e] = apply<DOC>({a[i][e], u[i][e]}, h[e]);
                const bool on = !DOC || (real >> i & 1);
                store2<E, VEC>(y.at(i), at.n, on ? h[0] : 0.f, on ? h[1] : 0.f);
            }
        }
        if (!more) break;
        at = next;
        __syncthreads();
    }
}

// c: the gradient that comes to the state behind a token from later ones; d = dy + c, and c = a d goes on
template <class E, int GATE, bool TIED, bool DOC, bool VEC, bool CHAIN>
__global__ __launch_bounds__(512, 4) void grec_bwd(const rwkv_grec_args p, const int tiles) {
    constexpr bool GROWS = GATE == RWKV_GATE_LOG;
    __shared__ float map_a[MAX_GROUPS][64], map_b[MAX_GROUPS][64], back_a[MAX_GROUPS][64], back_b[MAX_GROUPS][64], before[64], behind[64];
    const int64_t columns = static_cast<int64_t>((p.C + 63) / 64) * p.B, col = blockIdx.x % columns;
    Place at(p, tiles, col, CHAIN ? take_ticket(p.workspace, col) : 0, true);
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, wave = threadIdx.x >> 6, i64 = threadIdx.x & 63, c = at.c - 2 * lane + i64;
    const bool there = c < p.C;
    const int64_t row = static_cast<int64_t>(at.b) * p.C + c;
    typename Two<E>::raw wr[S], xr[S], yr[S];
    const auto load = [&](const Place& at) {
        const Rows<E, VEC> w(p.w, at, p.w_sb, p.w_st), x(p.x, at, p.x_sb, p.x_st), dy(p.dy, at, static_cast<int64_t>(p.T) * p.C, p.C);
        const int there = at.there(p);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            yr[i] = Two<E>::make(0.f, 0.f);
            if (i < there) {
                wr[i] = load2<E, VEC>(w.at(i), at.n);
                xr[i] = load2<E, VEC>(x.at(i), at.n);
                if (p.dy) yr[i] = load2<E, VEC>(dy.at(i), at.n);
            }
        }
    };
    load(at);
    float back = p.dhT && there ? p.dhT[row] : 0.f;              // of the wave that joins the ways back: the gradient behind the tile
    for (;;) {
        const int n = at.there(p);
        uint32_t real = 0, first = 0;
        if constexpr (DOC) marks(p, at, real, first);
        float a[S][2], rest[S][2], h[S][2];                     // h: the input's part of the step, then the state before it
        Map m[2] = {{1.f, 0.f}, {1.f, 0.f}}, r[2] = {{1.f, 0.f}, {1.f, 0.f}};
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool on = i < n && (!DOC || (real >> i & 1));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[i][e] = 1.f;
                rest[i][e] = 0.f;
                h[i][e] = 0.f;
                if (on) {
                    gate_of<GATE>(e ? Two<E>::hi(wr[i]) : Two<E>::lo(wr[i]), a[i][e], rest[i][e]);
                    const float z = e ? Two<E>::hi(xr[i]) : Two<E>::lo(xr[i]);
                    h[i][e] = TIED ? rest[i][e] * z : z;
                }
                m[e] = after<DOC>({DOC && (first >> i & 1) ? __uint_as_float(CUT) : a[i][e], h[i][e]}, m[e]);
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool on = !DOC || (real >> i & 1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = DOC && (first >> i & 1) ? __uint_as_float(CUT) : a[i][e], d = on ? (e ? Two<E>::hi(yr[i]) : Two<E>::lo(yr[i])) : 0.f;
                r[e] = after<DOC>({f, DOC && is_cut(f) ? 0.f : f * d}, r[e]);
            }
        }
        if constexpr (sizeof(E) == 2) {                          // (kept as pairs, not as the 32 floats that were just made of them)
#pragma unroll
            for (int i = 0; i < S; ++i) asm("" : "+v"(xr[i]), "+v"(yr[i]));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            map_a[g][2 * lane + e] = m[e].a, map_b[g][2 * lane + e] = m[e].b;
            back_a[g][2 * lane + e] = r[e].a, back_b[g][2 * lane + e] = r[e].b;
        }
        __syncthreads();
        if (wave == 0) {
            Map all = {1.f, 0.f};
#pragma unroll 4
            for (int k = 0; k < at.groups; ++k) {
                const Map own = {map_a[k][i64], map_b[k][i64]};
                map_a[k][i64] = all.a;
                map_b[k][i64] = all.b;
                all = after<DOC, GROWS>(own, all);
            }
            before[i64] = there ? p.saved[(static_cast<int64_t>(at.b) * tiles + at.tile) * p.C + c] : 0.f;
        }
        if (wave == (at.groups > 2 ? 1 : 0)) {
            const int64_t value = at.value + i64;
            Map all = {1.f, 0.f};
#pragma unroll 4
            for (int k = at.groups - 1; k >= 0; --k) {
                const Map own = {back_a[k][i64], back_b[k][i64]};
                back_a[k][i64] = all.a;
                back_b[k][i64] = all.b;
                all = after<DOC, GROWS>(own, all);
            }
            if constexpr (CHAIN) {
                const Chain chain(p.workspace, columns, tiles);
                const int done = tiles - 1 - at.tile;
                if (done > 0) {
                    if (at.tile > 0) chain.publish(value, all);
                    back = chain.look_back<DOC, GROWS>(value, done);
                }
                if (at.tile > 0) chain.publish(value, apply<DOC, GROWS>(all, back));
            }
            behind[i64] = back;
            back = apply<DOC, GROWS>(all, back);
            if (there && at.tile == 0 && p.dh0) p.dh0[row] = back;
        }
        __syncthreads();
        if (at.n > 0) {
            float d[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float s = apply<DOC, GROWS>({map_a[g][2 * lane + e], map_b[g][2 * lane + e]}, before[2 * lane + e]);
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const float input = h[i][e];
                    if (DOC && (first >> i & 1)) s = 0.f;
                    h[i][e] = s;
                    s = fmaf(a[i][e], s, input);
                }
                d[e] = apply<DOC, GROWS>({back_a[g][2 * lane + e], back_b[g][2 * lane + e]}, behind[2 * lane + e]);
            }
            const Rows<E, VEC> dw(p.dw, at, static_cast<int64_t>(p.T) * p.C, p.C), dx(p.dx, at, static_cast<int64_t>(p.T) * p.C, p.C);
#pragma unroll
            for (int i = S - 1; i >= 0; --i) {
                if (i >= n) continue;
                float gw[2] = {0.f, 0.f}, gx[2] = {0.f, 0.f};
                if (!DOC || (real >> i & 1)) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        d[e] += e ? Two<E>::hi(yr[i]) : Two<E>::lo(yr[i]);
                        const float z = TIED ? h[i][e] - (e ? Two<E>::hi(xr[i]) : Two<E>::lo(xr[i])) : h[i][e];
                        gw[e] = d[e] * z * (GATE == RWKV_GATE_SIGMOID ? a[i][e] * rest[i][e] : a[i][e]);
                        gx[e] = TIED ? d[e] * rest[i][e] : d[e];
                        d[e] = DOC && (first >> i & 1) ? 0.f : d[e] * a[i][e];
                    }
                }
                store2<E, VEC>(dw.at(i), at.n, gw[0], gw[1]);
                store2<E, VEC>(dx.at(i), at.n, gx[0], gx[1]);
            }
        }
        if (CHAIN || at.tile == 0) break;
        at.go(at.tile - 1);
        load(at);
        __syncthreads();
    }
}

int check_grec(const rwkv_grec_args* p, bool backward) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if (p->dtype < 0 || p->dtype > RWKV_DTYPE_FP32 || p->gate < 0 || p->gate > RWKV_GATE_LOG || p->B <= 0 || p->T <= 0 || p->C <= 0 || p->B > 65535 || p->T > INT_MAX - 65536 || p->C > INT_MAX - 65536) return RWKV_ERR_SHAPE;
    if (p->w == nullptr || p->x == nullptr) return RWKV_ERR_NULL;
    if (backward ? p->dw == nullptr || p->dx == nullptr || p->saved == nullptr : p->y == nullptr || p->hT == nullptr) return RWKV_ERR_NULL;
    const uintptr_t eb = p->dtype == RWKV_DTYPE_FP32 ? 3 : 1;
    for (const void* q : {p->w, p->x, static_cast<const void*>(p->y), p->dy, static_cast<const void*>(p->dw), static_cast<const void*>(p->dx)})
        if (reinterpret_cast<uintptr_t>(q) & eb) return RWKV_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(p->h0), static_cast<const void*>(p->hT), static_cast<const void*>(p->dhT), static_cast<const void*>(p->dh0), static_cast<const void*>(p->doc)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    if (!aligned16(p->saved)) return RWKV_ERR_ALIGN;
    if (p->saved != nullptr && p->saved_bytes < rwkv_grec_saved_bytes(p->B, p->T, p->C)) return RWKV_ERR_WORKSPACE;
    if (rwkv_grec_workspace_bytes(p->B, p->T, p->C) > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < rwkv_grec_workspace_bytes(p->B, p->T, p->C)))
        return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

template <class E, int GATE, bool TIED> int grec_run(hipStream_t st, const rwkv_grec_args& p, const bool backward) {
    const int tiles = tiles_of(p.T), groups = groups_of(p.T);
    const int64_t columns = static_cast<int64_t>((p.C + 63) / 64) * p.B;
    const bool chain = chained(p.B, p.T, p.C);
    const int64_t blocks = chain ? columns * tiles : columns;
    if (blocks > INT_MAX) return RWKV_ERR_SHAPE;
    if (chain) {
        const int64_t n = static_cast<int64_t>(rwkv_grec_workspace_bytes(p.B, p.T, p.C) / 16);
        hipLaunchKernelGGL(grec_clear, dim3(static_cast<unsigned>(n < 1024 * 256 ? (n + 255) / 256 : 1024)), dim3(256), 0, st, static_cast<uint4*>(p.workspace), n);
    }
    // pairs of channels as one access, with offsets of 32 bits within a tile: everything on a boundary of two elements and no token further from the next than that
    const uintptr_t pair = 2 * sizeof(E) - 1;
    const auto close = [&](const int64_t st) { return st >= 0 && st < 1ll << 32 && (S * MAX_GROUPS * st + p.C) * static_cast<int64_t>(sizeof(E)) < 1ll << 32; };
    bool vec = p.C % 2 == 0 && p.w_sb % 2 == 0 && p.w_st % 2 == 0 && p.x_sb % 2 == 0 && p.x_st % 2 == 0 && close(p.w_st) && close(p.x_st) && close(p.C);
    for (const void* q : {p.w, p.x, static_cast<const void*>(p.y), p.dy, static_cast<const void*>(p.dw), static_cast<const void*>(p.dx)}) vec = vec && (reinterpret_cast<uintptr_t>(q) & pair) == 0;
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(32 * groups), 0, st, p, tiles); return launch_status(); };
    const auto pick = [&](auto doc, auto pairs) {
        constexpr bool D = decltype(doc)::value, V = decltype(pairs)::value;
        if (chain) return backward ? go(grec_bwd<E, GATE, TIED, D, V, true>) : go(grec_fwd<E, GATE, TIED, D, V, true>);
        return backward ? go(grec_bwd<E, GATE, TIED, D, V, false>) : go(grec_fwd<E, GATE, TIED, D, V, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (p.doc) return vec ? pick(yes{}, yes{}) : pick(yes{}, no{});
    return vec ? pick(no{}, yes{}) : pick(no{}, no{});
}
template <class E> int grec_type(hipStream_t st, const rwkv_grec_args& p, const bool backward) {
    if (p.gate == RWKV_GATE_SIGMOID) return p.tied ? grec_run<E, RWKV_GATE_SIGMOID, true>(st, p, backward) : grec_run<E, RWKV_GATE_SIGMOID, false>(st, p, backward);
    return p.tied ? grec_run<E, RWKV_GATE_LOG, true>(st, p, backward) : grec_run<E, RWKV_GATE_LOG, false>(st, p, backward);
}
int grec_any(void* stream, const rwkv_grec_args* p, bool backward) {
    if (const int rc = check_grec(p, backward)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (p->dtype) {
        case RWKV_DTYPE_BF16: return grec_type<bf16_t>(st, *p, backward);
        case RWKV_DTYPE_FP16: return grec_type<half_t>(st, *p, backward);
        default: return grec_type<float>(st, *p, backward);
    }
}

}  // namespace
}  // namespace rwkv

extern "C" {

// the states entering each tile
size_t rwkv_grec_saved_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0) return 0;
    return static_cast<size_t>(B) * rwkv::tiles_of(T) * C * sizeof(float);
}
// a ticket (64 bytes) of each column of 64 channels, and a map (8 bytes) and a state of each tile and channel
size_t rwkv_grec_workspace_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0 || !rwkv::chained(B, T, C)) return 0;
    return static_cast<size_t>(B) * ((C + 63) / 64) * (64 + static_cast<size_t>(rwkv::tiles_of(T)) * 64 * 12);
}
int rwkv_grec_forward(void* stream, const rwkv_grec_args* args) { return rwkv::grec_any(stream, args, false); }
int rwkv_grec_backward(void* stream, const rwkv_grec_args* args) { return rwkv::grec_any(stream, args, true); }

}  // extern "C"
