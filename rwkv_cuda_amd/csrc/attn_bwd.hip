// Attention backward on the matrix cores, without atomics: the weights are made again from the forward's lse, once by the workgroups that own
// queries (dQ: three products a pair) and once by those that own keys (dK, dV: four), each sum in one wave's registers in a fixed order.
//
// Seven products where one kernel for all three would do with five: that one would have to add dQ from many workgroups, in an order that changes (atomics)
// or through memory.  Bound by issue, as the forward.  bf16, causal: B2 T8192 H32 Hk8 N128 with a cap and prefixes dK dV 2.4 ms, dQ 1.9 ms; B8 T4096 H32 N64 with
// slopes 1.16 ms (950 TFLOP/s) and 0.88 ms (940).
#include "attn_tile.h"

namespace rwkv {
namespace {

// fp16 weights as operands are 2^SHIFT times as large: those of thousands of keys would fall below its normal numbers
template <class E> constexpr float SHIFT = std::is_same_v<E, bf16_t> ? 0.f : 8.f;
template <class E> constexpr float UNSHIFT = std::is_same_v<E, bf16_t> ? 1.f : 1.f / 256.f;

// The gradients of the scores as fp16 operands: with thousands of keys and gradients of y as training has them most would be below fp16's normal numbers, and large
// gradients of y would bring them above its largest.  |ds| is at most |dy| |v| + |delta|, lengths of rows: attn_delta leaves the largest |dy| and |delta| of a batch element,
// attn_dkv finds the largest |v| of its keys and leaves it for attn_dq, and the operands are taken times the power of two that brings that bound to 2^14 .. 2^15: none
// overflows, and down to 2^-29 of the bound they keep all their bits.  Padding and rows that are not finite do not count.  dQ of 128 queries on 16384 keys, dy of 1e-3, against 64
// bits: off by 2.1e-2 of its size without, 1.3e-3 so, which its own rounding is; the times are the same (B8 T4096 H32 N64 fp16 backward 2.27 ms and 2.26).
template <class E> constexpr bool LIFTED = !std::is_same_v<E, bf16_t>;
DEVINL float lift_of(const float bound) {
    const int e = 14 - (static_cast<int>(__float_as_uint(bound) >> 23) - 127);
    return __uint_as_float(static_cast<uint32_t>(min(max(e, -40), 100) + 127) << 23);
}
DEVINL float inverse_of(const float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }       // of a power of two
// the sum of squares of a lane's part of a row and its partner's
template <class E, int D> DEVINL float squares(const u32x4 (&x)[D / 16]) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(unpack_lo<E>(x[c][i]), unpack_lo<E>(x[c][i]), fmaf(unpack_hi<E>(x[c][i]), unpack_hi<E>(x[c][i]), s));
    return s + other_half(s);
}
DEVINL float wave_max(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
    return x;
}

// lo .. hi of the documents of each tile's real tokens, and whether all of them are real (4 us at T3001: a launch)
__global__ __launch_bounds__(256) void attn_ranges(const int* doc, const int T, const int first, const int tiles, Range* out) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, b = blockIdx.y;
    if (t >= tiles) return;
    const int64_t j = first + wide(t) * TILE + lane;
    const int d = j < T ? doc[wide(b) * T + j] : -1;
    int lo = d < 0 ? INT_MAX : d, hi = max(d, -1);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) lo = min(lo, __shfl_xor(lo, m, 64)), hi = max(hi, __shfl_xor(hi, m, 64));
    const bool whole = __ballot(d >= 0) == ~0ull;
    if (lane == 0) out[wide(b) * tiles + t] = {lo, hi, whole, 0};
}

// The blocks of 128 queries (workgroup 0) and of `kb` keys (workgroup 1) in the order of their work: tiles that hold tokens of the block's documents, as the kernels
// walk over them.  The order changes no result.  One workgroup counts, a wave a block, and ranks; at T3001 with five documents 4 us.
__global__ __launch_bounds__(1024) void attn_order(const rwkv_attn_args p, const Range* keys, const Range* queries, const int q_items, int* q_order, const int k_items, int* k_order, const int kb) {
    __shared__ int work[MAX_ORDER];
    const bool for_keys = q_items == 0 || blockIdx.x == 1;
    const int items = for_keys ? k_items : q_items, block = for_keys ? kb : 128, tk = static_cast<int>(tiles_of(p.Tk)), tq = static_cast<int>(tiles_of(p.Tq)), shift = p.Tk - p.Tq;
    const int blocks = items / p.B, lane = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < items; i += 16) {
        const int b = i / blocks, at = i % blocks * block, end = min(at + block, for_keys ? p.Tk : p.Tq);
        const int reach = reach_of(p, b);
        const Range* own = keys + wide(b) * tk;
        const Range* other = for_keys ? queries + wide(b) * tq : own;
        int lo = INT_MAX, hi = -1;
        for (int t = ((for_keys ? 0 : shift) + at) / TILE; t <= ((for_keys ? 0 : shift) + end - 1) / TILE; ++t) lo = min(lo, own[t].lo), hi = max(hi, own[t].hi);
        const int first = for_keys && p.causal && at >= reach ? max(0, at - shift) / TILE : 0;
        const int last = for_keys ? tq : (p.causal ? max(shift + end - 1, reach - 1) : p.Tk - 1) / TILE + 1;
        int n = 0;
        for (int t = first + lane; t < last; t += 64) n += other[t].lo <= hi && other[t].hi >= lo;
        n = static_cast<int>(group_sum<64>(static_cast<float>(n)));
        if (lane == 0) work[i] = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += 1024) {
        int rank = 0;
        for (int j = 0; j < items; ++j) rank += work[j] > work[i] || (work[j] == work[i] && j < i);
        (for_keys ? k_order : q_order)[rank] = i;
    }
}

// delta = sum over the channels of dy y, y as the forward had it before it was rounded; a row has D / 8 lanes.  fp16: and the largest |dy|^2 and |delta| of a workgroup's rows,
// of one batch element (blockIdx.y).  Bound by memory: B8 T4096 H32 N64 bf16 0.073 ms, 405 MB, 5.5 TB/s.
template <class E, int D> __global__ __launch_bounds__(256) void attn_delta(const rwkv_attn_args p, float* delta, float2* most) {
    constexpr int LANES = D / 8, ROWS = 256 / LANES;
    __shared__ float2 of_wave[4];
    const int b = blockIdx.y, d = threadIdx.x % LANES * 8;
    const int64_t rows = wide(p.Tq) * p.H, first = b * rows;
    float longest = 0.f, largest = 0.f;
    for (int64_t at = blockIdx.x * wide(ROWS); at < rows; at += gridDim.x * wide(ROWS)) {
        const int64_t row = at + threadIdx.x / LANES;
        float s = 0.f, n = 0.f;
        if (row < rows && d < p.N) {
            const int64_t o = (first + row) * p.N + d;
            const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.dy) + o), y = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.y) + o),
                        z = *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.y_rest) + o);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s = fmaf(unpack_lo<E>(a[i]), unpack_lo<E>(y[i]) + unpack_lo<E>(z[i]), s);
                s = fmaf(unpack_hi<E>(a[i]), unpack_hi<E>(y[i]) + unpack_hi<E>(z[i]), s);
                if constexpr (LIFTED<E>) n = fmaf(unpack_lo<E>(a[i]), unpack_lo<E>(a[i]), fmaf(unpack_hi<E>(a[i]), unpack_hi<E>(a[i]), n));
            }
        }
        s = group_sum<LANES>(s);
        if constexpr (LIFTED<E>) {
            n = group_sum<LANES>(n);
            if (row < rows && n < INFINITY && fabsf(s) < INFINITY && (p.doc == nullptr || p.doc[wide(b) * p.Tk + p.Tk - p.Tq + row / p.H] >= 0)) longest = fmaxf(longest, n), largest = fmaxf(largest, fabsf(s));
        }
        if (row < rows && d == 0) delta[(wide(b) * p.H + row % p.H) * p.Tq + row / p.H] = s;
    }
    if constexpr (LIFTED<E>) {
        longest = wave_max(longest), largest = wave_max(largest);
        if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = make_float2(longest, largest);
        __syncthreads();
        if (threadIdx.x == 0)
            most[wide(b) * gridDim.x + blockIdx.x] = make_float2(fmaxf(fmaxf(of_wave[0].x, of_wave[1].x), fmaxf(of_wave[2].x, of_wave[3].x)), fmaxf(fmaxf(of_wave[0].y, of_wave[1].y), fmaxf(of_wave[2].y, of_wave[3].y)));
    }
}

// dQ: 4 waves of 32 queries over the keys that any of them sees; S^T = K Q^T and dP^T = V dY^T, dQ^T += K^T dS^T
// Three waves a SIMD with heads of 64, for 1 to 8 spilled registers where there is a bias (B8 T4096 H32 N64 with slopes, forward + backward 3.135 -> 3.086 ms).  The halves of
// a tile interleaved: one after the other, with four waves, is slower (2.77 -> 2.85 ms; heads of 128, two waves, dQ 1.91 -> 2.11).
template <class E, int D, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_dq(const rwkv_attn_args p, const float* delta, const float* v_most, const int blocks_k, const Range* ranges, const int* order, const int blocks_q, const int per_xcd) {
    constexpr int QB = 128;
    constexpr int PLANES = 4 * Plane<D>::BYTES;
    constexpr int SLOPE_VALUS = 4 + (CAP ? 6 : 0) + (BIAS ? 2 : 0), SLOPE_TRANS = CAP ? 3 : 1;      // instructions of a pair
    __shared__ __align__(16) char smem[PLANES + (DOC ? 8 * TILE : 0)];      // two planes of keys and of values, and the documents of two tiles
    int* const key_doc = reinterpret_cast<int*>(smem + PLANES);
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((DOC && order ? static_cast<int>(blockIdx.x) : id) >= wide(blocks_q) * p.H * p.B) return;
    int b = id / blocks_q / p.H, h = id / blocks_q % p.H, q0 = (blocks_q - 1 - id % blocks_q) * QB;
    if (DOC && order) {
        const int item = order[blockIdx.x / p.H];
        b = item / blocks_q, h = dealt(blockIdx.x % p.H, p.H), q0 = item % blocks_q * QB;
    }
    const int hk = h / (p.H / p.Hk);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5;
    const lds_t lds = lds_of(smem);
    constexpr int BUF = 2 * Plane<D>::BYTES;

    const E* kbase = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh;
    const E* vbase = static_cast<const E*>(p.v) + b * p.v_sb + hk * p.v_sh;
    const int* doc = DOC ? p.doc + wide(b) * p.Tk : nullptr;
    const int shift = p.Tk - p.Tq, reach = reach_of(p, b) - 1;

    const int i = q0 + wave * 32 + (lane & 31);
    const bool real = i < p.Tq;
    const int64_t row = ((wide(b) * p.Tq + (real ? i : 0)) * p.H + h) * p.N;
    u32x4 q[D / 16], dy[D / 16];
    load_rows<E, D>(q, static_cast<const E*>(p.q) + b * p.q_sb + (real ? i : 0) * p.q_st + h * p.q_sh, real, p.N);
    load_rows<E, D>(dy, static_cast<const E*>(p.dy) + row, real, p.N);
    const int qdoc = DOC && real ? doc[shift + i] : 0;
    const int lim = !real || qdoc < 0 ? -1 : (p.causal ? max(shift + i, reach) : p.Tk - 1);
    const float pos = static_cast<float>(shift + i);
    const int64_t stat = (wide(b) * p.H + h) * p.Tq + (real ? i : 0);
    const float lse = lim >= 0 ? p.lse[stat] : INFINITY;
    float dlt = lim >= 0 ? delta[stat] : 0.f, lift = 1.f;       // fp16: of the lane's query; dlt times it
    if constexpr (LIFTED<E>) {
        float v = 0.f;
        for (int x = lane; x < blocks_k; x += 64) v = fmaxf(v, v_most[(wide(b) * p.Hk + hk) * blocks_k + x]);
        lift = lift_of(fmaf(__builtin_sqrtf(squares<E, D>(dy)), wave_max(v), fabsf(dlt)));
        dlt *= lift;
    }
    const int row_lo = q0 + __builtin_amdgcn_readfirstlane(wave) * 32;
    // the last key that all of the wave's queries see, and one that none behind sees
    const int lim_lo = __ballot(lim < 0) != 0ull ? -1 : (p.causal ? max(shift + row_lo, reach) : p.Tk - 1);
    const int lim_hi = row_lo >= p.Tq ? -1 : (p.causal ? max(shift + min(row_lo + 31, p.Tq - 1), reach) : p.Tk - 1);
    int dlo = 0, dhi = 0;                                        // the documents of the block's queries (and of what shares their tiles)
    if constexpr (DOC) {
        ranges += b * tiles_of(p.Tk);
        const int t0 = (shift + q0) / TILE, t1 = (shift + min(q0 + QB, p.Tq) - 1) / TILE;
        dlo = INT_MAX, dhi = -1;
        for (int x = t0; x <= t1; ++x) dlo = min(dlo, ranges[x].lo), dhi = max(dhi, ranges[x].hi);
    }
    const int last = p.causal ? max(min(q0 + QB, p.Tq) - 1 + shift, reach) : p.Tk - 1;
    const int tiles = last / TILE + 1;

    RowReader<D> rows(lane);
    ColReader<D> cols(lane);
    rows.move(lds);
    cols.move(lds);
    const Fetch<D, 4> fetch(tid, p.N);
    const Scorer sc(p, h);
    const float mul = CAP || BIAS ? 1.f : sc.unit;
    f32x16 g[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) g[d] = f32x16{};

    int next_doc = -1;
    const auto bring = [&](const int t, const int slot) {
        const int j0 = t * TILE, n = p.Tk - j0;
        fetch.template operator()<false>(lds + slot * BUF, kbase + j0 * p.k_st, n, static_cast<int>(p.k_st) * 2, p.N, 0);
        fetch.template operator()<false>(lds + slot * BUF + Plane<D>::BYTES, vbase + j0 * p.v_st, n, static_cast<int>(p.v_st) * 2, p.N, 0);
        if constexpr (DOC) next_doc = lane < n ? doc[j0 + lane] : -1;
    };
    // half e of a tile: scores and the gradients of the weights
    const auto products = [&](f32x16& s, f32x16& dp, const int e) {
        s = dp = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            s = mma<E>(rows(0, e, c), q[c], s);
            dp = mma<E>(rows(Plane<D>::BYTES, e, c), dy[c], dp);
        }
    };
    // the gradients of the scores, in s
    constexpr bool LINE = BIAS && !CAP;                          // the bias as slope (key - query), right where no key stands behind a query; `turn` makes it right elsewhere
    const bool two_sided = LINE && (p.prefix != nullptr || !p.causal);
    const auto slopes = [&](f32x16& s, const f32x16& dp, const int j) {
        const float dist = pos - static_cast<float>(j + 4 * hi), base = fmaf(-sc.slope, dist, -lse);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = s[r], sq = sc.squash<CAP>(x);
            const float t = LINE ? fmaf(x, sc.unit, fmaf(sc.slope, 8 * (r >> 2) + (r & 3), base)) : fmaf(sc.t<CAP, BIAS>(x, sq, dist - (8 * (r >> 2) + (r & 3))), mul, -lse);
            float ds = __builtin_amdgcn_exp2f(t) * (LIFTED<E> ? fmaf(dp[r], lift, -dlt) : dp[r] - dlt);
            if constexpr (CAP) ds *= 4.f * sq * (1.f - sq);
            s[r] = ds;
        }
    };
    const auto turn = [&](f32x16& s, const int j) {
        asm volatile("");                                        // (a branch: few tiles come here)
        const float over = static_cast<float>(j + 4 * hi) - pos, twice = 2.f * sc.slope / sc.unit;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(fmaxf(over + (8 * (r >> 2) + (r & 3)), 0.f), -twice, s[r]);
    };
    const auto mask = [&](f32x16& s, const int j0, const int e, const int slot) {
        asm volatile("");                                        // (a branch: few tiles come here)
        const int room = lim - j0 - 4 * hi - 32 * e;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            u32x4 kd;
            if constexpr (DOC) kd = *reinterpret_cast<const u32x4*>(key_doc + slot * TILE + 32 * e + 8 * n + 4 * hi);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                bool on = 8 * n + r <= room;
                if constexpr (DOC) on = on && static_cast<int>(kd[r]) == qdoc;
                s[4 * n + r] = on ? s[4 * n + r] : 0.f;
            }
        }
    };
    const auto add = [&](const u32x4 (&w)[2], const int e) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) g[d] = mma<E>(cols(0, 2 * e + c, d), w[c], g[d]);
    };
    Walk<DOC, false> walk(ranges, dlo, dhi, 0, tiles);
    if (walk.more()) bring(walk.t, 0);
    int par = 0, step = BUF;
    while (walk.more()) {
        const int j0 = walk.t * TILE;
        const bool part = !walk.whole;
        if (DOC && tid < TILE) key_doc[par * TILE + tid] = next_doc;
        arrived();
        __syncthreads();
        walk.next();
        if (walk.more()) bring(walk.t, par ^ 1);
        if (DOC && part) clear_padding<D>(lds + par * BUF, key_doc + par * TILE);
        if (j0 <= lim_hi) {
            const bool masked = part || j0 + TILE - 1 > lim_lo;
            f32x16 s0, s1, p0, p1;
            u32x4 w[2];
            const bool ahead = two_sided && j0 + TILE - 1 > shift + row_lo;
            products(s0, p0, 0);
            if (ahead) turn(s0, j0);
            __builtin_amdgcn_sched_barrier(0);
            products(s1, p1, 1);
            slopes(s0, p0, j0);
            beside<2 * D / 16, D / 8, SLOPE_VALUS * 16, SLOPE_TRANS * 16>();
            __builtin_amdgcn_sched_barrier(0);
            if (masked) mask(s0, j0, 0, par);
            if (ahead) turn(s1, j0 + 32);
            w[0] = as_operand<E>(s0, 0), w[1] = as_operand<E>(s0, 1);
            __builtin_amdgcn_sched_barrier(0);
            add(w, 0);
            slopes(s1, p1, j0 + 32);
            beside<D / 16, D / 8, SLOPE_VALUS * 16, SLOPE_TRANS * 16>();
            __builtin_amdgcn_sched_barrier(0);
            if (masked) mask(s1, j0, 1, par);
            w[0] = as_operand<E>(s1, 0), w[1] = as_operand<E>(s1, 1);
            add(w, 1);
        }
        rows.move(step);
        cols.move(step);
        step = -step;
        par ^= 1;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store32<E>(g[d], LIFTED<E> ? p.scale * inverse_of(lift) : p.scale, static_cast<E*>(p.dq) + row, nullptr, 32 * d, p.N, real);
}

// dK, dV: 4 waves of 32 keys over the queries, of all heads that share them, that see any of them; S = Q K^T and dP = dY V^T,
// dV^T += dY^T P, dK^T += Q^T dS
//
// With heads of 128 the two sums take half of a wave's 256 registers and the keys a quarter of the rest: the values are read from LDS.  There a workgroup has 8 waves
// (256 keys; two waves a SIMD), or 4 where there are few workgroups (B2 T8192 H32 N128: with the values in registers and 4 waves 4.4 ms, so 2.5).
//
// The two halves of a tile go through one after the other; what a wave does not overlap others do.  With heads of 64 that leaves room for a third wave on a SIMD, except with
// documents (8 to 22 registers spilled): B8 T4096 H32 N64 forward + backward, with the halves interleaved and two waves, and so: plain 2.96 / 2.81 ms, with slopes 3.08 / 2.97,
// with a cap 4.16 / 3.97; with documents the same to 2 percent.
template <class E, int D, int WAVES, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(64 * WAVES, D == 128 ? (WAVES == 4 ? 1 : 2) : DOC ? 2 : 3) void attn_dkv(const rwkv_attn_args p, const float* delta, const float2* most, const int delta_blocks, float* v_most, const Range* key_ranges, const Range* ranges, const int* order, const int blocks_k, const int per_xcd, const int parts, float* part) {
    constexpr int KB = 32 * WAVES, PLANES = 4 * Plane<D>::BYTES, VALUES = D == 128 ? KB / TILE * Plane<D>::BYTES : 0;
    // two planes of queries and of dY (below 64 KB: what M0 can name), lse, delta and documents of two tiles, the values of the block's keys, three lengths of each wave
    __shared__ __align__(16) char smem[PLANES + 6 * 4 * TILE + VALUES + (LIFTED<E> ? 3 * 4 * WAVES : 0)];
    float *const row_lse = reinterpret_cast<float*>(smem + PLANES), *const row_delta = row_lse + 2 * TILE;
    int* const row_doc = reinterpret_cast<int*>(row_delta + 2 * TILE);
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((DOC && order ? static_cast<int>(blockIdx.x) : id) >= wide(blocks_k) * parts * p.Hk * p.B) return;
    int b = id / (blocks_k * parts) / p.Hk, hk = id / (blocks_k * parts) % p.Hk, mine = id / blocks_k % parts, k0 = id % blocks_k * KB;
    if (DOC && order) {
        const int groups = p.Hk * parts, item = order[blockIdx.x / groups], c = dealt(blockIdx.x % groups, groups);
        b = item / blocks_k, hk = c / parts, mine = c % parts, k0 = item % blocks_k * KB;
    }
    const int G = p.H / p.Hk / parts;
    const int first_head = (hk * parts + mine) * G;              // of G that the block does
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5;
    const lds_t lds = lds_of(smem);
    constexpr int BUF = 2 * Plane<D>::BYTES;

    const int shift = p.Tk - p.Tq, reach = reach_of(p, b);
    const int* doc = DOC ? p.doc + wide(b) * p.Tk : nullptr;
    const int j = k0 + wave * 32 + (lane & 31);
    const bool real = j < p.Tk;
    const E *kbase = static_cast<const E*>(p.k) + b * p.k_sb + hk * p.k_sh, *vbase = static_cast<const E*>(p.v) + b * p.v_sb + hk * p.v_sh;
    u32x4 k[D / 16], v[D == 128 ? 1 : D / 16];
    load_rows<E, D>(k, kbase + (real ? j : 0) * p.k_st, real, p.N);
    if constexpr (D == 64) load_rows<E, D>(v, vbase + (real ? j : 0) * p.v_st, real, p.N);
    else
        for (int x = tid; x < KB * D / 8; x += 64 * WAVES) {
            const int r = x / (D / 8), c = x % (D / 8);
            u32x4 z = {0, 0, 0, 0};
            if (k0 + r < p.Tk && 8 * c < p.N) z = *reinterpret_cast<const u32x4*>(vbase + (k0 + r) * p.v_st + 8 * c);
            lds_st(lds + PLANES + 6 * 4 * TILE + r / TILE * Plane<D>::BYTES + Plane<D>::at(r % TILE, c), z);
        }
    const int kdoc = DOC && real ? doc[j] : 0;
    const int from = kdoc < 0 ? INT_MAX : (!p.causal || j < reach ? 0 : j);            // the first position that sees the key; none that sees padding
    const int key_lo = k0 + __builtin_amdgcn_readfirstlane(wave) * 32, key_hi = min(key_lo + 31, p.Tk - 1);
    // the first position that sees any of the wave's keys, and one from which on all see them
    const int from_lo = key_lo >= p.Tk ? INT_MAX : (!p.causal || key_lo < reach ? 0 : key_lo);
    const int from_hi = __ballot(kdoc < 0) != 0ull ? INT_MAX : (!p.causal || key_hi < reach ? 0 : key_hi);
    int dlo = 0, dhi = 0;                                        // the documents of the block's keys
    if constexpr (DOC) {
        key_ranges += b * tiles_of(p.Tk) + k0 / TILE;
        ranges += b * tiles_of(p.Tq);
        dlo = INT_MAX, dhi = -1;
        for (int x = 0; x < KB / TILE && k0 + x * TILE < p.Tk; ++x) dlo = min(dlo, key_ranges[x].lo), dhi = max(dhi, key_ranges[x].hi);
    }
    const int first = !p.causal || k0 < reach ? 0 : max(0, k0 - shift) / TILE, tiles = (p.Tq + TILE - 1) / TILE;

    RowReader<D> rows(lane);
    ColReader<D> cols(lane);
    rows.move(lds);
    cols.move(lds);
    const lds_t values = lds + PLANES + 6 * 4 * TILE + wave / 2 * Plane<D>::BYTES;
    const RowReader<D> vrows(lane);
    const Fetch<D, WAVES> fetch(tid, p.N);
    float lift = 1.f;                                            // fp16: of the block's keys
    if constexpr (LIFTED<E>) {
        float* const of_wave = reinterpret_cast<float*>(smem + PLANES + 6 * 4 * TILE + VALUES);
        u32x4 x[D / 16];
        if constexpr (D == 128) __syncthreads();
#pragma unroll
        for (int c = 0; c < D / 16; ++c) x[c] = D == 64 ? v[D == 64 ? c : 0] : vrows(values, wave & 1, c);
        float n = squares<E, D>(x), longest = 0.f, largest = 0.f;
        n = wave_max(real && kdoc >= 0 && n < INFINITY ? n : 0.f);
        for (int i = tid; i < delta_blocks; i += 64 * WAVES) {
            const float2 z = most[wide(b) * delta_blocks + i];
            longest = fmaxf(longest, z.x), largest = fmaxf(largest, z.y);
        }
        longest = wave_max(longest), largest = wave_max(largest);
        if (lane == 0) of_wave[3 * wave] = n, of_wave[3 * wave + 1] = longest, of_wave[3 * wave + 2] = largest;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) n = fmaxf(n, of_wave[3 * i]), longest = fmaxf(longest, of_wave[3 * i + 1]), largest = fmaxf(largest, of_wave[3 * i + 2]);
        n = __builtin_sqrtf(n);
        if (tid == 0 && mine == 0) v_most[(wide(b) * p.Hk + hk) * blocks_k + k0 / KB] = n;
        lift = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(lift_of(fmaf(__builtin_sqrtf(longest), n, largest)))));
    }
    // 2^-SHIFT lift: to the gradients of the scores, from 2^SHIFT times the weights (by the exponent, in a scalar register)
    const float down = __uint_as_float(__float_as_uint(lift) - (static_cast<uint32_t>(SHIFT<E>) << 23));
    f32x16 gk[D / 32], gv[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) gk[d] = gv[d] = f32x16{};

    int next_doc = -1;
    float next_lse = 0.f, next_delta = 0.f;
    const auto bring = [&](const int h, const int t, const int slot) {
        const int i0 = t * TILE, n = p.Tq - i0;
        fetch.template operator()<false>(lds + slot * BUF, static_cast<const E*>(p.q) + b * p.q_sb + i0 * p.q_st + h * p.q_sh, n, static_cast<int>(p.q_st) * 2, p.N, 0);
        fetch.template operator()<false>(lds + slot * BUF + Plane<D>::BYTES, static_cast<const E*>(p.dy) + ((wide(b) * p.Tq + i0) * p.H + h) * p.N, n, p.H * p.N * 2, p.N, 0);
        if (tid < TILE) {
            const bool on = tid < n;
            const int64_t stat = (wide(b) * p.H + h) * p.Tq + (on ? i0 + tid : 0);
            next_lse = p.lse[stat];
            next_delta = delta[stat];
            if constexpr (DOC) next_doc = on ? doc[shift + i0 + tid] : -1;
        }
    };
    constexpr bool LINE = BIAS && !CAP;                          // as in attn_dq
    const bool two_sided = LINE && (p.prefix != nullptr || !p.causal);
    const auto note = [&](const int t, const int slot, const float slope) {
        if (tid < TILE) {
            const bool off = t * TILE + tid >= p.Tq || next_lse == -INFINITY;            // a row that is not there or sees nothing: weights of 0
            row_lse[slot * TILE + tid] = off ? INFINITY : (LINE ? fmaf(slope, tid, next_lse) : next_lse) - SHIFT<E>;      // with the query's part of the bias
            row_delta[slot * TILE + tid] = off ? 0.f : next_delta * down;
            if (DOC) row_doc[slot * TILE + tid] = next_doc;
        }
    };
    const auto products = [&](f32x16& s, f32x16& dp, const int e) {
        s = dp = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            s = mma<E>(rows(0, e, c), k[c], s);
            if constexpr (D == 64) dp = mma<E>(rows(Plane<D>::BYTES, e, c), v[c], dp);
            else dp = mma<E>(rows(Plane<D>::BYTES, e, c), vrows(values, wave & 1, c), dp);
        }
    };
    // weights in s, gradients of the scores in dp
    const auto slopes = [&](const Scorer& sc, f32x16& s, f32x16& dp, const int i0, const int e, const int slot) {
        const float dist = static_cast<float>(shift + i0 + 4 * hi + 32 * e) - static_cast<float>(j), mul = CAP || BIAS ? 1.f : sc.unit;
        const float base = sc.slope * (static_cast<float>(j) - static_cast<float>(shift + i0));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int o = slot * TILE + 32 * e + 8 * n + 4 * hi;
            const float4 ls = *reinterpret_cast<const float4*>(row_lse + o), dl = *reinterpret_cast<const float4*>(row_delta + o);
            const float lse[4] = {ls.x, ls.y, ls.z, ls.w}, dlt[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = 4 * n + r;
                const float x = s[at], sq = sc.squash<CAP>(x);
                const float t = LINE ? fmaf(x, sc.unit, base - lse[r]) : fmaf(sc.t<CAP, BIAS>(x, sq, dist + (8 * n + r)), mul, -lse[r]);
                const float w = __builtin_amdgcn_exp2f(t);
                float ds = w * (SHIFT<E> == 0.f ? dp[at] - dlt[r] : fmaf(dp[at], down, -dlt[r]));
                if constexpr (CAP) ds *= 4.f * sq * (1.f - sq);
                s[at] = w;
                dp[at] = ds;
            }
        }
    };
    const auto turn = [&](const Scorer& sc, f32x16& s, const int i) {
        asm volatile("");                                        // (a branch: few tiles come here)
        const float over = static_cast<float>(j) - static_cast<float>(shift + i + 4 * hi), twice = 2.f * sc.slope / sc.unit;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(fmaxf(over - (8 * (r >> 2) + (r & 3)), 0.f), -twice, s[r]);
    };
    const auto mask = [&](f32x16& s, f32x16& dp, const int i0, const int e, const int slot) {
        asm volatile("");                                        // (a branch: few tiles come here)
        const int need = from - shift - i0 - 4 * hi - 32 * e;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            u32x4 rd;
            if constexpr (DOC) rd = *reinterpret_cast<const u32x4*>(row_doc + slot * TILE + 32 * e + 8 * n + 4 * hi);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                bool on = 8 * n + r >= need;
                if constexpr (DOC) on = on && static_cast<int>(rd[r]) == kdoc;
                s[4 * n + r] = on ? s[4 * n + r] : 0.f;
                dp[4 * n + r] = on ? dp[4 * n + r] : 0.f;
            }
        }
    };
    const auto add = [&](const u32x4 (&w)[2], const u32x4 (&ds)[2], const int e) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                gv[d] = mma<E>(cols(Plane<D>::BYTES, 2 * e + c, d), w[c], gv[d]);
                gk[d] = mma<E>(cols(0, 2 * e + c, d), ds[c], gk[d]);
            }
    };
    int h = first_head, par = 0, step = BUF;
    Walk<DOC, false> walk(ranges, dlo, dhi, first, tiles);
    const Walk<DOC, false> start = walk;
    if (walk.more()) bring(h, walk.t, 0);
    while (walk.more()) {
        const int i0 = walk.t * TILE;
        const bool part = !walk.whole;
        const Scorer sc(p, h);
        note(walk.t, par, sc.slope);
        arrived();
        __syncthreads();
        walk.next();
        if (!walk.more() && h + 1 < first_head + G) walk = start, ++h;
        if (walk.more()) bring(h, walk.t, par ^ 1);
        if (DOC && part) {
            clear_padding<D, WAVES>(lds + par * BUF, row_doc + par * TILE);
            clear_padding<D, WAVES>(lds + par * BUF + Plane<D>::BYTES, row_doc + par * TILE);
        }
        if (shift + i0 + TILE - 1 >= from_lo) {
            const bool masked = part || shift + i0 < from_hi;
            u32x4 w[2], ds[2];
            const bool ahead = two_sided && shift + i0 < k0 + KB - 1;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                f32x16 s, dp;
                products(s, dp, e);
                if (ahead) turn(sc, s, i0 + 32 * e);
                __builtin_amdgcn_sched_barrier(0);
                slopes(sc, s, dp, i0, e, par);
                if (masked) mask(s, dp, i0, e, par);
                w[0] = as_operand<E>(s, 0), w[1] = as_operand<E>(s, 1), ds[0] = as_operand<E>(dp, 0), ds[1] = as_operand<E>(dp, 1);
                __builtin_amdgcn_sched_barrier(0);
                add(w, ds, e);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        rows.move(step);
        cols.move(step);
        step = -step;
        par ^= 1;
    }
    const int64_t row = ((wide(b) * p.Tk + (real ? j : 0)) * p.Hk + hk) * p.N;
    const float back = LIFTED<E> ? inverse_of(lift) : 1.f;
    if (parts > 1) {
        const int64_t size = wide(p.B) * p.Tk * p.Hk * p.N;
        float* to = part + 2 * mine * size + row;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int c = 32 * d + 8 * n + 4 * hi;
                if (!real || c >= p.N) continue;
                *reinterpret_cast<float4*>(to + c) = make_float4(gk[d][4 * n] * back, gk[d][4 * n + 1] * back, gk[d][4 * n + 2] * back, gk[d][4 * n + 3] * back);
                *reinterpret_cast<float4*>(to + size + c) = make_float4(gv[d][4 * n], gv[d][4 * n + 1], gv[d][4 * n + 2], gv[d][4 * n + 3]);
            }
        return;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        store32<E>(gk[d], p.scale * back, static_cast<E*>(p.dk) + row, nullptr, 32 * d, p.N, real);
        store32<E>(gv[d], UNSHIFT<E>, static_cast<E*>(p.dv) + row, nullptr, 32 * d, p.N, real);
    }
}

// adds the groups of heads: eight values a thread, y = 0 for dK, 1 for dV
template <class E> __global__ __launch_bounds__(256) void attn_dkv_sum(const rwkv_attn_args p, const int parts, const float* part) {
    const int64_t size = wide(p.B) * p.Tk * p.Hk * p.N, at = (blockIdx.x * wide(256) + threadIdx.x) * 8;
    if (at >= size) return;
    float s[8] = {};
    for (int i = 0; i < parts; ++i) {
        const float4* x = reinterpret_cast<const float4*>(part + (2 * i + blockIdx.y) * size + at);
        const float4 a = x[0], b = x[1];
        s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w, s[4] += b.x, s[5] += b.y, s[6] += b.z, s[7] += b.w;
    }
    const float f = blockIdx.y ? UNSHIFT<E> : p.scale;
    *reinterpret_cast<u32x4*>(static_cast<E*>(blockIdx.y ? p.dv : p.dk) + at) =
        u32x4{pack2<E>(s[0] * f, s[1] * f), pack2<E>(s[2] * f, s[3] * f), pack2<E>(s[4] * f, s[5] * f), pack2<E>(s[6] * f, s[7] * f)};
}

template <class E, int D> int run(hipStream_t st, const rwkv_attn_args& p) {
    const AttnPlan plan = attn_plan(p.B, p.Tq, p.Tk, p.H, p.Hk, p.N, p.doc != nullptr);
    const int64_t row_blocks = LIFTED<E> ? plan.delta_blocks : (wide(p.Tq) * p.H * (D / 8) + 255) / 256;
    const bool eight = plan.eight;
    const int blocks_q = (p.Tq + 127) / 128, blocks_k = eight ? (p.Tk + 255) / 256 : (p.Tk + 127) / 128;
    const int64_t per_q = (wide(blocks_q) * p.H * p.B + 7) / 8, per_k = (wide(blocks_k) * plan.key_parts * p.Hk * p.B + 7) / 8;
    const int64_t sums = (wide(p.B) * p.Tk * p.Hk * p.N / 8 + 255) / 256;
    if (row_blocks > INT_MAX || per_q * 8 > INT_MAX || per_k * 8 > INT_MAX || (plan.key_parts > 1 && sums > INT_MAX)) return RWKV_ERR_SHAPE;
    // the documents of tiles of keys and of tiles of queries, the orders, delta, the largest lengths, the sums of groups of heads
    Range *key_ranges = static_cast<Range*>(p.workspace), *ranges = key_ranges + (p.doc ? p.B * tiles_of(p.Tk) : 0);
    char* at = reinterpret_cast<char*>(ranges + (p.doc ? p.B * tiles_of(p.Tq) : 0));
    int *q_order = plan.q_items > 0 ? reinterpret_cast<int*>(at) : nullptr, *k_order = plan.k_items > 0 ? reinterpret_cast<int*>(at + plan.q_order) : nullptr;
    float* delta = reinterpret_cast<float*>(at + plan.q_order + plan.k_order);
    float2* most = reinterpret_cast<float2*>(reinterpret_cast<char*>(delta) + plan.delta);
    float* v_most = reinterpret_cast<float*>(most + wide(p.B) * plan.delta_blocks);
    float* part = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + plan.backward) - (plan.key_parts > 1 ? 2 * plan.key_parts * wide(p.B) * p.Tk * p.Hk * p.N : 0);
    if (p.doc) {
        launch_attn_ranges(st, p.doc, p.B, p.Tk, 0, key_ranges);
        if (p.Tq == p.Tk) ranges = key_ranges;
        else launch_attn_ranges(st, p.doc, p.B, p.Tk, p.Tk - p.Tq, ranges);
        if (q_order || k_order) launch_attn_order(st, p, key_ranges, ranges, plan, q_order, k_order);
    }
    hipLaunchKernelGGL((attn_delta<E, D>), dim3(static_cast<unsigned>(row_blocks), p.B), dim3(256), 0, st, p, delta, most);
    const auto go = [&](auto dq, auto dkv) {
        hipLaunchKernelGGL(dkv, dim3(static_cast<unsigned>(per_k * 8)), dim3(eight ? 512 : 256), 0, st, p, delta, most, plan.delta_blocks, v_most, key_ranges, ranges, k_order, blocks_k, static_cast<int>(per_k), plan.key_parts, part);
        if (plan.key_parts > 1) hipLaunchKernelGGL((attn_dkv_sum<E>), dim3(static_cast<unsigned>(sums), 2), dim3(256), 0, st, p, plan.key_parts, part);
        hipLaunchKernelGGL(dq, dim3(static_cast<unsigned>(per_q * 8)), dim3(256), 0, st, p, delta, v_most, blocks_k, key_ranges, q_order, blocks_q, static_cast<int>(per_q));
        return launch_status();
    };
    const auto masks = [&](auto cap, auto bias) {
        constexpr bool C = decltype(cap)::value, S = decltype(bias)::value;
        constexpr int W = D == 128 ? 8 : 4;
        if (p.doc) return go(attn_dq<E, D, C, S, true>, eight ? attn_dkv<E, D, W, C, S, true> : attn_dkv<E, D, 4, C, S, true>);
        return go(attn_dq<E, D, C, S, false>, eight ? attn_dkv<E, D, W, C, S, false> : attn_dkv<E, D, 4, C, S, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (p.cap > 0.f) return p.slopes ? masks(yes{}, yes{}) : masks(yes{}, no{});
    return p.slopes ? masks(no{}, yes{}) : masks(no{}, no{});
}
template <class E> int run_any(hipStream_t st, const rwkv_attn_args& p) { return p.N <= 64 ? run<E, 64>(st, p) : run<E, 128>(st, p); }

}  // namespace

void launch_attn_ranges(hipStream_t st, const int* doc, int B, int T, int first, Range* out) {
    const int tiles = static_cast<int>(tiles_of(T - first));
    hipLaunchKernelGGL(attn_ranges, dim3((tiles + 3) / 4, B), dim3(256), 0, st, doc, T, first, tiles, out);
}

void launch_attn_order(hipStream_t st, const rwkv_attn_args& p, const Range* keys, const Range* queries, const AttnPlan& plan, int* q_order, int* k_order) {
    const int q = q_order ? plan.q_items : 0, k = k_order ? plan.k_items : 0;
    hipLaunchKernelGGL(attn_order, dim3((q > 0) + (k > 0)), dim3(1024), 0, st, p, keys, queries, q, q_order, k, k_order, plan.eight ? 256 : 128);
}

int launch_attn_bwd(hipStream_t st, const rwkv_attn_args& p) { return p.dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, p) : run_any<half_t>(st, p); }

}  // namespace rwkv
