// Attention forward on the matrix cores.  A workgroup has 4 waves of 32 queries of one head each and walks over the keys that any of
// them sees, 64 at a time: S^T = K Q^T, one pass of the softmax with the running maximum and sum of a lane's query, O^T += V^T P^T.
//
// Bound by issue: a half tile of 32 x 32 pairs takes the matrix unit 256 clocks with heads of 64 (512 with 128), its exponentials 128 and the
// other vector instructions 300 and more of each SIMD.  So products and weights of neighbouring halves stand side by side in one stretch of code
// (all_three), and tiles come to LDS past the registers.  128 queries a workgroup: 64 a wave spilled.  Two workgroups a CU with heads of 128, three or
// four with 64.  bf16, causal: B1 T8192 H32 N128 980 TFLOP/s (770 with a cap), B8 T4096 H32 N64 780, with slopes 740 (710 where
// y_rest is written for a backward); a library product of 8192^3 reaches 1266.
#include "attn_tile.h"

namespace rwkv {
namespace {

// The maximum that weights are taken relative to follows the running one only when that has grown by 2^GROWTH: sums and weights stay far from fp32's
// and fp16's ends, and the accumulators are rarely scaled.
constexpr float GROWTH = 8.f;
using yes = std::true_type;
using no = std::false_type;
constexpr int READS = 6;

// parts > 1: the block does one part of the keys, and leaves sums and maxima in `part` for attn_join.
template <class E, int D, bool CAP, bool BIAS, bool DOC>
__global__ __launch_bounds__(256, 2) void attn_fwd(const rwkv_attn_args p, const Range* ranges, const int* order, const int blocks_q, const int per_xcd, const int parts, float* part) {
    constexpr int QB = 128;
    // two planes of keys and of values (below 64 KB: what M0 can name), and the documents of two tiles
    constexpr int PLANES = 4 * Plane<D>::BYTES;
    __shared__ __align__(16) char smem[PLANES + (DOC ? 8 * TILE : 0)];
    int* const key_doc = reinterpret_cast<int*>(smem + PLANES);
    const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3), mine = id % parts;
    const int64_t all = wide(blocks_q) * parts * p.H * p.B;
    if ((DOC && order ? static_cast<int>(blockIdx.x) : id) >= all) return;
    int b = id / (blocks_q * parts) / p.H, h = id / (blocks_q * parts) % p.H, q0 = (blocks_q - 1 - id / parts % blocks_q) * QB;
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
    u32x4 q[D / 16];
    load_rows<E, D>(q, static_cast<const E*>(p.q) + b * p.q_sb + (real ? i : 0) * p.q_st + h * p.q_sh, real, p.N);
    const int qdoc = DOC && real ? doc[shift + i] : 0;
    const int lim = !real || qdoc < 0 ? -1 : (p.causal ? max(shift + i, reach) : p.Tk - 1);      // the last key that the query sees; padding sees none
    const float pos = static_cast<float>(shift + i);
    const int row_lo = q0 + __builtin_amdgcn_readfirstlane(wave) * 32, pos_lo = shift + row_lo;
    // the last key that all of the wave's queries see
    const int lim_lo = __ballot(lim < 0) != 0ull ? -1 : (p.causal ? max(pos_lo, reach) : p.Tk - 1);
    int dlo = 0, dhi = 0;                                        // the documents of the block's queries (and of what shares their tiles)
    if constexpr (DOC) {
        ranges += b * tiles_of(p.Tk);
        const int t0 = (shift + q0) / TILE, t1 = (shift + min(q0 + QB, p.Tq) - 1) / TILE;
        dlo = INT_MAX, dhi = -1;
        for (int x = t0; x <= t1; ++x) dlo = min(dlo, ranges[x].lo), dhi = max(dhi, ranges[x].hi);
    }
    // the last key that the block's last query sees
    const int last = p.causal ? max(min(q0 + QB, p.Tq) - 1 + shift, reach) : p.Tk - 1;
    const int all_tiles = last / TILE + 1, first_tile = static_cast<int>(wide(all_tiles) * mine / parts), tiles = static_cast<int>(wide(all_tiles) * (mine + 1) / parts);

    RowReader<D> krow(lane);
    ColReader<D> vcol(lane);
    krow.move(lds);
    vcol.move(lds + Plane<D>::BYTES);
    const Fetch<D, 4> fetch(tid, p.N);
    const Scorer sc(p, h);
    const float mul = CAP || BIAS ? 1.f : sc.unit;

    f32x16 o[D / 32], sa, sb;
    u32x4 pa[2], pb[2];
    float m = -INFINITY, l = 0.f, f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) o[d] = f32x16{};
    // the scores of half e (32 keys) of a tile
    const auto scores = [&](f32x16& s, const int e) {
        s = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) s = mma<E>(krow(0, e, c), q[c], s);
    };
    // Before the weights: capped (with its bias), and -inf where a query does not see a key.  A bias alone is made with the weights, as slope (key - query), which is
    // right where no key stands behind a query; elsewhere (`ahead`) the scores are made right here.
    constexpr bool LINE = BIAS && !CAP;
    const auto bound = [&](f32x16& s, const int j0, const int e, const int slot, const bool masked, const bool ahead) {
        const float dist = pos - static_cast<float>(j0 + 4 * hi + 32 * e);
        if constexpr (CAP) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = sc.t<CAP, BIAS>(s[r], sc.squash<CAP>(s[r]), dist - (8 * (r >> 2) + (r & 3)));
        }
        if (LINE && ahead) {
            asm volatile("");                                    // (a branch: few tiles come here)
            const float twice = 2.f * sc.slope / sc.unit;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fmaf(fmaxf((8 * (r >> 2) + (r & 3)) - dist, 0.f), -twice, s[r]);
        }
        if (masked) {
            asm volatile("");
            const int room = lim - j0 - 4 * hi - 32 * e;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                u32x4 kd;
                if constexpr (DOC) kd = *reinterpret_cast<const u32x4*>(key_doc + slot * TILE + 32 * e + 8 * g + 4 * hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool on = 8 * g + i <= room;
                    if constexpr (DOC) on = on && static_cast<int>(kd[i]) == qdoc;
                    s[4 * g + i] = on ? s[4 * g + i] : -INFINITY;
                }
            }
        }
    };
    // the weights of the 32 keys from j on; what was summed before counts f times
    const auto weights = [&](f32x16& s, const int j, u32x4 (&w)[2]) {
        const float far = LINE ? sc.slope * (static_cast<float>(j + 4 * hi) - pos) : 0.f;      // what a lane's keys share of the bias
        if constexpr (LINE) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc.unit, sc.slope * (8 * (r >> 2) + (r & 3)));
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top += far;
        top = fmaxf(top, other_half(top));
        const bool grown = (top - m) * mul > GROWTH;             // always at a query's first key, never while it has seen none (-inf and -inf)
        const float to = grown ? top : m;
        f = grown ? __builtin_amdgcn_exp2f((m - to) * mul) : 1.f;
        m = to;
        const float base = to == -INFINITY ? 0.f : far - to * mul;
        float sum = l * f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = __builtin_amdgcn_exp2f(CAP || BIAS ? s[r] + base : fmaf(s[r], mul, base));
            sum += x;
            s[r] = x;
        }
        l = sum;
        w[0] = as_operand<E>(s, 0);
        w[1] = as_operand<E>(s, 1);
        here(w[0]);
        here(w[1]);
        here(l);
        return __ballot(grown) != 0ull;
    };
    const auto add = [&](const u32x4 (&w)[2], const int e) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) o[d] = mma<E>(vcol(0, 2 * e + c, d), w[c], o[d]);
    };
    const auto rescale = [&]() {
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= f;
    };
    // scores of one half and values of another, in turn, and the weights of the one between them beside
    const auto all_three = [&](f32x16& ahead, f32x16& now, const int j, const u32x4 (&wold)[2], u32x4 (&wnow)[2], const int e) {
        __builtin_amdgcn_sched_barrier(0);
        ahead = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            ahead = mma<E>(krow(0, e, c), q[c], ahead);
            o[c % (D / 32)] = mma<E>(vcol(0, 2 * e + c / (D / 32), c % (D / 32)), wold[c / (D / 32)], o[c % (D / 32)]);
        }
        const bool grown = weights(now, j, wnow);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);  // LDS reads ahead of the products
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (BIAS && !CAP ? 88 : 72) * 8 / D, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 16 * 8 / D, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (grown) rescale();
    };

    // Tiles go through in halves of 32 keys, three halves at a time: while the weights of one are made, the matrix cores make the scores of the next and
    // add the values of the one before, in one stretch of code.  The keys of a tile are therefore in LDS one tile before its values.
    int next_doc = -1;
    const auto fetch_keys = [&](const int t, const int slot) {
        const int j0 = t * TILE, rows = p.Tk - j0;
        fetch.template operator()<false>(lds + slot * BUF, kbase + j0 * p.k_st, rows, static_cast<int>(p.k_st) * 2, p.N, 0);
        if constexpr (DOC) next_doc = lane < rows ? doc[j0 + lane] : -1;
    };
    // (the values of padding may be anything: zeros instead)
    const auto fetch_values = [&](const int t, const int slot, const uint64_t real) {
        fetch.template operator()<DOC>(lds + slot * BUF + Plane<D>::BYTES, vbase + t * TILE * p.v_st, p.Tk - t * TILE, static_cast<int>(p.v_st) * 2, p.N, real);
    };
    // From the last key back: a bias falls from there, so that the maximum is found at once (B8 T4096 H32 N64 with slopes from 1/2: 1.00 ms forward in order).
    Walk<DOC, true> walk(ranges, dlo, dhi, first_tile, tiles);
    if (walk.more()) {
        int t = walk.t;
        bool whole = walk.whole;
        fetch_keys(t, 0);
        if (DOC && tid < TILE) key_doc[tid] = next_doc;
        const uint64_t there = DOC ? __ballot(next_doc >= 0) : 0;
        arrived();
        __syncthreads();
        fetch_values(t, 0, there);
        walk.next();
        if (walk.more()) fetch_keys(walk.t, 1);
        const auto is_masked = [&]() { return !whole || t * TILE + TILE - 1 > lim_lo; };
        const bool two_sided = LINE && (p.prefix != nullptr || !p.causal);
        const auto is_ahead = [&]() { return two_sided && t * TILE + TILE - 1 > pos_lo; };
        scores(sa, 0);
        scores(sb, 1);
        bound(sa, t * TILE, 0, 0, is_masked(), is_ahead());
        bound(sb, t * TILE, 1, 0, is_masked(), is_ahead());
        if (weights(sa, t * TILE, pa)) rescale();
        int par = 0, step = BUF;
        const auto meet = [&]() {                                // what is under way has come, for all waves
            if (DOC && walk.more() && tid < TILE) key_doc[(par ^ 1) * TILE + tid] = next_doc;
            arrived();
            __syncthreads();
        };
        meet();
        while (walk.more()) {
            const int j_old = t * TILE + 32;
            t = walk.t;
            whole = walk.whole;
            walk.next();
            fetch_values(t, par ^ 1, DOC ? __ballot(next_doc >= 0) : 0);
            if (walk.more()) fetch_keys(walk.t, par);
            krow.move(step);
            const bool masked = is_masked(), ahead = is_ahead();
            all_three(sa, sb, j_old, pa, pb, 0);
            bound(sa, t * TILE, 0, par ^ 1, masked, ahead);
            all_three(sb, sa, t * TILE, pb, pa, 1);
            bound(sb, t * TILE, 1, par ^ 1, masked, ahead);
            vcol.move(step);
            par ^= 1;
            step = -step;
            meet();
        }
        add(pa, 0);
        if (weights(sb, t * TILE + 32, pb)) rescale();
        add(pb, 1);
    }

    const float sum = l + other_half(l), inv = sum == 0.f ? 0.f : 1.f / sum;
    if (parts > 1) {
        if (!real) return;
        float* to = part + (((wide(b) * p.H + h) * p.Tq + i) * parts + mine) * (D + 4);
        if (hi == 0) to[0] = m * mul, to[1] = sum;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) *reinterpret_cast<float4*>(to + 4 + 32 * d + 8 * g + 4 * hi) = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
        return;
    }
    const int64_t at = ((wide(b) * p.Tq + (real ? i : 0)) * p.H + h) * p.N;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store32<E>(o[d], inv, static_cast<E*>(p.y) + at, p.y_rest ? static_cast<E*>(p.y_rest) + at : nullptr, 32 * d, p.N, real);
    if (p.lse && real && hi == 0) p.lse[(wide(b) * p.H + h) * p.Tq + i] = sum == 0.f ? -INFINITY : fmaf(m, mul, __builtin_amdgcn_logf(sum));
}

// joins the parts of a query: D / 4 lanes, four channels each
template <class E, int D> __global__ __launch_bounds__(256) void attn_join(const rwkv_attn_args p, const int parts, const float* part) {
    constexpr int LANES = D / 4;
    const int64_t row = blockIdx.x * wide(256 / LANES) + threadIdx.x / LANES;       // of [B,H,Tq]
    const int c = threadIdx.x % LANES * 4;
    if (row >= wide(p.B) * p.H * p.Tq || c >= p.N) return;
    const float* from = part + row * parts * (D + 4);
    float top = -INFINITY;
    for (int i = 0; i < parts; ++i) top = fmaxf(top, from[i * (D + 4)]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < parts; ++i) {
        const float* x = from + i * (D + 4);
        const float f = __builtin_amdgcn_exp2f(x[0] - base);
        const float4 o = *reinterpret_cast<const float4*>(x + 4 + c);
        sum = fmaf(x[1], f, sum);
        y[0] = fmaf(o.x, f, y[0]), y[1] = fmaf(o.y, f, y[1]), y[2] = fmaf(o.z, f, y[2]), y[3] = fmaf(o.w, f, y[3]);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const int i = row % p.Tq, h = row / p.Tq % p.H;
    const int64_t at = ((row / p.Tq / p.H * p.Tq + i) * p.H + h) * p.N + c;
    const u32x2 w = {pack2<E>(y[0] * f, y[1] * f), pack2<E>(y[2] * f, y[3] * f)};
    *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + at) = w;
    if (p.y_rest)
        *reinterpret_cast<u32x2*>(static_cast<E*>(p.y_rest) + at) = u32x2{pack2<E>(y[0] * f - unpack_lo<E>(w[0]), y[1] * f - unpack_hi<E>(w[0])), pack2<E>(y[2] * f - unpack_lo<E>(w[1]), y[3] * f - unpack_hi<E>(w[1]))};
    if (p.lse && c == 0) p.lse[row] = sum == 0.f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
}

template <class E, int D> int run(hipStream_t st, const rwkv_attn_args& p) {
    const int blocks_q = (p.Tq + 127) / 128;
    const AttnPlan plan = attn_plan(p.B, p.Tq, p.Tk, p.H, p.Hk, p.N, p.doc != nullptr);
    const int64_t all = wide(blocks_q) * plan.query_parts * p.H * p.B, per = (all + 7) / 8, join = (wide(p.B) * p.H * p.Tq * (D / 4) + 255) / 256;
    if (per * 8 > INT_MAX || (plan.query_parts > 1 && join > INT_MAX)) return RWKV_ERR_SHAPE;
    int* order = plan.q_items > 0 ? reinterpret_cast<int*>(static_cast<char*>(p.workspace) + plan.ranges) : nullptr;
    float* part = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + plan.ranges + plan.q_order);
    const dim3 grid(static_cast<unsigned>(per * 8)), block(256);
    Range* ranges = static_cast<Range*>(p.workspace);
    if (p.doc) launch_attn_ranges(st, p.doc, p.B, p.Tk, 0, ranges);
    if (order) launch_attn_order(st, p, ranges, ranges, plan, order, nullptr);
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, block, 0, st, p, ranges, order, blocks_q, static_cast<int>(per), plan.query_parts, part);
        if (plan.query_parts > 1) hipLaunchKernelGGL((attn_join<E, D>), dim3(static_cast<unsigned>(join)), block, 0, st, p, plan.query_parts, part);
        return launch_status();
    };
    const auto masks = [&](auto cap, auto bias) {
        return p.doc ? go(attn_fwd<E, D, decltype(cap)::value, decltype(bias)::value, true>) : go(attn_fwd<E, D, decltype(cap)::value, decltype(bias)::value, false>);
    };
    if (p.cap > 0.f) return p.slopes ? masks(yes{}, yes{}) : masks(yes{}, no{});
    return p.slopes ? masks(no{}, yes{}) : masks(no{}, no{});
}
template <class E> int run_any(hipStream_t st, const rwkv_attn_args& p) {
    return p.N <= 64 ? run<E, 64>(st, p) : run<E, 128>(st, p);
}

}  // namespace

int launch_attn_fwd(hipStream_t st, const rwkv_attn_args& p) { return p.dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, p) : run_any<half_t>(st, p); }

}  // namespace rwkv
