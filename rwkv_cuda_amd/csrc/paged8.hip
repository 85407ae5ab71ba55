// Attention of one new token a sequence over a paged cache in 8 bits (the arguments are explained in rwkv_hip.h).
//
// As paged.hip, with half the bytes: the codes of e4m3 are numbers of bf16 and of fp16 as they stand, so they are widened in registers (two a v_cvt_scalef32_pk) and
// multiplied on v_mfma_f32_16x16x32.  A key's scale multiplies its score.  A value's scale goes into the weight's exponent, w_j = 2^(s_j + log2 scale_j - m) with m the running
// maximum of that sum, so that weights stay within 1 in 16 bits whatever the scales, and O = sum w_j code_j.  The sum of the softmax is the sum of 2^(s_j - r), in 32 bits, with an r of its own: scales may lie 2^220 apart,
// and w_j / scale_j would be nothing where a page of zeros stands beside large ones.  Y = O 2^(m - r) / sum.  (What a small scale's values lose to 16-bit weights, 2^-24 of the largest in fp16, is less than the
// large scale's own codes round off.)
// A lane reads 16 codes of a key at once: of every 64 channels a group of 16 lanes has 16 neighbouring ones, eight for either of two products, and so has the query.
// Bound by memory where there is work: B64, up to 4096 tokens, H32 Hk32 N64 bf16, 554 MB in 125 to 130 us; B4, up to 131072, H64 Hk8 N128 fp16, 752 MB in 150 to 160 us.
#include "paged_tile.h"

namespace rwkv {
namespace {

DEVINL u32x4 join(const u32x2 a, const u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }
template <int HOW> DEVINL float other_lane(const float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), HOW, 0xf, 0xf, true)); }
// over 16 lanes: rotations by 8, 4, 2 and 1
DEVINL float row_max(float x) {
    x = fmaxf(x, other_lane<0x128>(x)), x = fmaxf(x, other_lane<0x124>(x)), x = fmaxf(x, other_lane<0x122>(x));
    return fmaxf(x, other_lane<0x121>(x));
}
DEVINL float row_add(float x) {
    x += other_lane<0x128>(x), x += other_lane<0x124>(x), x += other_lane<0x122>(x);
    return x + other_lane<0x121>(x);
}
// codes 4 x .. 4 x + 3 of a register as two registers of E
template <class E> DEVINL u32x2 widen(const uint32_t x) {
    if constexpr (std::is_same_v<E, bf16_t>)
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true))};
    else
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true))};
}
template <class E> DEVINL u32x4 widen8(const uint32_t x, const uint32_t y) {
    const u32x2 a = widen<E>(x), b = widen<E>(y);
    return u32x4{a[0], a[1], b[0], b[1]};
}

// A sum of 2^(s - ref) whose ref follows the largest s: far behind, as long as 32 bits hold it (2^31 terms of 2^FAR).
constexpr float FAR = 64.f;
DEVINL void raise(float& ref, float& sum, const float most) {
    const float to = fmaxf(ref, most);
    sum = to == -INFINITY ? 0.f : sum * __builtin_amdgcn_exp2f(ref - to);
    ref = to;
}

template <class E, int D, int W>
__global__ __launch_bounds__(64 * W, 2) void paged8_attn(const rwkv_paged8_args p, const int shift, const int pieces, const int chunks, const int group, const int shares, float* part) {
    constexpr int ROWS = 64 / (D / 16), VSTEPS = STEP / ROWS;       // rows of an access of a wave, accesses of 32 rows
    __shared__ __align__(16) char smem[W * STEP * 2 * D];
    __shared__ __align__(16) float scale_of_key[W][STEP], log_of_value[W][STEP];
    __shared__ float top_of[W][HEADS], sum_of[W][HEADS], ref_of[W][HEADS];
    // `group` neighbouring heads (with their chunks) are a share, and an XCD has whole shares; 0: the pieces of a head one after the other
    const int slot = group > 1 ? blockIdx.x >> 3 : blockIdx.x, share = group > 1 ? slot / group * 8 + (blockIdx.x & 7) : slot;
    if (share >= shares) return;
    const int heads = p.Hk * chunks, of_piece = heads / max(group, 1);
    const int y = group == 0 ? share / pieces % heads : share % of_piece * group + slot % group, piece = group == 0 ? share % pieces : share / of_piece % pieces;
    const int b = share / of_piece / pieces, hk = y / chunks, chunk = y % chunks, G = p.H / p.Hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    const int all = p.lens[b], n = tokens_of(p, b, shift), size = piece_of(n, pieces);
    const int64_t begin = wide(piece) * size;
    const int end = static_cast<int>(min(begin + size, wide(n)));
    const bool alone = pieces == 1;
    if (begin >= n && !alone) return;
    const int head = chunk * HEADS + col, h = hk * G + min(head, G - 1);
    const bool mine = head < G;
    const int* table = p.table + wide(b) * p.M;
    const uint8_t *kpages = static_cast<const uint8_t*>(p.k_pages) + hk * p.k_sh, *vpages = static_cast<const uint8_t*>(p.v_pages) + hk * p.v_sh;

    u32x4 q[D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        const int d = 64 * (s / 2) + 16 * grp + 8 * (s % 2);
        q[s] = mine && d < p.N ? *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.q) + (wide(b) * p.H + h) * p.N + d) : u32x4{0, 0, 0, 0};
    }
    const float unit = p.scale * LOG2E, in = p.cap > 0.f ? 2.f * unit / p.cap : 0.f, out = p.cap * LOG2E, slope = p.slopes ? p.slopes[h] * LOG2E : 0.f;
    const lds_t plane = lds_of(smem) + wave * STEP * 2 * D;
    lds_t vread[2];
    vread[0] = value_at<D>(4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);
    vread[1] = value_at<D>(16 + 4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);

    u32x4 kr[2][D / 64], vr[VSTEPS];
    float kscale, vscale;                                            // of token lane & 31
    bool on_of;
    const auto load = [&](const int j0) {
        const int own = j0 + (lane & 31);
        int page = own < end ? table[own >> shift] : -1;
        on_of = page >= 0 && page < p.P;
        page = on_of ? page : -1;
        kscale = on_of ? p.k_scales[wide(page) * p.Hk + hk] : 1.f;
        vscale = on_of ? p.v_scales[wide(page) * p.Hk + hk] : 1.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = j0 + 16 * e + col, pg = __shfl(page, 16 * e + col, 64);
            const uint8_t* row = kpages + pg * p.k_sp + (j & (p.page - 1)) * p.k_st;
#pragma unroll
            for (int s = 0; s < D / 64; ++s) {
                const int d = 64 * s + 16 * grp;
                kr[e][s] = pg >= 0 && d < p.N ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) {
            const int r = i * ROWS + lane / (D / 16), d = 16 * (lane % (D / 16)), j = j0 + r, pg = __shfl(page, r, 64);
            const uint8_t* row = vpages + pg * p.v_sp + (j & (p.page - 1)) * p.v_st;
            vr[i] = pg >= 0 && d < p.N ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
        }
    };

    f32x4_t o[D / 16];
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{};
    float m = -INFINITY, ref = -INFINITY, l = 0.f;                   // (ref and l are a lane's own)
    int j0 = static_cast<int>(begin) + wave * STEP;
    if (j0 < end) load(j0);
    for (; j0 < end; j0 += W * STEP) {
        f32x4_t s[2] = {f32x4_t{}, f32x4_t{}};
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                s[e] = mma16<E>(widen8<E>(kr[e][c][0], kr[e][c][1]), q[2 * c], s[e]);
                s[e] = mma16<E>(widen8<E>(kr[e][c][2], kr[e][c][3]), q[2 * c + 1], s[e]);
            }
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) {
            const int r = i * ROWS + lane / (D / 16), c = 2 * (lane % (D / 16));
            lds_st(plane + value_at<D>(r, c), widen8<E>(vr[i][0], vr[i][1]));
            lds_st(plane + value_at<D>(r, c + 1), widen8<E>(vr[i][2], vr[i][3]));
        }
        if (lane < 32) {
            scale_of_key[wave][lane] = kscale;
            log_of_value[wave][lane] = __builtin_amdgcn_logf(vscale);
        }
        const uint32_t on = static_cast<uint32_t>(__ballot(on_of));  // which of the 32 tokens count (twice)
        const int now = j0;
        if (j0 + W * STEP < end) load(j0 + W * STEP);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // the wave's own writes above
        float top = -INFINITY, most = -INFINITY, x[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const f32x4_t ks = *reinterpret_cast<const f32x4_t*>(&scale_of_key[wave][16 * e + 4 * grp]), lv = *reinterpret_cast<const f32x4_t*>(&log_of_value[wave][16 * e + 4 * grp]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * e + 4 * grp + r;
                const float dot = s[e][r] * ks[r];
                float y = dot * unit;
                if (p.cap > 0.f) y = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(dot * in)), -2.f * out, out);
                y = fmaf(static_cast<float>(all - 1 - now - t), -slope, y);
                x[e][r] = on >> t & 1 ? y : -INFINITY;
                s[e][r] = x[e][r] + lv[r];
                most = fmaxf(most, x[e][r]);
                top = fmaxf(top, s[e][r]);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__ballot(top > m) != 0ull) {
            const float to = fmaxf(top, m), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
            m = to;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][r] *= f;
        }
        if (__ballot(most > ref + FAR) != 0ull) raise(ref, l, most);
        const float base = m == -INFINITY ? 0.f : m, low = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[e][r] = __builtin_amdgcn_exp2f(s[e][r] - base);
                l += __builtin_amdgcn_exp2f(x[e][r] - low);
            }
        const u32x4 w = {pack2<E>(s[0][0], s[0][1]), pack2<E>(s[0][2], s[0][3]), pack2<E>(s[1][0], s[1][1]), pack2<E>(s[1][2], s[1][3])};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            typedef v4s __attribute__((address_space(3))) * ptr;
            const lds_t x = 32 * d;                                  // two pieces on: the swaps leave the lowest bit and are taken against it
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(plane + (vread[0] ^ x))), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(plane + (vread[1] ^ x)));
            const u32x2 y = __builtin_bit_cast(u32x2, lo), z = __builtin_bit_cast(u32x2, hi);
            o[d] = mma16<E>(u32x4{y[0], y[1], z[0], z[1]}, w, o[d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    raise(ref, l, fmaxf(__shfl_xor(ref, 16, 64), ref));
    raise(ref, l, fmaxf(__shfl_xor(ref, 32, 64), ref));
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);                    // [wave][head][D], pieces of four channels of a head turned by the head
    if (grp == 0) top_of[wave][col] = m, sum_of[wave][col] = l, ref_of[wave][col] = ref;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4_t*>(sums + (wave * HEADS + col) * D + 4 * ((4 * d + grp) ^ col)) = o[d];
    __syncthreads();
    for (int i = tid; i < HEADS * D / 4; i += 64 * W) {
        const int x = i / (D / 4), c = i % (D / 4), hd = chunk * HEADS + x;
        if (hd >= G || 4 * c >= p.N) continue;
        float top = -INFINITY, ref = -INFINITY;
#pragma unroll
        for (int k = 0; k < W; ++k) top = fmaxf(top, top_of[k][x]), ref = fmaxf(ref, ref_of[k][x]);
        const float base = top == -INFINITY ? 0.f : top, low = ref == -INFINITY ? 0.f : ref;
        float sum = 0.f;
        f32x4_t y = f32x4_t{};
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = __builtin_amdgcn_exp2f(top_of[k][x] - base);
            sum = fmaf(sum_of[k][x], __builtin_amdgcn_exp2f(ref_of[k][x] - low), sum);
            y += *reinterpret_cast<const f32x4_t*>(sums + (k * HEADS + x) * D + 4 * (c ^ x)) * f;
        }
        const int64_t row = wide(b) * p.H + hk * G + hd;
        if (alone) {
            const float f = sum == 0.f ? 0.f : 1.f / sum, g = __builtin_amdgcn_exp2f(0.5f * (base - low));     // (twice: up to 2^(120 + FAR))
            *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + row * p.N + 4 * c) = u32x2{pack2<E>(y[0] * f * g * g, y[1] * f * g * g), pack2<E>(y[2] * f * g * g, y[3] * f * g * g)};
        } else {
            float* to = part + (row * pieces + piece) * (D + 4);
            *reinterpret_cast<f32x4_t*>(to + 4 + 4 * c) = y;
            if (c == 0) to[0] = top, to[1] = sum, to[2] = ref;
        }
    }
}

// The same for at most 8 query heads of a key head, 64 tokens a step.  There a product of 16 keys and 16 heads would have empty columns, and the softmax, which costs most of the instructions, would
// run over them; so the heads' side of the product has the heads once for each of TILES tiles of 16 tokens, in rows of their own, zero elsewhere, and TILES products add up to scores that fill the
// lanes: 4 tiles of one or two heads (a lane has a token, and R heads), or 2 tiles of up to 8 (R = 4).  A lane has its own token's scales.  The weights go to the other product through LDS, 128 bytes a head.
template <class E, int D, int TILES, int R, int W>
__global__ __launch_bounds__(64 * W, 2) void paged8_few(const rwkv_paged8_args p, const int shift, const int pieces, const int group, const int shares, float* part) {
    constexpr int PER = 16 / TILES, SETS = 4 / TILES, TOKENS = 64, ROWS = 64 / (D / 16), VSTEPS = TOKENS / ROWS, WPITCH = 2 * TOKENS + 16;
    __shared__ __align__(16) char smem[W * STEP * 2 * D];
    __shared__ __align__(16) char weights[W][PER * WPITCH];
    __shared__ float top_of[W][PER], sum_of[W][PER], ref_of[W][PER];
    const int slot = group > 1 ? blockIdx.x >> 3 : blockIdx.x, share = group > 1 ? slot / group * 8 + (blockIdx.x & 7) : slot;
    if (share >= shares) return;
    const int of_piece = p.Hk / max(group, 1);
    const int hk = group == 0 ? share / pieces % p.Hk : share % of_piece * group + slot % group, piece = group == 0 ? share % pieces : share / of_piece % pieces;
    const int b = share / of_piece / pieces, G = p.H / p.Hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
    const int all = p.lens[b], n = tokens_of(p, b, shift), size = piece_of(n, pieces);
    const int64_t begin = wide(piece) * size;
    const int end = static_cast<int>(min(begin + size, wide(n)));
    const bool alone = pieces == 1;
    if (begin >= n && !alone) return;
    const int* table = p.table + wide(b) * p.M;
    const uint8_t *kpages = static_cast<const uint8_t*>(p.k_pages) + hk * p.k_sh, *vpages = static_cast<const uint8_t*>(p.v_pages) + hk * p.v_sh;
    const float *kscales = p.k_scales + hk, *vscales = p.v_scales + hk;

    u32x4 q[TILES][D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        const int d = 64 * (s / 2) + 16 * grp + 8 * (s % 2), head = col % PER;
        const u32x4 x = head < G && d < p.N ? *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.q) + (wide(b) * p.H + hk * G + head) * p.N + d) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < TILES; ++t) q[t][s] = x & (col / PER == t ? ~0u : 0u);
    }
    const float unit = p.scale * LOG2E, in = p.cap > 0.f ? 2.f * unit / p.cap : 0.f, out = p.cap * LOG2E;
    float slope[R];
#pragma unroll
    for (int r = 0; r < R; ++r) slope[r] = p.slopes ? p.slopes[hk * G + min((4 * grp + r) % PER, G - 1)] * LOG2E : 0.f;
    const lds_t plane = lds_of(smem) + wave * STEP * 2 * D, weight = lds_of(weights[wave]);
    lds_t vread[2];
    vread[0] = value_at<D>(4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);
    vread[1] = value_at<D>(16 + 4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);
    const lds_t wread = weight + min(col % PER, (R - 1) | (PER - 4)) * WPITCH + 8 * grp;

    const int own = 16 * (grp * TILES / 4) + col;                    // a lane's token, of each set of 16 TILES
    const int kd = 16 * grp, vd = 16 * (lane % (D / 16));
    u32x4 kr[4][D / 64], vr[VSTEPS];
    float kscale[SETS], vscale[SETS];
    bool on[SETS];
    int page[SETS], ahead[SETS];                                     // ahead: of the step after the next, so that nothing waits for a page's number
    const auto load_pages = [&](const int j0) {
#pragma unroll
        for (int a = 0; a < SETS; ++a) ahead[a] = table[min(j0 + 16 * TILES * a + own, end - 1) >> shift];
    };
    const auto page_of = [&](const int tile, const int row) { return static_cast<uint32_t>(__shfl(page[tile / TILES], 64 / TILES * (tile % TILES) + row, 64)); };
    const auto load_keys = [&](const int j0) {
#pragma unroll
        for (int a = 0; a < SETS; ++a) {
            on[a] = j0 + 16 * TILES * a + own < end && static_cast<unsigned>(ahead[a]) < static_cast<unsigned>(p.P);
            page[a] = on[a] ? ahead[a] : 0;                          // (a page that there is; what is read of it does not count)
            const float k = kscales[wide(page[a]) * p.Hk], v = vscales[wide(page[a]) * p.Hk];
            kscale[a] = k, vscale[a] = on[a] ? v : 1.f;
        }
        if (j0 + W * TOKENS < end) load_pages(j0 + W * TOKENS);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t* row = kpages + page_of(t, col) * p.k_sp + ((j0 + 16 * t + col) & (p.page - 1)) * p.k_st;
#pragma unroll
            for (int s = 0; s < D / 64; ++s) kr[t][s] = *reinterpret_cast<const u32x4*>(row + (64 * s + kd < p.N ? 64 * s + kd : 0));
        }
    };
    const auto load_values = [&](const int j0) {
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) {
            const int r = i * ROWS + lane / (D / 16);
            const uint8_t* row = vpages + page_of(i * ROWS / 16, r & 15) * p.v_sp + ((j0 + r) & (p.page - 1)) * p.v_st;
            vr[i] = *reinterpret_cast<const u32x4*>(row + (vd < p.N ? vd : 0));
        }
    };

    f32x4_t o[D / 16];
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{};
    float m[R], ref[R], l[R];                                        // (ref and l are a lane's own)
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = ref[r] = -INFINITY, l[r] = 0.f;
    int j0 = static_cast<int>(begin) + wave * TOKENS;
    if (j0 < end) load_pages(j0), load_keys(j0), load_values(j0);
    for (; j0 < end; j0 += W * TOKENS) {
        // what belongs to no token that counts, or stands behind a row's end, is zero: a weight of 0 would leave values that are no numbers, and keys' meet in the sums of the tiles' products
        bool whole = p.N == D;
        uint64_t counts[SETS];
#pragma unroll
        for (int a = 0; a < SETS; ++a) {
            counts[a] = __ballot(on[a]);
            whole &= counts[a] == ~0ull;
        }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t keep = counts[t / TILES] >> (64 / TILES * (t % TILES) + col) & 1 ? ~0u : 0u;
#pragma unroll
                for (int s = 0; s < D / 64; ++s) kr[t][s] &= 64 * s + kd < p.N ? keep : 0u;
            }
#pragma unroll
            for (int i = 0; i < VSTEPS; ++i) {
                const int tile = i * ROWS / 16, r = (i * ROWS + lane / (D / 16)) & 15;
                vr[i] &= vd < p.N && counts[tile / TILES] >> (64 / TILES * (tile % TILES) + r) & 1 ? ~0u : 0u;
            }
        }
        f32x4_t s[SETS];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4_t& to = s[t / TILES];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                to = mma16<E>(q[t % TILES][2 * c], widen8<E>(kr[t][c][0], kr[t][c][1]), c == 0 && t % TILES == 0 ? f32x4_t{} : to);
                to = mma16<E>(q[t % TILES][2 * c + 1], widen8<E>(kr[t][c][2], kr[t][c][3]), to);
            }
        }
        float ks[SETS], lv[SETS];
        bool is[SETS];
#pragma unroll
        for (int a = 0; a < SETS; ++a) ks[a] = kscale[a], lv[a] = __builtin_amdgcn_logf(vscale[a]), is[a] = on[a];
        const int next = j0 + W * TOKENS;
        if (next < end) load_keys(next);
        float x[SETS][R], top[R], most[R];
#pragma unroll
        for (int r = 0; r < R; ++r) top[r] = most[r] = -INFINITY;
#pragma unroll
        for (int a = 0; a < SETS; ++a) {
            const float ago = static_cast<float>(all - 1 - j0 - 16 * TILES * a - own);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float dot = s[a][r] * ks[a];
                float y = dot * unit;
                if (p.cap > 0.f) y = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(dot * in)), -2.f * out, out);
                y = fmaf(ago, -slope[r], y);
                x[a][r] = is[a] ? y : -INFINITY;
                most[r] = fmaxf(most[r], x[a][r]);
                top[r] = fmaxf(top[r], x[a][r] + lv[a]);
            }
        }
        bool rises = false, leaves = false;
#pragma unroll
        for (int r = 0; r < R; ++r) rises |= top[r] > m[r], leaves |= most[r] > ref[r] + FAR;
        if (__ballot(rises) != 0ull) {
            float f[R], mine = 1.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float to = row_max(top[r]);
                if constexpr (TILES == 4) to = fmaxf(to, __shfl_xor(to, 16, 64));
                to = fmaxf(fmaxf(to, __shfl_xor(to, 32, 64)), m[r]);
                f[r] = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - to);
                m[r] = to;
                const float other = PER == 4 ? f[r] : __shfl(f[r], col % PER / 4 * 16, 64);
                mine = R == 1 || (col & 3) == r ? other : mine;
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][r] *= mine;
        }
        if (__ballot(leaves) != 0ull)
#pragma unroll
            for (int r = 0; r < R; ++r) raise(ref[r], l[r], most[r]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float base = m[r] == -INFINITY ? 0.f : m[r], low = ref[r] == -INFINITY ? 0.f : ref[r];
#pragma unroll
            for (int a = 0; a < SETS; ++a) {
                const float w = __builtin_amdgcn_exp2f(x[a][r] + lv[a] - base);
                l[r] += __builtin_amdgcn_exp2f(x[a][r] - low);
                lds_st(weight + (4 * grp + r) % PER * WPITCH + 2 * (16 * TILES * a + own), __builtin_bit_cast(uint16_t, from_f<E>(w)));
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < VSTEPS / 2; ++i) {
                const int r = i * ROWS + lane / (D / 16), c = 2 * (lane % (D / 16));
                const u32x4 y = vr[half * VSTEPS / 2 + i];
                lds_st(plane + value_at<D>(r, c), widen8<E>(y[0], y[1]));
                lds_st(plane + value_at<D>(r, c + 1), widen8<E>(y[2], y[3]));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own writes above
            if (half == 1 && next < end) load_values(next);
            const u32x4 w = join(lds_ld<u32x2>(wread + 64 * half), lds_ld<u32x2>(wread + 64 * half + 32));
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                typedef v4s __attribute__((address_space(3))) * ptr;
                const lds_t at = 32 * d;                             // two pieces on: the swaps leave the lowest bit and are taken against it
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(plane + (vread[0] ^ at))), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(plane + (vread[1] ^ at)));
                const u32x2 y = __builtin_bit_cast(u32x2, lo), z = __builtin_bit_cast(u32x2, hi);
                o[d] = mma16<E>(u32x4{y[0], y[1], z[0], z[1]}, w, o[d]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float to = row_max(ref[r]);
        if constexpr (TILES == 4) to = fmaxf(to, __shfl_xor(to, 16, 64));
        raise(ref[r], l[r], fmaxf(to, __shfl_xor(to, 32, 64)));
        l[r] = row_add(l[r]);
        if constexpr (TILES == 4) l[r] += __shfl_xor(l[r], 16, 64);
        l[r] += __shfl_xor(l[r], 32, 64);
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);                    // [wave][head][D], pieces of four channels of a head turned by the head
    if (col == 0 && grp < PER / 4)
#pragma unroll
        for (int r = 0; r < R; ++r) top_of[wave][4 * grp + r] = m[r], sum_of[wave][4 * grp + r] = l[r], ref_of[wave][4 * grp + r] = ref[r];
    if (col < PER)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4_t*>(sums + (wave * PER + col) * D + 4 * ((4 * d + grp) ^ col)) = o[d];
    __syncthreads();
    for (int i = tid; i < G * D / 4; i += 64 * W) {
        const int h = i / (D / 4), c = i % (D / 4);
        if (4 * c >= p.N) continue;
        float top = -INFINITY, ref = -INFINITY;
#pragma unroll
        for (int k = 0; k < W; ++k) top = fmaxf(top, top_of[k][h]), ref = fmaxf(ref, ref_of[k][h]);
        const float base = top == -INFINITY ? 0.f : top, low = ref == -INFINITY ? 0.f : ref;
        float sum = 0.f;
        f32x4_t y = f32x4_t{};
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = __builtin_amdgcn_exp2f(top_of[k][h] - base);
            sum = fmaf(sum_of[k][h], __builtin_amdgcn_exp2f(ref_of[k][h] - low), sum);
            y += *reinterpret_cast<const f32x4_t*>(sums + (k * PER + h) * D + 4 * (c ^ h)) * f;
        }
        const int64_t row = wide(b) * p.H + hk * G + h;
        if (alone) {
            const float f = sum == 0.f ? 0.f : 1.f / sum, g = __builtin_amdgcn_exp2f(0.5f * (base - low));     // (twice: up to 2^(120 + FAR))
            *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + row * p.N + 4 * c) = u32x2{pack2<E>(y[0] * f * g * g, y[1] * f * g * g), pack2<E>(y[2] * f * g * g, y[3] * f * g * g)};
        } else {
            float* to = part + (row * pieces + piece) * (D + 4);
            *reinterpret_cast<f32x4_t*>(to + 4 + 4 * c) = y;
            if (c == 0) to[0] = top, to[1] = sum, to[2] = ref;
        }
    }
}

// How many pieces a sequence is cut into; 0: it stays whole, a workgroup of eight waves each, and is not joined: where two rounds of those are enough, or where there are so many sequences and heads that pieces
// would be small.  us, in pieces and whole: heads of 128, 8 keys' heads, 4 query heads each, room for 500 tokens, 1 row 9.3 9.6, 8 rows 10.2 9.8, 32 rows 16.4 10.0, 64 rows 28 19;  for 1000 tokens (four
// rounds) 9.0 14.1, 10.6 14.2, 25.0 15.2, 34 27;  for 2000, 32 rows 33 25.5, 64 rows 46 42.5;   heads of 64, 32 keys' heads, one query head, 500 tokens 8.4 6.1, 11.7 6.2, 1000 tokens 8.5 7.7, 15.2 11.5;
// 8 keys' heads, 4 query heads, 1000 tokens, 32 rows 21.0 10.8.  (32 keys' heads and 64 rows are 2048 workgroups that stay whole with four waves: with eight 45 us instead of 30.)
inline int plan_of(int B, int H, int Hk, int N, int page, int M) {
    const int64_t blocks = static_cast<int64_t>(B) * Hk * chunks_of(H, Hk), round = N <= 64 && H / Hk <= 8 ? 512 : 256, rounds = (static_cast<int64_t>(M) * page + round - 1) / round;
    const int pieces = pieces_of(B, H, Hk, page, M);
    return pieces > 1 && (rounds <= 2 || (blocks >= 128 && rounds <= 8)) ? 0 : pieces;
}

// Rows of 64 bytes: sixteen or eight neighbouring heads on one XCD, whose L2 reads lines of 128 bytes.  B64, up to 4096 tokens, H32 Hk32 N64: 196 us one by one, 158 in twos, 142 in eights, 133 in
// sixteens; B64 H32 Hk8 N64 54, 45, 45.  Rows of 128 bytes gain nothing: there the heads of a piece come one after the other, or where pieces are many the pieces of a head: B16, up to 8192 tokens,
// H32 Hk8 N128, 16 pieces, 54 us and 58 (in eights 58); B4, up to 131072, H64 Hk8 N128, 64 pieces, 181 and 171 (in eights 177).
inline int group_of(int N, int heads, int pieces, int64_t blocks) {
    if (N <= 64 && blocks >= 64 * 8)
        for (const int group : {16, 8})
            if (heads % group == 0) return group;
    return pieces >= 32 ? 0 : 1;
}

// W waves a workgroup
template <class E, int D, int W> int run(hipStream_t st, const rwkv_paged8_args& p, const int pieces) {
    const int shift = __builtin_ctz(p.page), chunks = chunks_of(p.H, p.Hk);
    float* part = static_cast<float*>(p.workspace);
    const int64_t blocks = static_cast<int64_t>(pieces) * p.Hk * chunks * p.B;
    const int group = group_of(p.N, p.Hk * chunks, pieces, blocks);
    const int64_t shares = blocks / std::max(group, 1), grid = group > 1 ? (shares + 7) / 8 * 8 * group : blocks;
    if (grid > INT_MAX) return RWKV_ERR_SHAPE;
    const auto few = [&](auto tiles, auto heads) {
        hipLaunchKernelGGL((paged8_few<E, D, decltype(tiles)::value, decltype(heads)::value, W>), dim3(static_cast<unsigned>(grid)), dim3(64 * W), 0, st, p, shift, pieces, group, static_cast<int>(shares), part);
    };
    using std::integral_constant;
    // us, B16, up to 8192 tokens, heads of 64 (16 keys' heads) and of 128 (8); paged8_few with 4 tiles, with 2, paged8_attn:
    //   1 query head a key head 35.5 40.4 43.2, 42.9 46.4 45.0;   2: 36.8 41.2 43.8, 47.2 45.9 44.1;   4: 45.1 42.1 45.1, 54.0 46.0 45.2;   8: - 42.9 45.4, - 47.2 45.1
    // but B4, up to 131072 tokens, 8 heads of 128: 171 and 180.  (Four copies of the queries take 64 registers where heads have 128 channels.)
    const int G = p.H / p.Hk;
    if (G == 1) few(integral_constant<int, 4>(), integral_constant<int, 1>());
    else if (D == 64 && G == 2) few(integral_constant<int, 4>(), integral_constant<int, D == 64 ? 2 : 1>());
    else if (G <= 8 && (D == 64 || G > 4)) few(integral_constant<int, 2>(), integral_constant<int, 4>());
    else hipLaunchKernelGGL((paged8_attn<E, D, W>), dim3(static_cast<unsigned>(grid)), dim3(64 * W), 0, st, p, shift, pieces, chunks, group, static_cast<int>(shares), part);
    if (pieces > 1) hipLaunchKernelGGL((paged_join<rwkv_paged8_args, E, D, true>), dim3(p.H, p.B), dim3(256), 0, st, p, shift, pieces, part);
    return launch_status();
}
template <class E> int run_any(hipStream_t st, const rwkv_paged8_args& p) {
    const int pieces = plan_of(p.B, p.H, p.Hk, p.N, p.page, p.M);
    if (pieces == 0) return p.N <= 64 ? run<E, 64, 8>(st, p, 1) : run<E, 128, 8>(st, p, 1);
    return p.N <= 64 ? run<E, 64, WAVES>(st, p, pieces) : run<E, 128, WAVES>(st, p, pieces);
}

int check_paged8(const rwkv_paged8_args* p) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 || p->N <= 0 || p->N > 128 || p->N % 16 != 0 ||
        p->P <= 0 || p->M <= 0 || p->page <= 0 || (p->page & (p->page - 1)) != 0 || static_cast<int64_t>(p->M) * p->page > INT_MAX - 65536 || p->B > 65535 || p->H > 65535 || !scores_ok(p->scale, p->cap)) return RWKV_ERR_SHAPE;
    for (const int64_t s : {p->k_sp, p->k_st, p->k_sh, p->v_sp, p->v_st, p->v_sh}) if (s % 16 != 0) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k_pages, p->v_pages, p->y})) return rc;
    if (p->table == nullptr || p->lens == nullptr || p->k_scales == nullptr || p->v_scales == nullptr) return RWKV_ERR_NULL;
    for (const void* q : {static_cast<const void*>(p->table), static_cast<const void*>(p->lens), static_cast<const void*>(p->slopes), static_cast<const void*>(p->k_scales), static_cast<const void*>(p->v_scales)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    const size_t need = rwkv_paged8_workspace_bytes(p->B, p->H, p->Hk, p->N, p->page, p->M);
    if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" {

// a maximum, a sum and an output of each piece and head
size_t rwkv_paged8_workspace_bytes(int B, int H, int Hk, int N, int page, int M) {
    if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || N > 128 || page <= 0 || M <= 0 || B > 65535 || H > 65535) return 0;
    const int pieces = rwkv::plan_of(B, H, Hk, N, page, M);
    return pieces > 1 ? static_cast<size_t>(B) * H * pieces * (rwkv::width_of(N) + 4) * sizeof(float) : 0;
}

int rwkv_paged8_attn(void* stream, const rwkv_paged8_args* args) {
    using namespace rwkv;
    if (const int rc = check_paged8(args)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return args->dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, *args) : run_any<half_t>(st, *args);
}

}  // extern "C"
