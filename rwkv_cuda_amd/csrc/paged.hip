// Attention of one new token a sequence over a cache in pages (the arguments are explained in rwkv_hip.h).
//
// Bound by reading the cache: each of its rows is read once for all (up to 16) query heads that share it.  A workgroup takes a piece of a sequence's
// tokens for one key head; its waves take 32 tokens in turn.  On v_mfma_f32_16x16x32 a lane holds one head's scores of eight tokens, S^T = K Q^T with
// the keys as they come from memory, and the weights, packed, are the second operand of O^T += V^T P^T, whose first comes through LDS
// (ds_read_b64_tr_b16).  Waves are joined in LDS, pieces by a second kernel.  The next 32 tokens' rows are on their way while these are worked on; the vector unit is busy
// a third of the time.  bf16 B64 up to 4096 tokens (2111 on average) H32 Hk32 N64: 0.226 ms, 4.9 TB/s; fp16 B4 up to 131072 (91750) H64 Hk8 N128: 0.285 ms, 5.3 TB/s
// (a read-only stream reaches 7.3).  Three or four workgroups a CU and tables in order or shuffled are the same to 5 percent; lengths that are equal take 0.204 of 0.226.
#include <algorithm>
#include <climits>

#include "paged_tile.h"

namespace rwkv {
namespace {

template <class E, int D>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attn(const rwkv_paged_args p, const int shift, const int pieces, const int chunks, const int group, const int shares, float* part) {
    constexpr int ROWS = 64 / (D / 8), VSTEPS = STEP / ROWS;        // rows of an access of a wave, accesses of 32 rows
    __shared__ __align__(16) char smem[WAVES * STEP * 2 * D];
    __shared__ float top_of[WAVES][HEADS], sum_of[WAVES][HEADS];
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
    const E *knew = p.k ? static_cast<const E*>(p.k) + (wide(b) * p.Hk + hk) * p.N : nullptr, *vnew = p.v ? static_cast<const E*>(p.v) + (wide(b) * p.Hk + hk) * p.N : nullptr;
    E *kpages = static_cast<E*>(p.k_pages) + hk * p.k_sh, *vpages = static_cast<E*>(p.v_pages) + hk * p.v_sh;

    u32x4 q[D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        const int d = 32 * s + 8 * grp;
        q[s] = mine && d < p.N ? *reinterpret_cast<const u32x4*>(static_cast<const E*>(p.q) + (wide(b) * p.H + h) * p.N + d) : u32x4{0, 0, 0, 0};
    }
    const float unit = p.scale * LOG2E, in = p.cap > 0.f ? 2.f * unit / p.cap : 0.f, out = p.cap * LOG2E, slope = p.slopes ? p.slopes[h] * LOG2E : 0.f;
    const lds_t plane = lds_of(smem) + wave * STEP * 2 * D;
    lds_t vread[2];
    vread[0] = value_at<D>(4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);
    vread[1] = value_at<D>(16 + 4 * grp + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);

    u32x4 kr[2][D / 32], vr[VSTEPS];
    bool kon[2];
    // the tokens from j0 on: the keys as operands, the values by rows
    const auto load = [&](const int j0) {
        const int own = j0 + (lane & 31);
        const int page = own < end ? table[own >> shift] : -1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = j0 + 16 * e + col, pg = __shfl(page, 16 * e + col, 64);
            kon[e] = pg >= 0 && pg < p.P;
            E* row = kpages + pg * p.k_sp + (j & (p.page - 1)) * p.k_st;
            const bool fresh = knew && j == all - 1;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const int d = 32 * s + 8 * grp;
                kr[e][s] = u32x4{0, 0, 0, 0};
                if (kon[e] && d < p.N) {
                    kr[e][s] = *reinterpret_cast<const u32x4*>((fresh ? knew : row) + d);
                    if (fresh && chunk == 0) *reinterpret_cast<u32x4*>(row + d) = kr[e][s];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) {
            const int r = i * ROWS + lane / (D / 8), d = 8 * (lane % (D / 8)), j = j0 + r, pg = __shfl(page, r, 64);
            E* row = vpages + pg * p.v_sp + (j & (p.page - 1)) * p.v_st;
            const bool fresh = vnew && j == all - 1;
            vr[i] = u32x4{0, 0, 0, 0};
            if (pg >= 0 && pg < p.P && d < p.N) {
                vr[i] = *reinterpret_cast<const u32x4*>((fresh ? vnew : row) + d);
                if (fresh && chunk == 0) *reinterpret_cast<u32x4*>(row + d) = vr[i];
            }
        }
    };

    f32x4_t o[D / 16];
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{};
    float m = -INFINITY, l = 0.f;
    int j0 = static_cast<int>(begin) + wave * STEP;
    if (j0 < end) load(j0);
    for (; j0 < end; j0 += WAVES * STEP) {
        f32x4_t s[2] = {f32x4_t{}, f32x4_t{}};
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) s[e] = mma16<E>(kr[e][c], q[c], s[e]);
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) lds_st(plane + value_at<D>(i * ROWS + lane / (D / 8), lane % (D / 8)), vr[i]);
        // which of the 32 tokens count (lanes 0 .. 15 hold them by column)
        const uint32_t on = static_cast<uint32_t>(__ballot(kon[0]) & 0xffffu) | static_cast<uint32_t>(__ballot(kon[1]) & 0xffffu) << 16;
        const int now = j0;
        if (j0 + WAVES * STEP < end) load(j0 + WAVES * STEP);
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * e + 4 * grp + r;
                float x = s[e][r] * unit;
                if (p.cap > 0.f) x = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[e][r] * in)), -2.f * out, out);
                x = fmaf(static_cast<float>(all - 1 - now - t), -slope, x);
                s[e][r] = on >> t & 1 ? x : -INFINITY;
                top = fmaxf(top, s[e][r]);
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__ballot(top > m) != 0ull) {
            const float to = fmaxf(top, m), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][r] *= f;
        }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[e][r] = __builtin_amdgcn_exp2f(s[e][r] - base);
                l += s[e][r];
            }
        const u32x4 w = {pack2<E>(s[0][0], s[0][1]), pack2<E>(s[0][2], s[0][3]), pack2<E>(s[1][0], s[1][1]), pack2<E>(s[1][2], s[1][3])};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // the wave's own writes above
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
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);                    // [wave][head][D], pieces of four channels of a head turned by the head
    if (grp == 0) top_of[wave][col] = m, sum_of[wave][col] = l;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4_t*>(sums + (wave * HEADS + col) * D + 4 * ((4 * d + grp) ^ col)) = o[d];
    __syncthreads();
    for (int i = tid; i < HEADS * D / 4; i += 64 * WAVES) {
        const int x = i / (D / 4), c = i % (D / 4), hd = chunk * HEADS + x;
        if (hd >= G || 4 * c >= p.N) continue;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) top = fmaxf(top, top_of[k][x]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        f32x4_t y = f32x4_t{};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float f = __builtin_amdgcn_exp2f(top_of[k][x] - base);
            sum = fmaf(sum_of[k][x], f, sum);
            y += *reinterpret_cast<const f32x4_t*>(sums + (k * HEADS + x) * D + 4 * (c ^ x)) * f;
        }
        const int64_t row = wide(b) * p.H + hk * G + hd;
        if (alone) {
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<u32x2*>(static_cast<E*>(p.y) + row * p.N + 4 * c) = u32x2{pack2<E>(y[0] * f, y[1] * f), pack2<E>(y[2] * f, y[3] * f)};
        } else {
            float* to = part + (row * pieces + piece) * (D + 4);
            *reinterpret_cast<f32x4_t*>(to + 4 + 4 * c) = y;
            if (c == 0) to[0] = top, to[1] = sum;
        }
    }
}

// Rows of 128 bytes: eight neighbouring heads on one XCD, which then reads a kilobyte of a token.  B64, up to 4096 tokens, H32 Hk32 N64: 0.247 ms one by one, 0.226 in eights,
// 0.233 in sixteens; B1 65536 tokens 0.123, 0.113, 0.113; B64 up to 4096 H32 Hk8 N64 0.063, 0.061, 0.060.  Rows of 256 bytes (B4 H64 Hk8 N128 0.299, 0.294; B16 up to 4096 H32 Hk8
// N128 0.036, 0.041) gain nothing.
// Otherwise the heads of a piece come one after the other, or where pieces are many the pieces of a head: B4 H64 Hk8 N128, 64 pieces, 0.299 ms and 0.285; B8, 32 pieces,
// 0.150 and 0.143; B16, 16 pieces, 0.036 and 0.041.
inline int group_of(int N, int heads, int pieces, int64_t blocks) {
    if (N <= 64 && heads % 8 == 0 && blocks >= 64 * 8) return 8;
    return pieces >= 32 ? 0 : 1;
}

template <class E, int D> int run(hipStream_t st, const rwkv_paged_args& p) {
    const int shift = __builtin_ctz(p.page), pieces = pieces_of(p.B, p.H, p.Hk, p.page, p.M), chunks = chunks_of(p.H, p.Hk);
    float* part = static_cast<float*>(p.workspace);
    const int64_t blocks = static_cast<int64_t>(pieces) * p.Hk * chunks * p.B;
    const int group = group_of(p.N, p.Hk * chunks, pieces, blocks);
    const int64_t shares = blocks / std::max(group, 1), grid = group > 1 ? (shares + 7) / 8 * 8 * group : blocks;
    if (grid > INT_MAX) return RWKV_ERR_SHAPE;
    hipLaunchKernelGGL((paged_attn<E, D>), dim3(static_cast<unsigned>(grid)), dim3(64 * WAVES), 0, st, p, shift, pieces, chunks, group, static_cast<int>(shares), part);
    if (pieces > 1) hipLaunchKernelGGL((paged_join<rwkv_paged_args, E, D>), dim3(p.H, p.B), dim3(256), 0, st, p, shift, pieces, part);
    return launch_status();
}
template <class E> int run_any(hipStream_t st, const rwkv_paged_args& p) { return p.N <= 64 ? run<E, 64>(st, p) : run<E, 128>(st, p); }

int check_paged(const rwkv_paged_args* p) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if ((p->dtype != RWKV_DTYPE_BF16 && p->dtype != RWKV_DTYPE_FP16) || p->B <= 0 || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk != 0 || p->N <= 0 || p->N > 128 || p->N % 8 != 0 ||
        p->P <= 0 || p->M <= 0 || p->page <= 0 || (p->page & (p->page - 1)) != 0 || static_cast<int64_t>(p->M) * p->page > INT_MAX - 65536 || p->B > 65535 || p->H > 65535 || !scores_ok(p->scale, p->cap)) return RWKV_ERR_SHAPE;
    for (const int64_t s : {p->k_sp, p->k_st, p->k_sh, p->v_sp, p->v_st, p->v_sh}) if (s % 8 != 0) return RWKV_ERR_ALIGN;
    if (const int rc = check_ptrs({p->q, p->k_pages, p->v_pages, p->y})) return rc;
    if (p->table == nullptr || p->lens == nullptr || (p->k == nullptr) != (p->v == nullptr)) return RWKV_ERR_NULL;
    if (!aligned16(p->k) || !aligned16(p->v)) return RWKV_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(p->table), static_cast<const void*>(p->lens), static_cast<const void*>(p->slopes)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return RWKV_ERR_ALIGN;
    const size_t need = rwkv_paged_workspace_bytes(p->B, p->H, p->Hk, p->N, p->page, p->M);
    if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) return RWKV_ERR_WORKSPACE;
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" {

// a maximum, a sum and an output of each piece and head
size_t rwkv_paged_workspace_bytes(int B, int H, int Hk, int N, int page, int M) {
    if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || N <= 0 || N > 128 || page <= 0 || M <= 0 || B > 65535 || H > 65535) return 0;
    const int pieces = rwkv::pieces_of(B, H, Hk, page, M);
    return pieces > 1 ? static_cast<size_t>(B) * H * pieces * (rwkv::width_of(N) + 4) * sizeof(float) : 0;
}

int rwkv_paged_attn(void* stream, const rwkv_paged_args* args) {
    using namespace rwkv;
    if (const int rc = check_paged(args)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return args->dtype == RWKV_DTYPE_BF16 ? run_any<bf16_t>(st, *args) : run_any<half_t>(st, *args);
}

}  // extern "C"
