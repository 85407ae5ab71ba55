// Page tables and slots of requests that grow (the arguments are explained in rwkv_hip.h).
//
// Two prefix sums over the rows, of new tokens and of new pages, and then everything is a row's or a token's own.  The sums are short (a thousand rows take a workgroup
// one scan) beside a second launch or a wait between workgroups, so each workgroup makes all of them for itself, a tile of rows after the other, and keeps a
// tile's in LDS (a token each for 256 rows 5.3 us, a chain of loads, the scan, loads).  It then writes the new pages of every gridDim-th row, a wave a row, and the slots of a range of tokens, which find their row by bisection.
#include <algorithm>
#include <climits>

#include "common.h"

namespace rwkv {
namespace {

// TOKENS a workgroup: a token's bisection is ten reads of LDS in a row.  1024 rows, 358000 tokens: 13.5 us with 2048, 9.9 with 1024, 9.0 with 512, 11.1 with 256 (every workgroup scans the rows).
constexpr int THREADS = 256, OWN = 4, ROWS = THREADS * OWN, TOKENS = 512, MAX_BLOCKS = 2048, ROWS_A_BLOCK = 16;

struct Growth { int64_t tokens, pages; };
DEVINL Growth growth_of(const rwkv_tables_args& p, const int row, const int shift, int& len, int& have) {
    len = max(p.lens[row], 0);
    const int64_t room = (static_cast<int64_t>(p.M) << shift) - len, add = min(static_cast<int64_t>(max(p.more[row], 0)), room > 0 ? room : 0);
    const int64_t mask = (1 << shift) - 1, before = (len + mask) >> shift, after = (len + add + mask) >> shift;
    have = static_cast<int>(before);
    return {add, after - before};
}
DEVINL int held31(const int64_t x) { return static_cast<int>(min(x, static_cast<int64_t>(INT_MAX))); }

__global__ __launch_bounds__(THREADS) void tables_extend(const rwkv_tables_args p, const int shift, const int64_t share) {
    __shared__ int64_t start[ROWS], first[ROWS];                 // of a row's new tokens; of its new pages, in the pool
    __shared__ int lens[ROWS], haves[ROWS], mores[ROWS];
    __shared__ int64_t wave_tokens[4], wave_pages[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t lo = blockIdx.x * share, hi = min(lo + share, static_cast<int64_t>(p.n));
    int64_t tokens = 0, pages = p.taken[0];
    for (int base = 0; base < p.B; base += ROWS) {
        const int rows = min(ROWS, p.B - base);
        Growth mine[OWN], sum = {0, 0};
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const int r = OWN * tid + i;
            mine[i] = {0, 0};
            if (r < rows) {
                mine[i] = growth_of(p, base + r, shift, lens[r], haves[r]);
                mores[r] = static_cast<int>(mine[i].pages);
            }
            sum.tokens += mine[i].tokens;
            sum.pages += mine[i].pages;
        }
        Growth upto = sum;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int64_t a = __shfl_up(upto.tokens, x, 64), b = __shfl_up(upto.pages, x, 64);
            if (lane >= x) upto.tokens += a, upto.pages += b;
        }
        if (lane == 63) wave_tokens[wave] = upto.tokens, wave_pages[wave] = upto.pages;
        __syncthreads();
        int64_t t = tokens + upto.tokens - sum.tokens, g = pages + upto.pages - sum.pages, end = tokens;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < wave) t += wave_tokens[w], g += wave_pages[w];
            end += wave_tokens[w];
            pages += wave_pages[w];
        }
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const int r = OWN * tid + i;
            if (r < rows) start[r] = t, first[r] = g;
            t += mine[i].tokens;
            g += mine[i].pages;
        }
        __syncthreads();
        // this workgroup's rows
        const int offset = static_cast<int>((blockIdx.x + gridDim.x - base % gridDim.x) % gridDim.x);
        for (int64_t x = offset + static_cast<int64_t>(wave) * gridDim.x; x < rows; x += 4ll * gridDim.x) {
            const int r = static_cast<int>(x);
            if (lane == 0) {
                p.starts[base + r] = held31(start[r]);
                p.held[base + r] = static_cast<int>(lens[r] + (r + 1 < rows ? start[r + 1] : end) - start[r]);
            }
            int* to = p.table + static_cast<int64_t>(base + r) * p.M + haves[r];
            for (int c = lane; c < mores[r]; c += 64) {
                const int64_t at = first[r] + c;
                to[c] = at >= 0 && at < p.F ? p.pool[at] : -1;
            }
        }
        // this workgroup's tokens
        for (int64_t i = max(lo, tokens) + tid; i < min(hi, end); i += THREADS) {
            int a = 0, b = rows;                                 // the last row that starts at or before i
            while (b - a > 1) {
                const int m = (a + b) >> 1;
                if (start[m] <= i) a = m;
                else b = m;
            }
            const int64_t place = lens[a] + (i - start[a]);
            const int c = static_cast<int>(place >> shift);
            int64_t page = -1;
            if (c < haves[a]) page = p.table[static_cast<int64_t>(base + a) * p.M + c];
            else {
                const int64_t at = first[a] + (c - haves[a]);
                if (at >= 0 && at < p.F) page = p.pool[at];
            }
            const int64_t slot = (page << shift) + (place & ((1 << shift) - 1));
            p.slots[i] = page >= 0 && slot <= INT_MAX ? static_cast<int>(slot) : -1;
        }
        tokens = end;
        __syncthreads();                                         // before the next tile takes the LDS
    }
    for (int64_t i = max(lo, tokens) + tid; i < hi; i += THREADS) p.slots[i] = -1;
    if (blockIdx.x == 0 && tid == 0) {
        p.starts[p.B] = held31(tokens);
        p.taken_out[0] = held31(pages);
    }
}

int check_tables(const rwkv_tables_args* p) {
    if (p == nullptr) return RWKV_ERR_NULL;
    if (p->B <= 0 || p->M <= 0 || p->F <= 0 || p->n < 0 || p->page <= 0 || (p->page & (p->page - 1)) != 0 || static_cast<int64_t>(p->M) * p->page > INT_MAX - 65536 ||
        static_cast<int64_t>(p->B) * p->M > INT_MAX || p->B > INT_MAX - ROWS) return RWKV_ERR_SHAPE;
    if (p->n > 0 && p->slots == nullptr) return RWKV_ERR_NULL;
    for (const void* x : {static_cast<const void*>(p->lens), static_cast<const void*>(p->more), static_cast<const void*>(p->table), static_cast<const void*>(p->pool), static_cast<const void*>(p->taken),
                          static_cast<const void*>(p->starts), static_cast<const void*>(p->held), static_cast<const void*>(p->taken_out)}) {
        if (x == nullptr) return RWKV_ERR_NULL;
        if (reinterpret_cast<uintptr_t>(x) & 3) return RWKV_ERR_ALIGN;
    }
    return reinterpret_cast<uintptr_t>(p->slots) & 3 ? RWKV_ERR_ALIGN : RWKV_OK;
}

}  // namespace
}  // namespace rwkv

extern "C" int rwkv_tables_extend(void* stream, const rwkv_tables_args* args) {
    using namespace rwkv;
    if (const int rc = check_tables(args)) return rc;
    const rwkv_tables_args& p = *args;
    const int64_t blocks = std::min<int64_t>(MAX_BLOCKS, std::max<int64_t>((static_cast<int64_t>(p.n) + TOKENS - 1) / TOKENS, (static_cast<int64_t>(p.B) + ROWS_A_BLOCK - 1) / ROWS_A_BLOCK));
    const int64_t share = (p.n + blocks - 1) / blocks;
    hipLaunchKernelGGL(tables_extend, dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), p, __builtin_ctz(p.page), share);
    return launch_status();
}
