// A step planned on the GPU: from the requests' lengths, the pages they need
// (taken from a free list that lies on the GPU), their block tables, and the
// step's per-token metadata. The counterparts on the host are pkv_kv_reserve,
// pkv_kv_fill, pkv_kv_pad and pkv_kv_truncate; a captured decode loop cannot
// call those.
//
// Row s feeds n_s = |ntok_s| tokens. Two prefix sums over the rows decide
// everything: I_s of the tokens (row s holds tokens I_{s-1} .. I_s - 1) and P_s
// of the pages that the rows need; row s takes the pages free[F - P_s + i],
// i < P_s - P_{s-1}, which are the last ones of the list as it stands after
// the rows before it, in list order: the order of pkv_pool_take. Both sums
// saturate just above their limits (T, F), so no length overflows them.
#pragma once
#include "pkv_common.h"

namespace pkv {

struct PlanParams {
    const int *len, *held, *ntok;
    int nrows;
    int* table;
    int max_blocks, block_size, num_blocks;
    const int *free_list, *free_count;  // null: the tables are as they are
    int T;
    int *pos, *slot_map, *tok_seq, *cu, *limits, *len_out, *held_out, *free_out, *status;
};

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_INVALID = 1, PLAN_NO_BLOCKS = 802;  // PKV_ERR_INVALID, PKV_ERR_NO_BLOCKS

// Slot of position p of a row: -1 where the page id is outside the pool.
__device__ __forceinline__ int plan_slot(const int* table, int block_size, int num_blocks, int p) {
    const int pg = p / block_size, id = table[pg];
    return id >= 0 && id < num_blocks ? id * block_size + (p - pg * block_size) : -1;
}

// Inclusive prefix sums over the workgroup of two values that saturate at
// `ca` and `cb` (values at most those; ca, cb < 2^30), on top of what came
// before (a, b start as the carried sums, uniform). Leaves the carried sums of
// the next round in `a_all`, `b_all`.
__device__ __forceinline__ void plan_scan(int& a, int& b, int ca, int cb, int& a_all, int& b_all, int (*part)[2]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(a, o), v = __shfl_up(b, o);
        if (lane >= o) {
            a = min(a + u, ca);
            b = min(b + v, cb);
        }
    }
    if (lane == 63) {
        part[wave][0] = a;
        part[wave][1] = b;
    }
    __syncthreads();
    // lane w of every wave holds wave w's sums; their prefix
    int wa = lane < PLAN_THREADS / 64 ? part[lane][0] : 0, wb = lane < PLAN_THREADS / 64 ? part[lane][1] : 0;
    if (lane == 0) {
        wa = min(wa + a_all, ca);
        wb = min(wb + b_all, cb);
    }
#pragma unroll
    for (int o = 1; o < PLAN_THREADS / 64; o <<= 1) {
        const int u = __shfl_up(wa, o), v = __shfl_up(wb, o);
        if (lane >= o) {
            wa = min(wa + u, ca);
            wb = min(wb + v, cb);
        }
    }
    const int pa = __shfl(wa, max(wave - 1, 0)), pb = __shfl(wb, max(wave - 1, 0));
    a = min(a + (wave ? pa : a_all), ca);
    b = min(b + (wave ? pb : b_all), cb);
    a_all = __shfl(wa, PLAN_THREADS / 64 - 1);
    b_all = __shfl(wb, PLAN_THREADS / 64 - 1);
}

// The first i with end[i] > x among the round's ascending ends (the last one if none).
__device__ __forceinline__ int plan_find(const int* end, int x) {
    int lo = 0, hi = PLAN_THREADS - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// One workgroup: rounds of 1,024 rows, each decided by the two sums, then its
// pages and (TOKENS) its tokens spread over the threads. Without TOKENS a row
// writes its first token, and plan_tokens_kernel the others.
template <bool TOKENS>
__global__ void __launch_bounds__(PLAN_THREADS) plan_rows_kernel(PlanParams p) {
    __shared__ int part[PLAN_THREADS / 64][2];
    __shared__ int tok_end[PLAN_THREADS], page_end[PLAN_THREADS], first[PLAN_THREADS], held0[PLAN_THREADS];
    __shared__ int most[2];
    const int tid = threadIdx.x, T = p.T, bs = p.block_size;
    const int F = p.free_list ? max(0, min(p.free_count[0], p.num_blocks)) : 0;
    int tok_all = 0, page_all = 0;  // sums of the rounds before (saturated)
    int tokens = 0, pages = 0;      // placed tokens, granted pages so far
    if (tid == 0) p.cu[0] = 0;
    for (int c = 0; c < p.nrows; c += PLAN_THREADS) {
        const int i = c + tid;
        const bool row = i < p.nrows;
        const int n = row ? p.ntok[i] : 0, len = row ? p.len[i] : 0, held = row ? p.held[i] : 0;
        const int count = (int)min((unsigned)(n < 0 ? -(unsigned)n : (unsigned)n), (unsigned)T + 1u);
        // (a row that does not fit has no tokens, so its need is not asked; a
        // sum that saturates stays so, so those rows are the last ones)
        const long end = (long)len + n;
        const bool wrong = n > 0 && (len < 0 || held < 0 || held > p.max_blocks || end > (long)p.max_blocks * bs);
        int need = n > 0 && !wrong ? max(0, (int)((end + bs - 1) / bs) - held) : 0;
        // first the tokens alone decide who is in: both sums in one scan need
        // the page sum without rows that do not fit, and such a row's tokens
        // saturate the sum for every later row, so their needs only add to
        // sums that nobody takes pages by
        int incl = count, asked = min(need, F + 1);
        if (tid < 2) most[tid] = tid ? pages : tokens;
        plan_scan(incl, asked, T + 1, F + 1, tok_all, page_all, part);
        const bool fits = incl <= T, live = n > 0 && fits && !wrong;
        const bool given = need == 0 || asked <= F;
        const bool good = live && given;
        if (row && fits) atomicMax(&most[0], incl);
        if (good && need > 0) atomicMax(&most[1], asked);
        __syncthreads();
        const int tokens0 = tokens, pages0 = pages;
        tokens = most[0];
        pages = most[1];
        tok_end[tid] = row ? min(incl, tokens) : tokens;
        page_end[tid] = min(asked, pages);
        first[tid] = good ? len : -1;
        held0[tid] = held;
        if (row) {
            const int have = good ? held + need : held;
            p.cu[i + 1] = min(incl, tokens);
            p.limits[i] = good || n == 0 ? have * bs - 1 : -1;
            p.len_out[i] = good ? (int)end : len;
            p.held_out[i] = have;
            p.status[i] = (count > 0 && !fits) || (wrong && fits) ? PLAN_INVALID
                          : n > 0 && !given ? (p.free_list ? PLAN_NO_BLOCKS : PLAN_INVALID) : 0;
        }
        __syncthreads();
        // pages pages0 .. pages - 1 of the step
        for (int f = pages0 + tid; f < pages; f += PLAN_THREADS) {
            const int r = plan_find(page_end, f), e = page_end[r], j = f - (r ? page_end[r - 1] : pages0);
            p.table[(size_t)(c + r) * p.max_blocks + held0[r] + j] = p.free_list[F - e + j];
        }
        __syncthreads();
        if constexpr (TOKENS) {
            for (int t = tokens0 + tid; t < tokens; t += PLAN_THREADS) {
                const int r = plan_find(tok_end, t), k = t - (r ? tok_end[r - 1] : tokens0), f = first[r];
                p.pos[t] = f < 0 ? k : f + k;
                p.slot_map[t] =
                    f < 0 ? -1 : plan_slot(p.table + (size_t)(c + r) * p.max_blocks, bs, p.num_blocks, f + k);
                p.tok_seq[t] = c + r;
            }
        } else if (row && fits && count > 0) {
            const int t = incl - count;
            p.pos[t] = good ? len : 0;
            p.slot_map[t] = good ? plan_slot(p.table + (size_t)i * p.max_blocks, bs, p.num_blocks, len) : -1;
            p.tok_seq[t] = i;
        }
        __syncthreads();  // the round's arrays are rewritten by the next one
    }
    if (tid == 0 && p.free_out) p.free_out[0] = F - pages;
    if constexpr (TOKENS) {
        // tokens behind the last row: no slot, so nothing is written for them
        for (int t = tokens + tid; t < T; t += PLAN_THREADS) {
            p.pos[t] = 0;
            p.slot_map[t] = -1;
            p.tok_seq[t] = 0;
        }
    }
}

// The tokens that are not a row's first one (which plan_rows_kernel<false>
// wrote, with the row's first position): a thread each. A row whose tokens
// have slots has a limit, the others have none.
__global__ void __launch_bounds__(256) plan_tokens_kernel(PlanParams p) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= p.T) return;
    if (t >= p.cu[p.nrows]) {
        p.pos[t] = 0;
        p.slot_map[t] = -1;
        p.tok_seq[t] = 0;
        return;
    }
    // the row with cu[r] <= t < cu[r + 1]
    int lo = 0, hi = p.nrows - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int a = p.cu[lo], k = t - a;
    if (k == 0) return;
    const bool good = p.limits[lo] >= 0;
    const int at = good ? p.pos[a] + k : k;
    p.pos[t] = at;
    p.slot_map[t] = good ? plan_slot(p.table + (size_t)lo * p.max_blocks, p.block_size, p.num_blocks, at) : -1;
    p.tok_seq[t] = lo;
}

// Rows cut to new_len positions (below 0 or above the row's length: left as
// they are): the pages wholly past it go back to the end of the free list, row
// by row, in table order, as pkv_kv_truncate with free_pages gives them back.
struct TruncateParams {
    const int* new_len;
    int *len, *held;
    int nrows;
    const int* table;
    int max_blocks, block_size, num_blocks;
    int *free_list, *free_count;
};
__global__ void __launch_bounds__(PLAN_THREADS) plan_truncate_kernel(TruncateParams p) {
    __shared__ int part[PLAN_THREADS / 64][2];
    __shared__ int page_end[PLAN_THREADS], keep0[PLAN_THREADS];
    const int tid = threadIdx.x, bs = p.block_size;
    const int F = max(0, min(p.free_count[0], p.num_blocks)), room = p.num_blocks - F;
    int pages = 0, unused = 0;
    for (int c = 0; c < p.nrows; c += PLAN_THREADS) {
        const int i = c + tid;
        const bool row = i < p.nrows;
        const int want = row ? p.new_len[i] : -1, len = row ? p.len[i] : 0, held = row ? p.held[i] : 0;
        const bool cut = want >= 0 && want <= len && held >= 0 && held <= p.max_blocks;
        const int keep = cut ? min(held, (int)(((long)want + bs - 1) / bs)) : held;
        // (more pages than the pool has room for: a state that no plan left;
        // the list ends at the pool's size)
        int gone = cut ? min(held - keep, room + 1) : 0, zero = 0;
        const int pages0 = pages;
        plan_scan(gone, zero, room + 1, 1, pages, unused, part);
        page_end[tid] = min(gone, room);
        keep0[tid] = keep;
        if (cut) {
            p.len[i] = want;
            p.held[i] = keep;
        }
        __syncthreads();
        for (int f = pages0 + tid; f < min(pages, room); f += PLAN_THREADS) {
            const int r = plan_find(page_end, f), j = f - (r ? page_end[r - 1] : pages0);
            p.free_list[F + f] = p.table[(size_t)(c + r) * p.max_blocks + keep0[r] + j];
        }
        __syncthreads();
    }
    if (tid == 0) p.free_count[0] = F + min(pages, room);
}

}  // namespace pkv
