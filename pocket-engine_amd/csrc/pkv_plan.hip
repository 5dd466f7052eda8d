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
#include "pkv_wave.h"

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

constexpr int PLAN_INVALID = 1, PLAN_NO_BLOCKS = 802;  // PKV_ERR_INVALID, PKV_ERR_NO_BLOCKS

// Slot of offset `off` in page `id`: -1 where the page is outside the pool.
__device__ __forceinline__ int plan_slot(int id, int off, int block_size, int num_blocks) {
    return id >= 0 && id < num_blocks ? id * block_size + off : -1;
}

// Sums that saturate: values and caps below 2^30.
struct CappedSum {
    int cap;
    __device__ __forceinline__ int operator()(int a, int b) const { return min(a + b, cap); }
};

// Inclusive prefix sums over a workgroup of NW waves of two values that
// saturate at `ca` and `cb`, on top of the sums a_all and b_all (uniform) of
// the rounds before, which become those of the rounds up to here.
template <int NW>
__device__ __forceinline__ void plan_scan(int& a, int& b, int ca, int cb, int& a_all, int& b_all, int (*part)[2]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const CappedSum sa{ca}, sb{cb};
    a = wave_prefix(a, sa);
    b = wave_prefix(b, sb);
    if (lane == 63) {
        part[wave][0] = a;
        part[wave][1] = b;
    }
    __syncthreads();
    // lane w holds wave w's sums; their prefix, the carried sums in front
    int wa = lane < NW ? part[lane][0] : 0, wb = lane < NW ? part[lane][1] : 0;
    if (lane == 0) {
        wa = sa(wa, a_all);
        wb = sb(wb, b_all);
    }
    wa = wave_prefix(wa, sa);
    wb = wave_prefix(wb, sb);
    a = sa(a, wave ? __builtin_amdgcn_readlane(wa, wave - 1) : a_all);
    b = sb(b, wave ? __builtin_amdgcn_readlane(wb, wave - 1) : b_all);
    a_all = __builtin_amdgcn_readlane(wa, NW - 1);
    b_all = __builtin_amdgcn_readlane(wb, NW - 1);
}

// The first i < n with end[i] > x among the round's ascending ends (n - 1 if none).
__device__ __forceinline__ int plan_find(const int* end, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Rounds of 64 NW rows, each decided by the two sums, then its rows' state (by
// workgroup 0), pages and (TOKENS) tokens spread over the grid's threads: every
// workgroup works the sums out for itself, which takes 2 us of one launch where
// a second launch takes 4. That needs the state read apart from the state
// written; a step in place takes one workgroup, or, with many tokens, leaves
// them (all but the rows' first ones) to plan_tokens_kernel. Nothing that is
// stored is read again (a slot on a new page comes from the free list), so no
// barrier waits for stores.
template <bool TOKENS, int NW>
__global__ void __launch_bounds__(64 * NW) plan_rows_kernel(PlanParams p) {
    constexpr int THREADS = 64 * NW;
    __shared__ int part[NW][2], most[NW][2];
    __shared__ int tok_end[THREADS], page_end[THREADS], first[THREADS], held0[THREADS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, T = p.T, bs = p.block_size;
    const int at0 = blockIdx.x * THREADS + tid, stride = gridDim.x * THREADS;  // of the grid's threads
    const int F = p.free_list ? max(0, min(p.free_count[0], p.num_blocks)) : 0;
    int tok_all = 0, page_all = 0;  // sums of the rounds before (saturated)
    int tokens = 0, pages = 0;      // placed tokens, granted pages so far
    for (int c = 0; c < p.nrows; c += THREADS) {
        const int i = c + tid, here = min(THREADS, p.nrows - c);
        const bool row = tid < here;
        const int n = row ? p.ntok[i] : 0, len = row ? p.len[i] : 0, held = row ? p.held[i] : 0;
        const int count = (int)min((unsigned)(n < 0 ? -(unsigned)n : (unsigned)n), (unsigned)T + 1u);
        const long end = (long)len + n;
        const bool wrong = n > 0 && (len < 0 || held < 0 || held > p.max_blocks || end > (long)p.max_blocks * bs);
        const int need = n > 0 && !wrong ? max(0, (int)((end + bs - 1) / bs) - held) : 0;
        // (a row whose tokens do not fit saturates the tokens' sum for every
        // later row: what those and it would need changes no sum that a row
        // takes pages by)
        int incl = count, asked = min(need, F + 1);
        plan_scan<NW>(incl, asked, T + 1, F + 1, tok_all, page_all, part);
        const bool fits = incl <= T, live = n > 0 && fits && !wrong;
        const bool given = need == 0 || asked <= F;
        const bool good = live && given;
        const int wt = wave_max(row && fits ? incl : 0), wp = wave_max(good && need > 0 ? asked : 0);
        if (lane == 0) {
            most[wave][0] = wt;
            most[wave][1] = wp;
        }
        __syncthreads();
        const int tokens0 = tokens, pages0 = pages;
        tokens = max(tokens, wave_max(lane < NW ? most[lane][0] : 0));
        pages = max(pages, wave_max(lane < NW ? most[lane][1] : 0));
        tok_end[tid] = min(incl, tokens);
        page_end[tid] = min(asked, pages);
        first[tid] = good ? len : -1;
        held0[tid] = held;
        __syncthreads();
        // page j of row c + r that the row takes now
        auto new_page = [&](int r, int j) { return p.free_list[F - page_end[r] + j]; };
        if (row && blockIdx.x == 0) {
            const int have = good ? held + need : held;
            if (i == 0) p.cu[0] = 0;
            p.cu[i + 1] = min(incl, tokens);
            p.limits[i] = good || n == 0 ? have * bs - 1 : -1;
            p.len_out[i] = good ? (int)end : len;
            p.held_out[i] = have;
            p.status[i] = (count > 0 && !fits) || (wrong && fits) ? PLAN_INVALID
                          : n > 0 && !given ? (p.free_list ? PLAN_NO_BLOCKS : PLAN_INVALID) : 0;
        }
        // the round's pages pages0 .. pages - 1
        for (int f = pages0 + at0; f < pages; f += stride) {
            const int r = plan_find(page_end, here, f), j = f - (r ? page_end[r - 1] : pages0);
            p.table[(size_t)(c + r) * p.max_blocks + held0[r] + j] = new_page(r, j);
        }
        auto put = [&](int t, int r, int k) {
            const int f = first[r], at = f < 0 ? k : f + k;
            int slot = -1;
            if (f >= 0) {
                const int pg = at / bs, j = pg - held0[r];
                const int id = j >= 0 ? new_page(r, j) : p.table[(size_t)(c + r) * p.max_blocks + pg];
                slot = plan_slot(id, at - pg * bs, bs, p.num_blocks);
            }
            p.pos[t] = at;
            p.slot_map[t] = slot;
            p.tok_seq[t] = c + r;
        };
        if constexpr (TOKENS) {
            for (int t = tokens0 + at0; t < tokens; t += stride) {
                const int r = plan_find(tok_end, here, t);
                put(t, r, t - (r ? tok_end[r - 1] : tokens0));
            }
        } else if (row && fits && count > 0) {
            put(incl - count, tid, 0);
        }
        if (c + THREADS < p.nrows) __syncthreads();  // the round's arrays are rewritten by the next one
    }
    if (at0 == 0) {
        if (p.nrows == 0) p.cu[0] = 0;
        if (p.free_out) p.free_out[0] = F - pages;
    }
    if constexpr (TOKENS) {
        // tokens behind the last row: no slot, so nothing is written for them
        for (int t = tokens + at0; t < T; t += stride) {
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
    const int pg = at / p.block_size;
    p.slot_map[t] = good ? plan_slot(p.table[(size_t)lo * p.max_blocks + pg], at - pg * p.block_size, p.block_size,
                                     p.num_blocks)
                         : -1;
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
__global__ void __launch_bounds__(1024) plan_truncate_kernel(TruncateParams p) {
    constexpr int THREADS = 1024;
    __shared__ int part[THREADS / 64][2];
    __shared__ int page_end[THREADS], keep0[THREADS];
    const int tid = threadIdx.x, bs = p.block_size;
    const int F = max(0, min(p.free_count[0], p.num_blocks)), room = p.num_blocks - F;
    int pages = 0, unused = 0;
    for (int c = 0; c < p.nrows; c += THREADS) {
        const int i = c + tid;
        const bool row = i < p.nrows;
        const int want = row ? p.new_len[i] : -1, len = row ? p.len[i] : 0, held = row ? p.held[i] : 0;
        const bool cut = want >= 0 && want <= len && held >= 0 && held <= p.max_blocks;
        const int keep = cut ? min(held, (int)(((long)want + bs - 1) / bs)) : held;
        // (more pages than the pool has room for: a state that no plan left;
        // the list ends at the pool's size)
        int gone = cut ? min(held - keep, room + 1) : 0, zero = 0;
        const int pages0 = pages;
        plan_scan<THREADS / 64>(gone, zero, room + 1, 1, pages, unused, part);
        page_end[tid] = min(gone, room);
        keep0[tid] = keep;
        if (cut) {
            p.len[i] = want;
            p.held[i] = keep;
        }
        __syncthreads();
        for (int f = pages0 + tid; f < min(pages, room); f += THREADS) {
            const int r = plan_find(page_end, min(THREADS, p.nrows - c), f), j = f - (r ? page_end[r - 1] : pages0);
            p.free_list[F + f] = p.table[(size_t)(c + r) * p.max_blocks + keep0[r] + j];
        }
        __syncthreads();
    }
    if (tid == 0) p.free_count[0] = F + min(pages, room);
}

}  // namespace pkv
