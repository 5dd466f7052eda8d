// Attention over whole prompts that are kept in no cache (pkv_attn_packed):
// packed rows of sequences of different lengths, causal, grouped heads, bf16
// or fp16, heads of 64, 128 or 256 dims.
//
// For query i of a sequence and head h, with kv head h / G:
//   x_j = scale q_i . k_j,  j = 0 .. i
//   out = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m),  m = max_j x_j,
// times sigmoid(gate) where gate rows are given. One pass over the keys with
// the running maximum (kept in log2 units), sum and weighted values.
//
// A workgroup takes RW consecutive rows of one sequence and one kv head, a row
// being a (query, head of the group) pair, row = query * G + head: every G
// shares a K / V tile among its heads, short prompts fill tiles, and a wave's
// 32 rows span only 32 / G queries, so little of a diagonal tile is masked
// work. Scores are computed transposed, S^T[key][row] = K Q^T: a lane then
// holds one row's 16 scores of a 32-key block (keys 8 (r / 4) + 4 (lane / 32)
// + r % 4), the softmax needs one exchange between the lane's halves, and the
// weights are the B operand of O^T[dim][row] += V^T P^T as they stand; V^T
// fragments are read from the row-major V tile by ds_read_b64_tr_b16.
//
// Bound: a 32-key tile of 32 rows takes D / 8 products of 32 x 32 x 16 (32
// cycles each), 16 exponentials a lane, and 128 D bytes of LDS, which the CU's
// 128 bytes a cycle serve to its 4 SIMDs in just those cycles: products and LDS
// reads are even, and the softmax between them is what other waves of the SIMD
// cover. Wider waves (64 rows, half the LDS reads) leave one wave to a SIMD and
// were slower (16,384 tokens at 32 / 8 heads of 128 2,360 us against 2,010).
// That prompt runs at 1,080 to 1,140 TFLOP/s (80 % of the 1,361 that a library
// product of 16,384^3 reaches), its matrix units busy 60 % at 1.7 GHz; 24 prompts
// of 60 to 4,096 tokens 371 us, 881 TFLOP/s; one of 4,096 at 24 / 4 heads of 256
// 216 us, 955 TFLOP/s (cards differ by 5 %). Batches whose longest prompt alone outlasts the rest are bound by
// that prompt's chain of tiles (1.1 to 1.3 us each at 256 dims).
#pragma once
#include "pkv_rows.h"
#include "pkv_wave.h"

namespace pkv {

// 1 / (1 + e^-g); 0 for gates below -87.3, where e^-g passes the reciprocal's
// normal results (the value there is below 1.2e-38).
__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * g));
}

struct PackedParams {
    const uint16_t *q, *k, *v, *gate;  // gate: null for none
    uint16_t* out;
    // row (token) and head strides in elements
    long q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head, o_row, o_head;
    const int* cu;
    int seqs, T, Hkv, G;
    uint32_t g_mul;  // query of a row: its number divided by G (div_group)
    int g_shift;
    int band_shift;  // find_packed_tile
    float scale2;  // scale * log2(e)
};

// r / G for 0 <= r < 2^31 by one product (Granlund and Montgomery): with l =
// ceil(log2 G) and g_mul = floor(2^(31 + l) / G) + 1, the error of r g_mul /
// 2^(31 + l) stays below 1 / G. g_shift = 31 + l.
__device__ __forceinline__ int div_group(const PackedParams& p, int r) {
    return (int)(((uint64_t)(uint32_t)r * p.g_mul) >> p.g_shift);
}

// Shapes of a workgroup for heads of D dims: RG x KS waves, RG of them with 32
// rows each, KS times over: key group g of KS takes the 32-key tiles g, g + KS,
// .. through NST stages of its own, and the groups' sums are joined at the end.
template <int D, int RG, int KS, int NST>
struct PackedTile {
    static constexpr int RW = 32 * RG, NW = RG * KS, THREADS = 64 * NW;
    // A tile of K or V in LDS: NG groups of 1,024 bytes, one LDS DMA
    // instruction each; row r lies in group r % NG at (r / NG) 2 D bytes.
    // K groups are 1,056 bytes apart (1,040 at 256 dims) and rows with bit 3
    // set have their 16-byte pieces swapped in pairs, so the 16 rows that a
    // quarter-wave reads with ds_read_b128 start at distinct 16-byte places
    // modulo 256; V groups are 1,088 bytes apart, so the 4 rows x 64 bytes of
    // a half-wave's transposing read lie on distinct banks.
    static constexpr int NG = D / 16;
    static constexpr int KG = D == 256 ? 1040 : 1056, VG = 1088;
    static constexpr int STAGE = NG * (KG + VG);
    static constexpr int PER = NG / RG;  // groups of K (and of V) that a wave requests per tile
    static constexpr int STAGES = NST * KS * STAGE;
    // Output passes of PW dims, rows staged in f32 (RR floats apart): as many
    // as the stages' LDS holds where the waves join their sums, a barrier each
    // way (one prompt of 300 tokens at 256 dims 13.3 -> 12.8 us), else 64 (32 at
    // 64 dims, where the stages are small and more workgroups fit a CU with
    // less).
    static constexpr int epi(int pw) { return NW * 32 * (pw + 4) * 4; }
    static constexpr int PW = D == 64 && KS < 4 ? 32 : KS > 1 && epi(D) <= STAGES ? D : 64;
    static constexpr int RR = PW + 4, EPI = epi(PW);
    static constexpr int LPR = PW / 8, RPI = 64 / LPR;  // lanes per row, rows a wave writes at once
    static constexpr int LDS = STAGES > EPI ? STAGES : EPI;
    static_assert(NG % RG == 0 && 32 % (RPI * KS) == 0, "whole groups a wave, whole pieces of rows a key group");
    static_assert(NST == 2 || (RG == 1 && NST == 1), "two stages, or one where a wave has it for itself");
    static __device__ __forceinline__ constexpr int swap(int r) { return D == 256 ? 0 : (r >> 3) & 1; }
};

// This workgroup's sequence (rows c0 .. c0 + n - 1) and its tile x of it. False
// where the grid has more workgroups than the batch has tiles. Every wave finds
// them for itself, without LDS or barriers.
//
// LEVEL_SEQS sequences or fewer: a tile x of any sequence attends up to (x + 1)
// RW / G keys, so the order of the tiles is the order of their work, and the
// longest are started first, whatever the sequences' order: with c_s tiles in
// sequence s, N(j) = sum_s max(0, c_s - j) tiles have x >= j, so the tile of
// rank r has the largest x with N(x) > r, found by halving, 4 sequences to a lane
// (about 0.5 us beside the offsets' load). Where the grid has many turns its
// tiles are ordered so by bands of 2^band_shift levels only, and within a band
// sequence by sequence: tiles of one sequence that run together read K and V
// from memory once (255 prompts of up to 2,000 tokens at 32 / 8 heads of 128
// 4,290 -> 2,750 us; but 16 of 200 at 16 / 4 of 256, one turn, 23.8 -> 25.5).
//
// More sequences: sequence s owns the ids from floor(cu[s] G / RW) + s on, as
// many as it has tiles or one more, and is found among them by steps of 64: one
// of 5,000 in 3 loads (a prefix sum over all offsets took longer than a short
// sequence's attention: 2,000 sequences of 64 tokens at 12 / 12 heads of 64 278
// -> 178 us, 5,000 of 1 to 8 at 32 / 8 of 128 552 -> 304).
constexpr int LEVEL_SEQS = 256;
template <int RW>
__device__ __forceinline__ bool find_packed_tile(const PackedParams& p, int tile, int& c0, int& n, int& x) {
    const int lane = threadIdx.x & 63;
    // offsets outside [0, T] are clamped: no row out of range is touched
    auto at = [&](int s) { return max(0, min(p.cu[s], p.T)); };
    auto tiles = [&](int a, int b) { return b > a ? ((b - a) * p.G + RW - 1) / RW : 0; };
    if (p.seqs == 1) {
        c0 = at(0);
        n = at(1) - c0;
        x = tiles(c0, c0 + n) - 1 - tile;
        return x >= 0;
    }
    if (p.seqs <= LEVEL_SEQS) {
        int off[5], c[4], most = 0, sum = 0;
#pragma unroll
        for (int i = 0; i < 5; i++) off[i] = at(min(4 * lane + i, p.seqs));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[i] = tiles(off[i], off[i + 1]);
            most = max(most, c[i]);
            sum += c[i];
        }
        const int total = wave_sum(sum);
        if (tile >= total) return false;
        auto above = [&](int j) {
            int k = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) k += max(0, c[i] - j);
            return wave_sum(k);
        };
        // in bands: N(lo's first level) > tile; after = N(that of hi + 1)
        const int band = 1 << p.band_shift;
        int lo = 0, hi = (wave_max(most) - 1) >> p.band_shift, after = 0;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1, k = above(mid << p.band_shift);
            if (k > tile) {
                lo = mid;
            } else {
                hi = mid - 1;
                after = k;
            }
        }
        // the band's tiles, sequence by sequence, the longest first
        int d[4], k = 0;
        lo <<= p.band_shift;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            d[i] = max(0, min(c[i] - lo, band));
            k += d[i];
        }
        const int incl = wave_prefix(k);
        int r = tile - after - (incl - k), a = 0, b = 0;
        const unsigned long long hit = __ballot(r >= 0 && r < k);
        if (hit == 0) return false;  // offsets that decrease, with counts past 31 bits
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (r >= 0 && r < d[i]) {
                a = off[i];
                b = off[i + 1];
                x = lo + d[i] - 1 - r;
            }
            r -= d[i];
        }
        const int l = __ffsll((long long)hit) - 1;
        c0 = __builtin_amdgcn_readlane(a, l);
        n = __builtin_amdgcn_readlane(b, l) - c0;
        x = __builtin_amdgcn_readlane(x, l);
        return true;
    }
    // (Ids without a tile often lie at every second place. Workgroups go to the
    // card's parts in turn, so 64 ids have their even ones first: 3,000 sequences
    // of 32 tokens at 12 / 12 heads of 64 152 -> 127 us.)
    if ((tile & ~63) + 64 <= (int)(gridDim.x / p.Hkv)) tile = (tile & ~63) + ((tile & 31) << 1) + ((tile >> 5) & 1);
    // The last sequence that starts at or before id `tile`.
    auto start = [&](int s) { return at(s) * p.G / RW + s; };
    int s = 0;
    for (int left = p.seqs; left > 1;) {
        const int step = (left + 63) / 64, i = lane * step;
        const int k = __popcll(__ballot(i < left && start(min(s + i, p.seqs)) <= tile));
        if (k == 0) return false;
        s += (k - 1) * step;
        left = min(step, left - (k - 1) * step);
    }
    c0 = at(s);
    n = at(s + 1) - c0;
    const int c = tiles(c0, c0 + n);
    x = c - 1 - (tile - start(s));
    return x >= 0 && x < c;
}

// s_waitcnt lgkmcnt(0) that leaves the other counters alone, and keeps memory
// accesses on their sides.
__device__ __forceinline__ void wait_lds() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// `odd`: 2 D + 1 words: per dim the first keys with values that are not finite
// (tame, below), and whether there are any.
template <class E, int D, int RG, int KS, int NST>
__device__ __forceinline__ void packed_tile(const PackedParams& p, char* smem, int* odd, int c0, int n, int x, int kvh) {
    using S = PackedTile<D, RG, KS, NST>;
    constexpr int NG = S::NG, BK = 32, NW = S::NW;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lq = lane & 31,
              lh = lane >> 5;
    const int rg = wave % RG, kg = wave / RG;  // row group, key group
    const int rows = n * p.G;                  // of the sequence
    const int row0 = x * S::RW;                // first of this tile
    const int wrow = row0 + 32 * rg;           // first of this wave
    // Query and head in the group of row r; rows past the sequence stand for
    // its last one and are not written.
    auto split = [&](int r, int& qi, int& hh) {
        r = min(r, rows - 1);
        qi = div_group(p, r);
        hh = r - qi * p.G;
    };
    const int L = div_group(p, min(row0 + S::RW, rows) - 1) + 1;  // keys of this tile
    const int ntiles = (L + BK - 1) / BK;
    const int first_q = div_group(p, row0);                        // of the tile
    const int wfirst = div_group(p, min(wrow, rows - 1));          // of the wave
    const int last = wrow < rows ? div_group(p, min(wrow + 32, rows) - 1) : -1;  // the wave's last (no rows: none)

    // Requests of K and V rows, straight to LDS: the wave's PER groups of its
    // key group's tile, lane i bringing 16 bytes of row g + NG (i / (D / 8))
    // (K: of the piece that belongs at its place).
    constexpr int CH = D / 8;  // 16-byte pieces per row
    char* const stage = smem + kg * (NST * S::STAGE);
    const int g0 = rg * S::PER;
    const int lb = lane / CH, lc = lane % CH;
    const uint32_t k_row2 = (uint32_t)p.k_row * 2, v_row2 = (uint32_t)p.v_row * 2;
    const uint32_t piece_k = 16 * (lc ^ (D == 128 ? lb & 1 : D == 64 ? (lb >> 1) & 1 : 0)), piece_v = 16 * lc;
    const uint32_t off_k = (uint32_t)(NG * lb) * k_row2 + piece_k, off_v = (uint32_t)(NG * lb) * v_row2 + piece_v;
    const char* kb = reinterpret_cast<const char*>(p.k + c0 * p.k_row + kvh * p.k_head);
    const char* vb = reinterpret_cast<const char*>(p.v + c0 * p.v_row + kvh * p.v_head);
    const uint32_t lds0 = lds_addr(stage);
    auto request = [&](int k0, int buf) __attribute__((always_inline)) {
        const uint32_t lk = lds0 + buf * S::STAGE + g0 * S::KG;
        const uint32_t lv = lds0 + buf * S::STAGE + NG * S::KG + g0 * S::VG;
        const int r0 = k0 + g0;
        if (k0 + BK <= L) {
            const char* ks = kb + (size_t)r0 * k_row2;
            const char* vs = vb + (size_t)r0 * v_row2;
#pragma unroll
            for (int i = 0; i < S::PER; i++) dma16_s(ks + (size_t)i * k_row2, off_k, lk + i * S::KG);
#pragma unroll
            for (int i = 0; i < S::PER; i++) dma16_s(vs + (size_t)i * v_row2, off_v, lv + i * S::VG);
        } else {
            // the last tile: rows past the keys stand for the last key; a lane's
            // row goes up with the group until it is that one
            const char* ks = kb + (size_t)k0 * k_row2;
            const char* vs = vb + (size_t)k0 * v_row2;
            const int end = L - 1 - k0, first = min(g0 + NG * lb, end);
            uint32_t ok = (uint32_t)first * k_row2 + piece_k, ov = (uint32_t)first * v_row2 + piece_v;
#pragma unroll
            for (int i = 0; i < S::PER; i++) {
                dma16_s(ks, ok, lk + i * S::KG);
                dma16_s(vs, ov, lv + i * S::VG);
                const bool up = g0 + i + NG * lb < end;
                ok += up ? k_row2 : 0;
                ov += up ? v_row2 : 0;
            }
        }
    };

    if (kg < ntiles) request(kg * BK, 0);
    for (int i = tid; i <= 2 * D; i += S::THREADS) odd[i] = i < 2 * D ? 0x7fffffff : 0;
    uint4 qf[D / 16];
    int qi;
    {
        int hh;
        split(wrow + lq, qi, hh);
        const uint16_t* src = p.q + (size_t)(c0 + qi) * p.q_row + (size_t)(kvh * p.G + hh) * p.q_head + 8 * lh;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) qf[kk] = *reinterpret_cast<const uint4*>(src + 16 * kk);
    }
    // The gates of the rows that a lane writes at the end (pass ps, row k). With
    // several key groups they are few enough to be requested here (at 256 dims
    // they would push the sums out of the first 256 registers); else they come
    // before the first output pass.
    constexpr int PW = S::PW, RPI = S::RPI, RK = 32 / (RPI * KS);  // RK rows a lane
    const int er = lane / S::LPR, ec = lane % S::LPR;
    uint4 gr[D / PW][RK];
    auto load_gates = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < RK; k++) {
            int qq, hh;
            split(wrow + RPI * (RK * kg + k) + er, qq, hh);
            const uint16_t* src = p.gate + (size_t)(c0 + qq) * p.g_row + (size_t)(kvh * p.G + hh) * p.g_head + 8 * ec;
#pragma unroll
            for (int ps = 0; ps < D / PW; ps++) gr[ps][k] = *reinterpret_cast<const uint4*>(src + PW * ps);
        }
    };
    constexpr bool EARLY = KS > 1 && D < 256;
    if (EARLY && p.gate) load_gates();
    f32x16 o[D / 32];
    // running maximum (log2 units; 0 before the first key; may lag, below) and
    // the lane's own part of the sum
    float m = 0.f, l = 0.f, limit = -1.f;
    bool fresh = true;  // uniform: some row of the wave has no key yet
#pragma unroll
    for (int db = 0; db < D / 32; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[db][r] = 0.f;

    // Lane addresses in a tile of K and V (bytes).
    const int k_at = (lq % NG) * S::KG + lq / NG * (2 * D) + 16 * (lh ^ S::swap(lq));
    const int tr_r = 4 * lh + ((lane & 15) >> 2);  // + 16 kk + 8 h: row of the transposing read
    const int v_at = NG * S::KG + tr_r % NG * S::VG + tr_r / NG * (2 * D) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    // row + 8 h + 16 kk of the tile, from v_at
    auto v_step = [](int kk, int h) constexpr { return D == 256 ? h * 8 * S::VG + kk * 2 * D : (16 * kk + 8 * h) / NG * 2 * D; };
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

    auto compute = [&](int buf, int k0) __attribute__((always_inline)) {
        const char* K = stage + buf * S::STAGE + k_at;
        const char* V = stage + buf * S::STAGE + v_at;
        f32x16 st;
#pragma unroll
        for (int r = 0; r < 16; r++) st[r] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) st = E::mfma(*reinterpret_cast<const uint4*>(K + 32 * kk), qf[kk], st);
        if (k0 + BK - 1 > wfirst) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (k0 + 8 * (r >> 2) + 4 * lh + (r & 3) > qi) st[r] = -INFINITY;
        }
        // Weights against the maximum as it stands. P is rounded to the type of
        // the rows, as the matrix units take it; the sum is of the rounded
        // weights, so they still add up to 1.
        uint4 pb[2];
        float sum;
        auto weigh = [&](float base) __attribute__((always_inline)) {
            sum = 0.f;
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float s0 = st[8 * kk + 2 * i], s1 = st[8 * kk + 2 * i + 1];
                    w[i] = E::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(s0, p.scale2, -base)),
                                   __builtin_amdgcn_exp2f(__builtin_fmaf(s1, p.scale2, -base)));
                    sum = E::dot(w[i], E::ONE, sum);
                }
                pb[kk] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        };
        // The maximum is looked for only before a row's first key (`limit` is
        // -1) and where the tile's weights outgrow it (a lane's 16 add up to
        // more than 2^10): weights up to 2^10, all of a row relative to the
        // same power, lose no digit, and almost every tile is spared the
        // search, the rescaling of O and the wait for both between the two
        // products.
        bool search = fresh;
        if (!fresh) {
            weigh(m);
            search = __any(sum > limit);
        }
        if (search) {
            float mx = st[0];
#pragma unroll
            for (int r = 1; r < 16; r++) mx = fmaxf(mx, st[r]);
            mx = fmaxf(max_xor32(mx) * p.scale2, limit < 0.f ? -INFINITY : m);
            // scores of -inf so far: their weight is 0, not NaN
            const float base = mx == -INFINITY ? 0.f : mx;
            const float corr = limit < 0.f ? 0.f : __builtin_amdgcn_exp2f(m - base);
            m = base;
            limit = mx == -INFINITY ? -1.f : 1024.f;
            fresh = __any(limit < 0.f);
            l *= corr;
#pragma unroll
            for (int db = 0; db < D / 32; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[db][r] *= corr;
            weigh(m);
        }
        l += sum;
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int db = 0; db < D / 32; db++) {
                const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(V + v_step(kk, 0) + 64 * db));
                const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(V + v_step(kk, 1) + 64 * db));
                o[db] = E::mfma(__builtin_bit_cast(uint4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)), pb[kk], o[db]);
            }
    };

    // A weight of 0 times an infinite or NaN value is NaN, so a value must not
    // meet the weights of rows that do not attend its key. Only tiles with
    // keys behind the workgroup's first query can hold such a pair: there the
    // wave looks through the values that it brought, takes out what is not
    // finite, and notes for its dim the first key with (+inf or NaN) and with
    // (-inf or NaN). A row attends a key if and only if the key is not behind
    // it, so those two say what the finished rows get.
    auto tame = [&](int k0, int buf) __attribute__((always_inline)) {
        if (k0 + BK - 1 <= first_q) return;
        uint4* at = reinterpret_cast<uint4*>(stage + buf * S::STAGE + NG * S::KG + g0 * S::VG + 16 * lane);
        bool bad = false;
        if constexpr (D == 256 && KS == 1) {
            // (4 groups. Looked at together as below they leave the loop's
            // registers 2 % slower: one prompt of 4,096 tokens at 24 / 4 heads
            // 212 -> 216 us.)
            auto odd_pair = [](uint32_t w) {  // a half whose exponent is all ones
                const uint32_t u = ~w & E::EXP;
                return (u & 0xffffu) == 0 || u < 0x10000u;
            };
#pragma unroll
            for (int i = 0; i < S::PER; i++) {
                const uint4 x = at[i * (S::VG / 16)];
                bad |= odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w);
            }
        } else {
            // All the wave's groups are read before one is looked at: by the
            // largest exponent bits of either half (a wave with 16 groups
            // 4,400 -> 900 cycles; one prompt of 37 tokens 9.7 -> 8.2 us).
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            u16x2 top = {0, 0};
#pragma unroll
            for (int i = 0; i < S::PER; i++) {
                const uint4 x = at[i * (S::VG / 16)];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; e++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[e] & E::EXP));
            }
            const unsigned short all = (unsigned short)E::EXP;
            bad = top.x == all || top.y == all;
        }
        if (!__any(bad)) return;
#pragma unroll 1
        for (int i = 0; i < S::PER; i++) {
            if (!bad) continue;
            const uint4 x = at[i * (S::VG / 16)];
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            const int key = k0 + g0 + i + NG * lb;
#pragma unroll 1
            for (int e = 0; e < 8; e++) {
                const uint32_t y = w[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                if ((~y & E::EXP & 0xffffu) != 0) continue;
                const bool nan = y & E::MANT & 0xffffu, minus = y >> 15;
                if (nan || !minus) atomicMin(odd + 8 * lc + e, key);
                if (nan || minus) atomicMin(odd + D + 8 * lc + e, key);
                w[e >> 1] &= ~(0xffffu << (16 * (e & 1)));
            }
            at[i * (S::VG / 16)] = make_uint4(w[0], w[1], w[2], w[3]);
            odd[2 * D] = 1;
        }
    };

    __syncthreads();  // `odd` is set
    if constexpr (RG == 1) {
        // The wave has its tiles for itself: no barriers.
        for (int it = kg, buf = 0; it < ntiles; it += KS) {
            const int k0 = it * BK;
            const bool more = it + KS < ntiles;
            wait_vm<0>();
            tame(k0, buf);
            wave_sync();
            if (NST == 2 && more) request(k0 + KS * BK, buf ^ 1);
            if (k0 <= last) compute(buf, k0);
            wait_lds();  // the stage is read before the next request writes it
            if (NST == 1 && more) request(k0 + KS * BK, 0);
            if (NST == 2) buf ^= 1;
        }
    } else {
        // Two stages: a step requests its key group's next tile into the stage
        // that the barrier before it freed, computes its tile, waits for its own
        // requests, and the barrier publishes the next tile.
        wait_vm<0>();
        if (kg < ntiles) tame(kg * BK, 0);
        __syncthreads();
        for (int it = 0, buf = 0; it < ntiles; it += KS, buf ^= 1) {
            const int k0 = (it + kg) * BK, k1 = k0 + KS * BK;
            if (k1 < L) request(k1, buf ^ 1);
            if (k0 <= last) compute(buf, k0);
            if (it + KS < ntiles) {
                wait_vm<0>();
                if (k1 < L) tame(k1, buf ^ 1);
                __syncthreads();
            }
        }
    }

    // Rows out: a lane holds 4-dim pieces of one row, so 32 columns are 32 rows
    // and go through LDS (PW dims a pass, f32: the one rounding comes after the
    // gate), and leave as 16-byte pieces, LPR lanes per row. With several key
    // groups their sums, brought to the same maximum, are added there, each
    // group's wave finishing its part of the 32 rows.
    __shared__ float join[KS > 1 ? NW : 1][2][32];
    if constexpr (KS > 1) {
        l = add_xor32(l);
        if (lh == 0) {
            join[wave][0][lq] = limit < 0.f ? -INFINITY : m;  // no key yet
            join[wave][1][lq] = l;
        }
    }
    __syncthreads();  // every wave is past the last tile's stage
    float* const out_stage = reinterpret_cast<float*>(smem) + rg * 32 * S::RR;  // key group g's: + g RG 32 RR
    const bool any_odd = odd[2 * D] != 0;
    size_t t[RK];
    int head[RK], query[RK];
    bool ok[RK];
#pragma unroll
    for (int k = 0; k < RK; k++) {
        const int r = wrow + RPI * (RK * kg + k) + er;
        int hh;
        split(r, query[k], hh);
        ok[k] = r < rows;
        t[k] = (size_t)(c0 + query[k]);
        head[k] = kvh * p.G + hh;
    }
    if (!EARLY && p.gate) load_gates();
    float inv;
    if constexpr (KS > 1) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int g = 0; g < KS; g++) top = fmaxf(top, join[g * RG + rg][0][lq]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int g = 0; g < KS; g++) sum += join[g * RG + rg][1][lq] * __builtin_amdgcn_exp2f(join[g * RG + rg][0][lq] - base);
        inv = __builtin_amdgcn_exp2f(join[wave][0][lq] - base) / sum;
    } else {
        inv = 1.f / add_xor32(l);
    }
#pragma unroll
    for (int ps = 0; ps < D / PW; ps++) {
#pragma unroll
        for (int db = PW / 32 * ps; db < PW / 32 * (ps + 1); db++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const f32x16& y = o[db];
                *reinterpret_cast<float4*>(out_stage + kg * (RG * 32 * S::RR) + lq * S::RR + 32 * (db - PW / 32 * ps) + 8 * g +
                                           4 * lh) =
                    make_float4(y[4 * g] * inv, y[4 * g + 1] * inv, y[4 * g + 2] * inv, y[4 * g + 3] * inv);
            }
        if (KS > 1) __syncthreads();
        else wave_sync();
#pragma unroll
        for (int k = 0; k < RK; k++) {
            const float* src = out_stage + (RPI * (RK * kg + k) + er) * S::RR + 8 * ec;
            float y[8];
#pragma unroll
            for (int g = 0; g < KS; g++) {
                const float4 a = *reinterpret_cast<const float4*>(src + g * (RG * 32 * S::RR)),
                             b = *reinterpret_cast<const float4*>(src + g * (RG * 32 * S::RR) + 4);
                const float z[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = g == 0 ? z[i] : y[i] + z[i];
            }
            if (any_odd) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (query[k] >= odd[PW * ps + 8 * ec + i]) y[i] += INFINITY;
                    if (query[k] >= odd[D + PW * ps + 8 * ec + i]) y[i] -= INFINITY;
                }
            }
            if (p.gate) {
                const uint4 g = gr[ps][k];
                const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    y[2 * i] *= sigmoid(E::lo(gw[i]));
                    y[2 * i + 1] *= sigmoid(E::hi(gw[i]));
                }
            }
            if (ok[k])
                *reinterpret_cast<uint4*>(p.out + t[k] * p.o_row + (size_t)head[k] * p.o_head + PW * ps + 8 * ec) =
                    make_uint4(E::pack(y[0], y[1]), E::pack(y[2], y[3]), E::pack(y[4], y[5]), E::pack(y[6], y[7]));
        }
        // the region is rewritten by the next pass
        if (KS > 1) __syncthreads();
        else wave_sync();
    }
}

// 1-D grid of at least (tiles of the batch) x Hkv workgroups, kv heads first:
// workgroup ids go to the 8 XCDs in turn, so with 1, 2, 4 or a multiple of 8
// kv heads an XCD reads the K and V of few heads through its L2.
template <class E, int D, int RG, int KS, int NST, int OCC>
__global__ void __launch_bounds__(64 * RG * KS, OCC) packed_kernel(PackedParams p) {
    using S = PackedTile<D, RG, KS, NST>;
    __shared__ __align__(16) char smem[S::LDS];
    __shared__ int odd[2 * D + 1];
    const int kvh = blockIdx.x % p.Hkv;
    int c0, n, x;
    if (!find_packed_tile<S::RW>(p, blockIdx.x / p.Hkv, c0, n, x)) return;
    c0 = __builtin_amdgcn_readfirstlane(c0);  // scalars, for the requests' bases
    n = __builtin_amdgcn_readfirstlane(n);
    x = __builtin_amdgcn_readfirstlane(x);
    packed_tile<E, D, RG, KS, NST>(p, smem, odd, c0, n, x, kvh);
}

}  // namespace pkv
