// Rotary positions on three axes (time, height, width) and rows rotated by
// them.
//
// Positions. A sequence is text with media spans in it: span i holds the
// t h w tokens from index start_i on, laid out [t][h][w]. Text advances all
// three axes by one per token; a span that starts at position b gives its
// token (i, j, k) the position (b + i step, b + j, b + k), and what follows it
// starts at b + extent, extent = max((t - 1) step + 1, h, w). So
//   base_i = start_i + sum_{j < i} (extent_j - t_j h_j w_j),
// a prefix sum over the spans, made once per request (rope_spans); a step's
// row then needs the last span at or before it (rope_positions). Both move next
// to nothing (20 bytes a span, 20 a row) and are bound by their launches: 64
// rows take 2.2 us of the GPU, 7,500 rows behind 600 spans 4.2 (ten dependent
// loads of the search), the spans of 4 requests with 600 each 2.9.
#pragma once
#include "pkv_rows.h"
#include "pkv_wave.h"

namespace pkv {

// Tokens and extent of a span; (0, 0) where a size is below 1, the step below
// 0 or a figure passes 31 bits (such a span moves nothing: its tokens are text).
struct SpanSize {
    int count, extent;
};
__device__ __forceinline__ SpanSize span_size(int t, int h, int w, int step) {
    if (t < 1 || h < 1 || w < 1 || step < 0) return {0, 0};
    const long hw = (long)h * w, time = (long)(t - 1) * step + 1;
    if (hw > 0x7fffffff || hw * t > 0x7fffffff || time > 0x7fffffff) return {0, 0};
    return {(int)(hw * t), max((int)time, max(h, w))};
}

// A workgroup of NW waves per request: the prefix sum in rounds of 64 NW
// spans. Sums wrap (they index nothing).
template <int NW>
__global__ void __launch_bounds__(64 * NW) rope_spans_kernel(const int* __restrict__ span_cu,
                                                             const int* __restrict__ spans, int n_spans,
                                                             int* __restrict__ base) {
    __shared__ int part[2][NW];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int a = max(0, min(span_cu[s], n_spans)), b = max(0, min(span_cu[s + 1], n_spans));
    unsigned carry = 0;
    for (int c = a, turn = 0; c < b; c += 64 * NW, turn ^= 1) {
        const int i = c + tid;
        int start = 0;
        unsigned gain = 0;
        if (i < b) {
            const int* sp = spans + (size_t)i * 5;
            start = sp[0];
            const SpanSize z = span_size(sp[1], sp[2], sp[3], sp[4]);
            gain = (unsigned)z.extent - (unsigned)z.count;
        }
        const unsigned incl = (unsigned)wave_prefix((int)gain);
        unsigned before = carry;
        if constexpr (NW > 1) {
            // (two turns of `part`: a wave a round ahead writes the other one)
            if (lane == 63) part[turn][wave] = (int)incl;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; w++) {
                if (w < wave) before += (unsigned)part[turn][w];
                carry += (unsigned)part[turn][w];
            }
        } else {
            carry += (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
        }
        if (i < b) base[i] = (int)((unsigned)start + before + incl - gain);
    }
}

// A thread per row.
__global__ void __launch_bounds__(256) rope_positions_kernel(const int* __restrict__ pos,
                                                             const int* __restrict__ tok_seq,
                                                             const int* __restrict__ span_cu,
                                                             const int* __restrict__ spans,
                                                             const int* __restrict__ base, int n_req, int n_spans, int T,
                                                             int* __restrict__ rope, int rope_stride) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= T) return;
    const int p = pos[t], s = tok_seq[t];
    int x = p, y = p, z = p;
    if (s >= 0 && s < n_req) {
        const int a = max(0, min(span_cu[s], n_spans)), b = max(0, min(span_cu[s + 1], n_spans));
        // the last span of the sequence with start <= p: in [a, hi)
        int lo = a, hi = max(a, b);
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (spans[(size_t)mid * 5] <= p) lo = mid + 1;
            else hi = mid;
        }
        if (lo > a) {
            const int* sp = spans + (size_t)(lo - 1) * 5;
            const int h = sp[2], w = sp[3], step = sp[4];
            const SpanSize size = span_size(sp[1], h, w, step);
            const unsigned j = (unsigned)p - (unsigned)sp[0], b0 = (unsigned)base[lo - 1];
            if (j < (unsigned)size.count) {
                const unsigned line = j / (unsigned)w;
                x = (int)(b0 + line / (unsigned)h * (unsigned)step);
                y = (int)(b0 + line % (unsigned)h);
                z = (int)(b0 + j - line * (unsigned)w);
            } else {
                x = y = z = (int)(b0 + (unsigned)size.extent + j - (unsigned)size.count);
            }
        }
    }
    rope[t] = x;
    rope[(size_t)rope_stride + t] = y;
    rope[2 * (size_t)rope_stride + t] = z;
}

// Rows normed and rotated.
struct RopeParams {
    const uint16_t *q, *k;
    uint16_t *q_out, *k_out;
    long q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
    const float *q_norm, *k_norm;  // null: no norm
    const int* rope;
    int rope_stride;
    const int* axes;
    const float* inv_freq;
    int Hq, Hkv, half, T;  // half: pairs that are rotated
    float eps;
};

// cos and sin of pos * inv. The product is taken in turns and in 64 bits (three
// roundings: within 2^-51 of its size), and reduced to an eighth of a turn
// there: in 32 bits the angle of a position of 2^17 at the highest frequencies
// would be off by 2^-8. The remainder's series
// (x^9 / 9! and x^10 / 10! last: below 2e-9 at pi / 4) are f32's own rounding.
__device__ __forceinline__ float2 turn_of(int pos, float inv) {
    const double turns = (double)pos * ((double)inv * 0.15915494309189533577);
    const double f = turns - __builtin_rint(turns);  // -1/2 .. 1/2
    const double quarter = __builtin_rint(4.0 * f);
    const float x = (float)(f - 0.25 * quarter) * 6.28318530717958647693f, x2 = x * x;
    const float s = x * (1.f + x2 * (-1.f / 6 + x2 * (1.f / 120 + x2 * (-1.f / 5040 + x2 * (1.f / 362880)))));
    const float c = 1.f + x2 * (-0.5f + x2 * (1.f / 24 + x2 * (-1.f / 720 + x2 * (1.f / 40320 + x2 * (-1.f / 3628800)))));
    const int n = (int)quarter;  // -2 .. 2
    const float cc = n & 1 ? s : c, ss = n & 1 ? c : s;
    // n = 1: (-s, c); 2, -2: (-c, -s); -1: (s, -c)
    return make_float2(n == 1 || (n & 3) == 2 ? -cc : cc, n == -1 || (n & 3) == 2 ? -ss : ss);
}

// A lane takes 16 dims of a head as two 16-byte pieces: where they are
// rotated, the pieces whose dims pair up (half-split pairs (i, i + half)) or
// any two (adjacent pairs (2 i, 2 i + 1)), so no value crosses lanes; D / 16
// lanes share a head and its norm's sum. A workgroup takes the heads of `tb`
// tokens, its threads going through the (token, head) pairs HPB at a time; the
// tokens' cos / sin are made once, in LDS, while the first pair's rows are on
// their way, and each pair's rows are requested before the pair ahead of it is
// worked on. Bound by HBM (every row read and written once): 16,384 rows at 32 /
// 8 heads of 128, 336 MB, take 50 us, 6.7 TB/s (a copy of 2 GiB 4.9; part of the
// rows stays in the last-level cache between calls). A few tokens are bound by
// the chain position -> angle -> row, 5.5 us for 64.
constexpr int rope_tokens(int D) { return 2048 / D; }  // tb at most (8 KiB of cos / sin)
template <class E, int D, bool ADJ, bool STREAM>
__global__ void __launch_bounds__(256) rope_rows_kernel(RopeParams p, int tb) {
    __shared__ __align__(16) float cs[rope_tokens(D)][2][D / 2];  // cos, sin
    constexpr int LPH = D / 16, HPB = 256 / LPH;               // lanes per head, heads at a time
    const int tid = threadIdx.x, t0 = blockIdx.x * tb, u = tid % LPH;
    const int H = p.Hq + p.Hkv, tokens = min(tb, p.T - t0);
    const int pieces = p.half / 8;  // pairs of pieces that are rotated
    const bool turned = u < pieces;
    const int d0 = 8 * (turned ? u : 2 * u), d1 = 8 * (turned ? u + pieces : 2 * u + 1);
    // the (token, head) pair of this thread, and its rows
    int tt = 0, hh = tid / LPH;
    while (hh >= H && tt < tokens) hh -= H, tt++;
    uint4 ra, rb;
    auto load = [&]() {
        const size_t t = t0 + tt;
        const uint16_t* src = hh < p.Hq ? p.q + t * p.q_row + (size_t)hh * p.q_head
                                        : p.k + t * p.k_row + (size_t)(hh - p.Hq) * p.k_head;
        ra = *reinterpret_cast<const uint4*>(src + d0);
        rb = *reinterpret_cast<const uint4*>(src + d1);
    };
    // Angles of (token j, pair f), D / 2 threads a token, of which `half` have
    // a pair; all three axes at once, so that no load waits for the axis.
    struct Angle {
        int time, height, width, axis;
        float inv;
    };
    auto angle = [&](int j, int f) {
        const int* at = p.rope + t0 + j;
        return Angle{at[0], at[p.rope_stride], at[2 * (size_t)p.rope_stride], p.axes[f], p.inv_freq[f]};
    };
    auto keep = [&](const Angle& y, int j, int f) {
        const float2 r = turn_of(y.axis == 1 ? y.height : y.axis == 2 ? y.width : y.time, y.inv);
        cs[j][0][f] = r.x;
        cs[j][1][f] = r.y;
    };
    if (p.half > 0) {
        // the first round's loads stand before those of the rows: loads return
        // in order, and the angles are worked out while the rows come
        constexpr int STEP = 256 / (D / 2);  // tokens a round
        const int f = tid % (D / 2), j = tid / (D / 2);
        const Angle y = angle(min(j, tokens - 1), min(f, p.half - 1));
        if (tt < tokens) load();
        if (f < p.half) {
            if (j < tokens) keep(y, j, f);
            for (int i = j + STEP; i < tokens; i += STEP) keep(angle(i, f), i, f);
        }
    } else if (tt < tokens) {
        load();
    }
    __syncthreads();
    while (tt < tokens) {
        const int t = t0 + tt;
        const bool is_q = hh < p.Hq;
        uint16_t* dst = is_q ? p.q_out + (size_t)t * p.qo_row + (size_t)hh * p.qo_head
                             : p.k_out + (size_t)t * p.ko_row + (size_t)(hh - p.Hq) * p.ko_head;
        const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[2 * i] = E::lo(wa[i]);
            a[2 * i + 1] = E::hi(wa[i]);
            b[2 * i] = E::lo(wb[i]);
            b[2 * i + 1] = E::hi(wb[i]);
        }
        const int row = tt;
        // the next pair's rows are requested before this one is worked on
        hh += HPB;
        while (hh >= H && tt < tokens) hh -= H, tt++;
        if (tt < tokens) load();
        const float* w = is_q ? p.q_norm : p.k_norm;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o);
            const float sc = 1.f / sqrtf(ss / D + p.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                a[i] *= sc * w[d0 + i];
                b[i] *= sc * w[d1 + i];
            }
        }
        uint32_t oa[4], ob[4];
        if (turned) {
            float c[8], s[8];
            // adjacent: frequencies of the first piece's 4 pairs, then of the second's
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const int f = ADJ ? (i ? d1 : d0) / 2 : d0 + i;
                *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(&cs[row][0][f]);
                *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(&cs[row][1][f]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (ADJ) {
                    oa[i] = E::pack(a[2 * i] * c[i] - a[2 * i + 1] * s[i], a[2 * i + 1] * c[i] + a[2 * i] * s[i]);
                    ob[i] = E::pack(b[2 * i] * c[4 + i] - b[2 * i + 1] * s[4 + i],
                                    b[2 * i + 1] * c[4 + i] + b[2 * i] * s[4 + i]);
                } else {
                    const int j = 2 * i;
                    oa[i] = E::pack(a[j] * c[j] - b[j] * s[j], a[j + 1] * c[j + 1] - b[j + 1] * s[j + 1]);
                    ob[i] = E::pack(b[j] * c[j] + a[j] * s[j], b[j + 1] * c[j + 1] + a[j + 1] * s[j + 1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                oa[i] = E::pack(a[2 * i], a[2 * i + 1]);
                ob[i] = E::pack(b[2 * i], b[2 * i + 1]);
            }
        }
        const u32x4 ya = {oa[0], oa[1], oa[2], oa[3]}, yb = {ob[0], ob[1], ob[2], ob[3]};
        u32x4 *pa = reinterpret_cast<u32x4*>(dst + d0), *pb = reinterpret_cast<u32x4*>(dst + d1);
        if constexpr (STREAM) {
            __builtin_nontemporal_store(ya, pa);
            __builtin_nontemporal_store(yb, pb);
        } else {
            *pa = ya;
            *pb = yb;
        }
    }
}

}  // namespace pkv
