// C-ABI entry point of the attention over packed prompts (include/pkv.h).
#include "pkv_packed.hip"
#include "pkv_entry.h"

#include <algorithm>
#include <cmath>

namespace {

// Tiles of RW rows that the batch can have: each sequence with rows rounds up
// once (many sequences: each has an id, find_packed_tile).
int64_t tile_bound(const pkv::PackedParams& p, int rw) {
    return ((int64_t)p.T * p.G + rw - 1) / rw + (p.seqs > pkv::LEVEL_SEQS ? p.seqs : std::min(p.seqs, p.T));
}

template <class E, int D, int RG, int KS, int NST, int OCC>
int launch(pkv::PackedParams p, hipStream_t stream) {
    using S = pkv::PackedTile<D, RG, KS, NST>;
    const int64_t grid = tile_bound(p, S::RW) * p.Hkv;
    // four turns of the grid or more: tiles by bands of 16 levels (find_packed_tile)
    p.band_shift = grid > (int64_t)4 * OCC * device_cus() ? 4 : 0;
    if (grid * S::THREADS >= (int64_t)1 << 32) return PKV_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((pkv::packed_kernel<E, D, RG, KS, NST, OCC>), dim3((unsigned)grid), dim3(S::THREADS), 0, stream, p);
    return launch_status();
}

// How the rows and keys are shared out, by an estimate of the time in key tiles
// of 32. RG waves with 32 rows each, KS times over for the keys: a workgroup's
// time is its share of the tiles plus A tiles' worth of start and end, at the
// mean length n = T / seqs, and the grid takes the longest workgroup or, where
// it holds more than the card's places, the places' turns at the mean (half the
// keys, causal). Measured, us, for 1 x 4, 2 x 2, 4 x 1 and 1 x 1 (RG x KS): 256
// dims at 16 / 4 heads, one prompt of 600 tokens 18 / 22 / 31 / -, 1,200 39 / 35 /
// 51 / -, 2,400 100 / 91 / 95 / -, 1,500 of 3 - / - / 88 / 58; 128 dims at 32 / 8,
// one of 500 10 / 11 / 16 / -, 1,200 29 / 23 / 32 / -, 16 of 200 44 / 29 / 21 / -,
// 257 of 512 - / - / 894 / 1,274, 1,000 of 16 - / - / 83 / 66; 64 dims at 12 / 2, one
// of 2,000 16 / 22 / 37 / -, 2,000 of 1 to 30 - / - / 30 / 24. One wave alone starts
// and ends without waiting for others (the smaller A), but its tiles come from
// one stage that no other wave shares (the pace), so it is for sequences of two
// tiles or fewer (4,000 and 30 of 50 tokens at 8 / 1 heads of 128: 93 us, with one
// wave 128). The estimate takes the fastest, or one within 17 %, in the 35 batches
// of few sequences and 70 of many that were timed; it knows no more of the
// lengths than their mean, so a long prompt among short ones on an idle card runs
// as long as its own chain of tiles.
struct Shape {
    int rows;      // of a workgroup
    double pace;   // tiles of a row at a time
    int places;    // workgroups a CU holds
    double start;  // A in turns
    double alone;  // A of the longest workgroup
};
int best_shape(const pkv::PackedParams& p, const Shape (&shapes)[4]) {
    const double tiles = (double)p.T / p.seqs / 32;
    int best = 0;
    double least = 0;
    for (int i = 0; i < 4; i++) {
        const Shape& s = shapes[i];
        if (s.pace < 1 && tiles > 2) continue;
        const double turns = (double)tile_bound(p, s.rows) * p.Hkv / ((double)s.places * device_cus());
        const double t = std::max(tiles / s.pace + s.alone, turns * (tiles / (2 * s.pace) + s.start));
        if (i == 0 || t < least) best = i, least = t;
    }
    return best;
}

template <class E>
int by_dims(const pkv::PackedParams& p, int D, hipStream_t stream) {
    if (D == 64) {
        static constexpr Shape shapes[4] = {
            {32, 4, 2, 10, 10}, {64, 2, 4, 10, 10}, {128, 1, 5, 10, 10}, {32, 0.5, 16, 13.5, 7}};
        switch (best_shape(p, shapes)) {
            case 0: return launch<E, 64, 1, 4, 2, 1>(p, stream);
            case 1: return launch<E, 64, 2, 2, 2, 4>(p, stream);
            case 2: return launch<E, 64, 4, 1, 2, 5>(p, stream);
            default: return launch<E, 64, 1, 1, 1, 4>(p, stream);
        }
    }
    if (D == 128) {
        static constexpr Shape shapes[4] = {
            {32, 4, 2, 20, 20}, {64, 2, 2, 20, 20}, {128, 1, 3, 20, 20}, {32, 0.5, 9, 21, 14}};
        switch (best_shape(p, shapes)) {
            case 0: return launch<E, 128, 1, 4, 1, 2>(p, stream);
            case 1: return launch<E, 128, 2, 2, 2, 2>(p, stream);
            case 2: return launch<E, 128, 4, 1, 2, 3>(p, stream);
            default: return launch<E, 128, 1, 1, 1, 3>(p, stream);
        }
    }
    static constexpr Shape shapes[4] = {
        {32, 4, 1, 25, 25}, {64, 2, 1, 25, 25}, {128, 1, 2, 25, 25}, {32, 0.5, 4, 30.5, 30}};
    switch (best_shape(p, shapes)) {
        case 0: return launch<E, 256, 1, 4, 1, 1>(p, stream);
        case 1: return launch<E, 256, 2, 2, 2, 1>(p, stream);
        case 2: return launch<E, 256, 4, 1, 2, 2>(p, stream);
        default: return launch<E, 256, 1, 1, 1, 1>(p, stream);
    }
}

}  // namespace

extern "C" int pkv_attn_packed(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                               const void* v, int64_t v_row, int64_t v_head, const void* gate, int64_t gate_row,
                               int64_t gate_head, void* out, int64_t out_row, int64_t out_head, const int32_t* cu, int seqs,
                               int T, int Hq, int Hkv, int D, int dtype, float scale, void* stream) {
    if (T < 0 || seqs < 0 || Hq <= 0 || Hkv <= 0 || !(scale > 0.f) || !std::isfinite(scale)) return PKV_ERR_INVALID;
    if (Hq % Hkv != 0 || (D != 64 && D != 128 && D != 256) || (dtype != PKV_BF16 && dtype != PKV_FP16))
        return PKV_ERR_UNSUPPORTED;
    if (T == 0 || seqs == 0) return PKV_OK;
    if (!q || !k || !v || !out || !cu || !aligned(cu, 4)) return PKV_ERR_INVALID;
    // whole 16-byte pieces; K and V rows at 32-bit byte offsets inside a tile
    const int64_t strides[] = {q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, gate ? gate_row : 0,
                               gate ? gate_head : 0};
    for (int64_t s : strides)
        if (!stride_ok(s)) return PKV_ERR_INVALID;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(gate, 16))
        return PKV_ERR_INVALID;
    if (!apart(out_row, out_head, T, Hq, D)) return PKV_ERR_INVALID;
    if ((int64_t)T * (Hq / Hkv) > (int64_t)1 << 30) return PKV_ERR_UNSUPPORTED;
    pkv::PackedParams p;
    p.q = (const uint16_t*)q;
    p.k = (const uint16_t*)k;
    p.v = (const uint16_t*)v;
    p.gate = (const uint16_t*)gate;
    p.out = (uint16_t*)out;
    p.q_row = q_row, p.q_head = q_head, p.k_row = k_row, p.k_head = k_head, p.v_row = v_row, p.v_head = v_head;
    p.g_row = gate_row, p.g_head = gate_head, p.o_row = out_row, p.o_head = out_head;
    p.cu = cu;
    p.seqs = seqs, p.T = T, p.Hkv = Hkv, p.G = Hq / Hkv;
    int l = 0;
    while (((int64_t)1 << l) < p.G) l++;
    p.g_shift = 31 + l;
    p.g_mul = (uint32_t)(((uint64_t)1 << (31 + l)) / (uint32_t)p.G + 1);
    p.scale2 = scale * pkv::LOG2E;
    return dtype == PKV_BF16 ? by_dims<pkv::Bf16>(p, D, (hipStream_t)stream)
                             : by_dims<pkv::Fp16>(p, D, (hipStream_t)stream);
}
