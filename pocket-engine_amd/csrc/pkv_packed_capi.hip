// C-ABI entry point of the attention over packed prompts (include/pkv.h).
#include "pkv_packed.hip"
#include "pkv_entry.h"

#include <algorithm>
#include <cmath>

namespace {

// Tiles of RW rows that the batch can have: each sequence with rows rounds up once.
int64_t tile_bound(const pkv::PackedParams& p, int rw) {
    return ((int64_t)p.T * p.G + rw - 1) / rw + std::min(p.seqs, p.T);
}

template <class E, int D, int NQB, int KB, int NW, int NST, bool SPLIT, int OCC>
int launch(const pkv::PackedParams& p, hipStream_t stream) {
    using S = pkv::PackedTile<D, NQB, KB, NW, NST, SPLIT>;
    const int64_t grid = tile_bound(p, S::RW) * p.Hkv;
    if (grid * S::THREADS >= (int64_t)1 << 32) return PKV_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((pkv::packed_kernel<E, D, NQB, KB, NW, NST, SPLIT, OCC>), dim3((unsigned)grid), dim3(S::THREADS), 0,
                       stream, p);
    return launch_status();
}

template <class E>
int by_dims(const pkv::PackedParams& p, int D, hipStream_t stream) {
    if (tile_bound(p, 128) * p.Hkv < 128) {
        if (D == 64) return launch<E, 64, 1, 1, 4, 2, true, 1>(p, stream);
        if (D == 128) return launch<E, 128, 1, 1, 4, 1, true, 2>(p, stream);
        return launch<E, 256, 1, 1, 4, 1, true, 1>(p, stream);
    }
    if (D == 64) return launch<E, 64, 1, 1, 4, 2, false, 4>(p, stream);
    if (D == 128) return launch<E, 128, 1, 1, 4, 2, false, 3>(p, stream);
    return launch<E, 256, 1, 1, 4, 2, false, 2>(p, stream);
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
        if (s < 0 || s % 8 != 0 || s > ((int64_t)1 << 24)) return PKV_ERR_INVALID;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(gate, 16))
        return PKV_ERR_INVALID;
    // rows of their own for every token and head
    if ((T > 1 && out_row < D) || (Hq > 1 && out_head < D)) return PKV_ERR_INVALID;
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
    p.scale2 = scale * pkv::LOG2E;
    return dtype == PKV_BF16 ? by_dims<pkv::Bf16>(p, D, (hipStream_t)stream)
                             : by_dims<pkv::Fp16>(p, D, (hipStream_t)stream);
}
