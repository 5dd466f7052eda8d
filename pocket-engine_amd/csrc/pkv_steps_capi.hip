// C-ABI entry points of the steps planned on the GPU and of the rotary
// positions and rows (include/pkv.h). As elsewhere every shape is checked on
// the host before a launch.
#include "pkv_plan.hip"
#include "pkv_rope.hip"
#include "pkv_entry.h"

#include <algorithm>

namespace {

constexpr int64_t INT_LIMIT = 0x7fffffff;

// Slots, limits and ids in 32 bits, and sums that saturate below 2^30.
int plan_sizes(int nrows, int max_blocks, int block_size, int64_t num_blocks) {
    if (nrows < 0 || max_blocks <= 0 || block_size <= 0 || num_blocks <= 0) return PKV_ERR_INVALID;
    if (num_blocks * block_size > INT_LIMIT || (int64_t)max_blocks * block_size > INT_LIMIT || num_blocks >= (1 << 29))
        return PKV_ERR_UNSUPPORTED;
    return PKV_OK;
}

bool words(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!p || !aligned(p, 4)) return false;
    return true;
}

bool strides_ok(std::initializer_list<int64_t> ss) {
    for (int64_t s : ss)
        if (!stride_ok(s)) return false;
    return true;
}

template <class E, int D, bool ADJ>
void launch_rope(const pkv::RopeParams& p, hipStream_t stream) {
    // Tokens a workgroup: as many as give its threads two and a half (token,
    // head) pairs each, while that leaves 2,048 workgroups.
    int tb = 1;
    while (tb < pkv::rope_tokens(D) && 2 * tb * (p.Hq + p.Hkv) * D <= 10240 && p.T / (2 * tb) >= 2048) tb *= 2;
    // Stores that leave no lines behind, where the rows pass what the caches keep
    // for their reader: 16,384 rows at 32 / 8 heads of 128 (168 MB) 65 -> 52 us,
    // with the attention over 16 prompts of them 244 -> 246. Below, the reader
    // loses more than the writer gains: 4,096 rows 44.5 -> 45.5 us with theirs.
    const bool large = (int64_t)p.T * (p.Hq + p.Hkv) * D * 2 > 160000000;
    const auto kernel = large ? pkv::rope_rows_kernel<E, D, ADJ, true> : pkv::rope_rows_kernel<E, D, ADJ, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.T - 1) / tb + 1)), dim3(256), 0, stream, p, tb);
}
template <class E, bool ADJ>
void rope_by_dims(const pkv::RopeParams& p, int D, hipStream_t stream) {
    if (D == 64) launch_rope<E, 64, ADJ>(p, stream);
    else if (D == 128) launch_rope<E, 128, ADJ>(p, stream);
    else launch_rope<E, 256, ADJ>(p, stream);
}

}  // namespace

extern "C" {

int pkv_plan_step(const int32_t* len, const int32_t* held, const int32_t* ntok, int nrows, int32_t* block_table,
                  int max_blocks, int block_size, int64_t num_blocks, const int32_t* free_list,
                  const int32_t* free_count, int T, int32_t* pos, int32_t* slot_map, int32_t* tok_seq, int32_t* cu,
                  int32_t* limits, int32_t* len_out, int32_t* held_out, int32_t* free_count_out, int32_t* status,
                  void* stream) {
    if (T < 0) return PKV_ERR_INVALID;
    const int st = plan_sizes(nrows, max_blocks, block_size, num_blocks);
    if (st != PKV_OK) return st;
    if (T >= (1 << 29)) return PKV_ERR_UNSUPPORTED;
    if (!words({cu}) || (nrows > 0 && !words({len, held, ntok, block_table, limits, len_out, held_out, status})) ||
        (T > 0 && !words({pos, slot_map, tok_seq})))
        return PKV_ERR_INVALID;
    // a free list with its count, or neither
    if ((free_list == nullptr) != (free_count == nullptr) || (free_list && !words({free_list, free_count})) ||
        (free_count_out && (!free_list || !aligned(free_count_out, 4))))
        return PKV_ERR_INVALID;
    pkv::PlanParams p;
    p.len = len, p.held = held, p.ntok = ntok, p.nrows = nrows;
    p.table = block_table, p.max_blocks = max_blocks, p.block_size = block_size, p.num_blocks = (int)num_blocks;
    p.free_list = free_list, p.free_count = free_count, p.T = T;
    p.pos = pos, p.slot_map = slot_map, p.tok_seq = tok_seq, p.cu = cu, p.limits = limits;
    p.len_out = len_out, p.held_out = held_out, p.free_out = free_count_out, p.status = status;
    // 256 threads where they hold the rows and, one workgroup, the tokens and
    // pages in two turns (64 rows 6.9 -> 4.2 us; but 256 rows with 127,000 tokens in
    // place 30 -> 15 with 1,024).
    const bool in_place = len_out == len || held_out == held || (free_count_out && free_count_out == free_count);
    const bool one = in_place && (T <= 2048 || nrows == 0), small = nrows <= 256 && (!in_place || T <= 512);
    const int threads = small ? 256 : 1024;
    const dim3 grid(in_place ? 1 : std::max(1, std::min(256, (T + threads - 1) / threads)));
    const hipStream_t hs = (hipStream_t)stream;
    if (one || !in_place) {
        hipLaunchKernelGGL((small ? pkv::plan_rows_kernel<true, 4> : pkv::plan_rows_kernel<true, 16>), grid, dim3(threads), 0,
                           hs, p);
        return launch_status();
    }
    hipLaunchKernelGGL((small ? pkv::plan_rows_kernel<false, 4> : pkv::plan_rows_kernel<false, 16>), grid, dim3(threads), 0,
                       hs, p);
    const int s = launch_status();
    if (s != PKV_OK) return s;
    hipLaunchKernelGGL(pkv::plan_tokens_kernel, dim3((T + 255) / 256), dim3(256), 0, (hipStream_t)stream, p);
    return launch_status();
}

int pkv_plan_truncate(const int32_t* new_len, int32_t* len, int32_t* held, int nrows, const int32_t* block_table,
                      int max_blocks, int block_size, int64_t num_blocks, int32_t* free_list, int32_t* free_count,
                      void* stream) {
    const int st = plan_sizes(nrows, max_blocks, block_size, num_blocks);
    if (st != PKV_OK || nrows == 0) return st;
    if (!words({new_len, len, held, block_table, free_list, free_count})) return PKV_ERR_INVALID;
    pkv::TruncateParams p;
    p.new_len = new_len, p.len = len, p.held = held, p.nrows = nrows;
    p.table = block_table, p.max_blocks = max_blocks, p.block_size = block_size, p.num_blocks = (int)num_blocks;
    p.free_list = free_list, p.free_count = free_count;
    hipLaunchKernelGGL(pkv::plan_truncate_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
    return launch_status();
}

int pkv_rope_spans(const int32_t* span_cu, const int32_t* spans, int n_req, int n_spans, int32_t* base, void* stream) {
    if (n_req < 0 || n_spans < 0) return PKV_ERR_INVALID;
    if (n_req == 0 || n_spans == 0) return PKV_OK;
    if (!words({span_cu, spans, base})) return PKV_ERR_INVALID;
    hipLaunchKernelGGL(pkv::rope_spans_kernel<4>, dim3(n_req), dim3(256), 0, (hipStream_t)stream, span_cu, spans, n_spans,
                       base);
    return launch_status();
}

int pkv_rope_positions(const int32_t* pos, const int32_t* tok_seq, int T, const int32_t* span_cu, const int32_t* spans,
                       const int32_t* base, int n_req, int n_spans, int32_t* rope, int rope_stride, void* stream) {
    if (T < 0 || n_req < 0 || n_spans < 0 || rope_stride < T) return PKV_ERR_INVALID;
    if (T == 0) return PKV_OK;
    if (!words({pos, tok_seq, rope}) || (n_req > 0 && !words({span_cu})) || (n_spans > 0 && !words({spans, base})))
        return PKV_ERR_INVALID;
    hipLaunchKernelGGL(pkv::rope_positions_kernel, dim3((T - 1) / 256 + 1), dim3(256), 0, (hipStream_t)stream, pos, tok_seq,
                       span_cu, spans, base, n_req, n_spans, T, rope, rope_stride);
    return launch_status();
}

int pkv_rope_rows(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                  void* q_out, int64_t q_out_row, int64_t q_out_head, void* k_out, int64_t k_out_row,
                  int64_t k_out_head, int Hq, int Hkv, int D, int dtype, const float* q_norm, const float* k_norm,
                  float eps, const int32_t* rope, int rope_stride, const int32_t* axes, const float* inv_freq, int rot,
                  int adjacent, int T, void* stream) {
    if (T < 0 || Hq < 0 || Hkv < 0 || rot < 0 || rope_stride < 0) return PKV_ERR_INVALID;
    if ((D != 64 && D != 128 && D != 256) || (dtype != PKV_BF16 && dtype != PKV_FP16) || rot % 16 != 0 || rot > D ||
        Hq > (1 << 20) || Hkv > (1 << 20))
        return PKV_ERR_UNSUPPORTED;
    if (T == 0 || Hq + Hkv == 0) return PKV_OK;
    if (Hq > 0 && (!q || !q_out || !aligned(q, 16) || !aligned(q_out, 16) ||
                   !strides_ok({q_row, q_head, q_out_row, q_out_head}) || !apart(q_out_row, q_out_head, T, Hq, D)))
        return PKV_ERR_INVALID;
    if (Hkv > 0 && (!k || !k_out || !aligned(k, 16) || !aligned(k_out, 16) ||
                    !strides_ok({k_row, k_head, k_out_row, k_out_head}) ||
                    !apart(k_out_row, k_out_head, T, Hkv, D)))
        return PKV_ERR_INVALID;
    if (rot > 0 && (!words({rope, axes, inv_freq}) || rope_stride < T)) return PKV_ERR_INVALID;
    if (!aligned(q_norm, 4) || !aligned(k_norm, 4)) return PKV_ERR_INVALID;
    pkv::RopeParams p;
    p.q = (const uint16_t*)q, p.k = (const uint16_t*)k, p.q_out = (uint16_t*)q_out, p.k_out = (uint16_t*)k_out;
    p.q_row = q_row, p.q_head = q_head, p.k_row = k_row, p.k_head = k_head;
    p.qo_row = q_out_row, p.qo_head = q_out_head, p.ko_row = k_out_row, p.ko_head = k_out_head;
    p.q_norm = q_norm, p.k_norm = k_norm, p.rope = rope, p.rope_stride = rope_stride, p.axes = axes;
    p.inv_freq = inv_freq, p.Hq = Hq, p.Hkv = Hkv, p.half = rot / 2, p.T = T, p.eps = eps;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == PKV_BF16)
        adjacent ? rope_by_dims<pkv::Bf16, true>(p, D, s) : rope_by_dims<pkv::Bf16, false>(p, D, s);
    else
        adjacent ? rope_by_dims<pkv::Fp16, true>(p, D, s) : rope_by_dims<pkv::Fp16, false>(p, D, s);
    return launch_status();
}

}  // extern "C"
