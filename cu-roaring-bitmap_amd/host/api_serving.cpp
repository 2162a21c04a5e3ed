// Host C++ API of the operators for serving language models (namespace
// cu_roaring) over the C ABI: each call forwards to the matching cr_* entry
// point and throws std::runtime_error on failure.
#include "cu_roaring/cu_roaring.hpp"

namespace cu_roaring {

static cr_stream_t S(hipStream_t s) { return reinterpret_cast<cr_stream_t>(s); }

void paged_plan(const GpuRoaring& free_pages, uint32_t n_pages, uint32_t page_size, const int32_t* d_cached,
                const int32_t* d_new, uint32_t n_requests, int32_t* d_table, uint32_t table_cols,
                uint64_t table_stride, int64_t* d_slots, uint32_t slots_cap, int32_t* d_starts, int32_t* d_kv_len,
                int32_t* d_taken, uint32_t taken_cap, int32_t* d_counts, hipStream_t stream)
{
    throw_on_error(cr_paged_plan(to_abi(&free_pages), n_pages, page_size, d_cached, d_new, n_requests, d_table,
                                 table_cols, table_stride, d_slots, slots_cap, d_starts, d_kv_len, d_taken, taken_cap,
                                 d_counts, S(stream)),
                   "paged_plan");
}

void paged_append(const void* d_k, const void* d_v, uint64_t k_token_stride, uint64_t k_head_stride,
                  uint64_t v_token_stride, uint64_t v_head_stride, uint32_t n_tokens, const int64_t* d_slots,
                  const PagedCache& cache, hipStream_t stream)
{
    throw_on_error(cr_paged_append(d_k, d_v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, n_tokens,
                                   d_slots, &cache, S(stream)),
                   "paged_append");
}

void paged_select(const GpuRoaring& visible, uint32_t n_pages, uint32_t page_size, const int32_t* d_table,
                  uint32_t table_cols, uint64_t table_stride, const int32_t* d_starts, const int32_t* d_kv_len,
                  uint32_t n_requests, uint32_t n_tokens, int32_t* d_sel, uint64_t sel_stride, int32_t* d_sel_len,
                  int32_t* d_limits, hipStream_t stream)
{
    throw_on_error(cr_paged_select(to_abi(&visible), n_pages, page_size, d_table, table_cols, table_stride, d_starts,
                                   d_kv_len, n_requests, n_tokens, d_sel, sel_stride, d_sel_len, d_limits, S(stream)),
                   "paged_select");
}

void paged_attention(const PagedAttentionArgs& args, const PagedCache& cache, hipStream_t stream)
{
    throw_on_error(cr_paged_attention(&args, &cache, S(stream)), "paged_attention");
}

void beam_select(const void* d_scores, uint32_t dtype, uint32_t batch, uint32_t beams, uint32_t vocab,
                 uint64_t batch_stride, uint64_t beam_stride, const float* d_cum, const float* d_lse,
                 const GpuRoaring* allowed, const uint32_t* d_allowed_bits, uint64_t bits_stride, uint32_t k,
                 float* d_out_scores, int32_t* d_out_tokens, int32_t* d_out_parents, hipStream_t stream)
{
    throw_on_error(cr_beam_select(d_scores, dtype, batch, beams, vocab, batch_stride, beam_stride, d_cum, d_lse,
                                  allowed ? to_abi(allowed) : nullptr, d_allowed_bits, bits_stride, k, d_out_scores,
                                  d_out_tokens, d_out_parents, S(stream)),
                   "beam_select");
}

void beam_reorder(const void* d_src, const int32_t* d_parents, uint32_t batch, uint32_t beams_in, uint32_t beams_out,
                  uint64_t row_bytes, uint64_t src_stride, uint64_t dst_stride, const int32_t* d_len,
                  uint64_t unit_bytes, void* d_dst, hipStream_t stream)
{
    throw_on_error(cr_beam_reorder(d_src, d_parents, batch, beams_in, beams_out, row_bytes, src_stride, dst_stride,
                                   d_len, unit_bytes, d_dst, S(stream)),
                   "beam_reorder");
}

}  // namespace cu_roaring
