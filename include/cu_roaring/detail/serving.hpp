// Operators for serving language models, gated by bitmaps (no reference
// counterpart; the contracts are those of the cr_paged_* and cr_beam_* calls in
// cu_roaring_abi.h).  All are stream-ordered and do not synchronise; they throw
// std::runtime_error on failure.
#pragma once
#include <hip/hip_runtime_api.h>

#include "cu_roaring/types.hpp"

namespace cu_roaring {

// Keys and values of a paged cache, and the arguments of its attention.
using PagedCache = ::cr_paged_cache;
using PagedAttentionArgs = ::cr_paged_attention_args;
// The arguments of the calls for long and speculative answers.
using PagedRotaryArgs = ::cr_paged_rotary_args;
using PagedWeightsArgs = ::cr_paged_weights_args;
using PagedEvictArgs = ::cr_paged_evict_args;
using DraftVerifyArgs = ::cr_draft_verify_args;

// Block tables and slot maps from the requests' lengths; the pages come from the
// bitmap of free ones.
void paged_plan(const GpuRoaring& free_pages, uint32_t n_pages, uint32_t page_size, const int32_t* d_cached,
                const int32_t* d_new, uint32_t n_requests, int32_t* d_table, uint32_t table_cols,
                uint64_t table_stride, int64_t* d_slots, uint32_t slots_cap, int32_t* d_starts, int32_t* d_kv_len,
                int32_t* d_taken, uint32_t taken_cap, int32_t* d_counts, hipStream_t stream = 0);

// New keys and values into their slots.
void paged_append(const void* d_k, const void* d_v, uint64_t k_token_stride, uint64_t k_head_stride,
                  uint64_t v_token_stride, uint64_t v_head_stride, uint32_t n_tokens, const int64_t* d_slots,
                  const PagedCache& cache, hipStream_t stream = 0);

// The slots of each request that the bitmap `visible` holds.
void paged_select(const GpuRoaring& visible, uint32_t n_pages, uint32_t page_size, const int32_t* d_table,
                  uint32_t table_cols, uint64_t table_stride, const int32_t* d_starts, const int32_t* d_kv_len,
                  uint32_t n_requests, uint32_t n_tokens, int32_t* d_sel, uint64_t sel_stride, int32_t* d_sel_len,
                  int32_t* d_limits, hipStream_t stream = 0);

// Attention of the requests' new tokens over the cache.
void paged_attention(const PagedAttentionArgs& args, const PagedCache& cache, hipStream_t stream = 0);

// New keys and values into their slots, keys and queries turned by their positions.
void paged_rotary(const PagedRotaryArgs& args, const PagedCache& cache, hipStream_t stream = 0);

// The attention weights that the cached tokens got from the new ones.
void paged_weights(const PagedWeightsArgs& args, const PagedCache& cache, hipStream_t stream = 0);

// Which tokens of each request stay, and the moves that close the holes.
void paged_evict(const PagedEvictArgs& args, hipStream_t stream = 0);

// Keys and values from slot to slot.
void paged_move(const int32_t* d_moves, uint32_t moves_cap, uint64_t moves_stride, const int32_t* d_n_moves,
                uint32_t n_requests, const PagedCache& cache, hipStream_t stream = 0);

// Drafted tokens against the model's probabilities, and the token behind the
// accepted ones.
void draft_verify(const DraftVerifyArgs& args, hipStream_t stream = 0);

// The k best continuations of each answer's beams; `allowed` (nullptr: every
// token) or d_allowed_bits say which tokens may follow.
void beam_select(const void* d_scores, uint32_t dtype, uint32_t batch, uint32_t beams, uint32_t vocab,
                 uint64_t batch_stride, uint64_t beam_stride, const float* d_cum, const float* d_lse,
                 const GpuRoaring* allowed, const uint32_t* d_allowed_bits, uint64_t bits_stride, uint32_t k,
                 float* d_out_scores, int32_t* d_out_tokens, int32_t* d_out_parents, hipStream_t stream = 0);

// The beams' states after it.
void beam_reorder(const void* d_src, const int32_t* d_parents, uint32_t batch, uint32_t beams_in, uint32_t beams_out,
                  uint64_t row_bytes, uint64_t src_stride, uint64_t dst_stride, const int32_t* d_len,
                  uint64_t unit_bytes, void* d_dst, hipStream_t stream = 0);

}  // namespace cu_roaring
