// Internal interface of the chunk attention (dc_chunk.hip) and its planner
// (dc_abi.cpp).
#pragma once

#include "dc_decode.h"

namespace dc {

constexpr int kChunkRows = 256;   // query rows of a work item
constexpr int kChunkStep = 128;   // token ranges begin at multiples of this (a multiple of every tile)
constexpr int kChunkXcds = 8;     // consecutive blocks go to consecutive dies, each with an L2 of its own

// Rows of one item of the few-row kernel at most, by what its registers hold.
constexpr int few_row_limit(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 48 : 16; }

struct ChunkArgs {
  dc_pool kpool, vpool;
  const int32_t* k_table;
  const int32_t* v_table;
  int32_t table_stride;
  const dc_chunk_item* items;
  int32_t n_items, n_seqs, n_kv_heads, n_q;
  int64_t n_tokens;
  int32_t n_partials;
  const void* q;
  int64_t q_token_stride, q_head_stride;
  int32_t dtype;
  float scale;  // positive ...
  float sign;   // ... and what the queries are multiplied by: 1, -1, or 0 (scale 1)
  void* out;
  int64_t o_token_stride, o_head_stride;
  float* part_o;   // [n_partials][head_dim]
  float* part_ml;  // [n_partials][2]
  uint32_t page_mul, page_shift;
  int32_t q_vec, o_vec;  // rows start at multiples of 16 (8) bytes
};

// A work item outside the call's shapes is skipped, not read: a fault guard
// only (hosts validate plans).
__device__ __forceinline__ bool chunk_item_ok(const dc_chunk_item& it, const ChunkArgs& a) {
  return it.seq >= 0 && it.seq < a.n_seqs && it.kv_head >= 0 && it.kv_head < a.n_kv_heads && it.row_begin >= 0 &&
         it.row_begin < it.row_end && it.row_end - it.row_begin <= kChunkRows && it.q_begin >= 0 &&
         int64_t(it.q_begin) + (it.row_end - 1) / a.n_q < a.n_tokens && it.kv_begin >= 0 && it.first >= 0 &&
         int64_t(it.partial) + (it.partial >= 0 ? it.row_end - it.row_begin : 0) <= a.n_partials;
}

__device__ __forceinline__ bool chunk_merge_ok(const dc_chunk_merge& m, const ChunkArgs& a) {
  return m.kv_head >= 0 && m.kv_head < a.n_kv_heads && m.row_begin >= 0 && m.row_begin < m.row_end &&
         m.row_end - m.row_begin <= kChunkRows && m.q_begin >= 0 &&
         int64_t(m.q_begin) + (m.row_end - 1) / a.n_q < a.n_tokens && m.partial_begin >= 0 && m.count > 0 &&
         int64_t(m.partial_begin) + int64_t(m.count) * (m.row_end - m.row_begin) <= a.n_partials;
}

__device__ __forceinline__ void store_value(void* p, int32_t dtype, int64_t i, float x) {
  if (dtype == DC_F32)
    reinterpret_cast<float*>(p)[i] = x;
  else if (dtype == DC_F16)
    reinterpret_cast<_Float16*>(p)[i] = _Float16(x);
  else
    reinterpret_cast<__bf16*>(p)[i] = __bf16(x);
}

}  // namespace dc
