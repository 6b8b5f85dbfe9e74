// Entry points of the chunk attention and the join of split ranges
// (dc_attend_chunk; kernels in dc_chunk_kernels.h).
#include "dc_chunk_kernels.h"

namespace dc {

// Joins the partial results of a row tile's token ranges: `lanes` lanes per
// row, VEC channels a lane and further ones in turn, kMergeBatch ranges' results
// in flight at once (their weights follow from running maxima, so that nothing
// is read twice).  Where a range of few rows was cut into many (kMergeMany), the
// block's lane groups share a row's partial results and join in LDS; otherwise
// each group has a row of its own.
constexpr int kMergeBlocks = 64, kMergeMany = 8, kMergeBatch = 4;

template <int VEC>
__global__ void __launch_bounds__(256) merge_chunk_kernel(ChunkArgs a, const dc_chunk_merge* merges, int32_t lanes) {
  __shared__ float joined[256 * VEC];
  __shared__ float sums[256], tops[256];
  const dc_chunk_merge mg = merges[blockIdx.x];
  if (!chunk_merge_ok(mg, a)) return;
  const int tid = threadIdx.x, groups = 256 / lanes, group = tid / lanes, lane = tid - group * lanes;
  const bool many = mg.count >= kMergeMany;  // (uniform)
  const int split = many ? groups : 1, part = many ? group : 0, per_block = many ? 1 : groups;
  const int hd = a.kpool.geometry.head_dim, rows = mg.row_end - mg.row_begin;
  for (int r0 = int(blockIdx.y) * per_block; r0 < rows; r0 += int(gridDim.y) * per_block) {  // (uniform)
    const int r = r0 + (many ? 0 : group), row = mg.row_begin + r;
    const bool has = r < rows;  // (the others take part in the barriers)
    const int64_t first = int64_t(mg.partial_begin) + (has ? r : 0);
    const int tok = row / a.n_q, head = mg.kv_head * a.n_q + (row - tok * a.n_q);
    const int64_t off = int64_t(mg.q_begin + tok) * a.o_token_stride + int64_t(head) * a.o_head_stride;
    for (int c0 = 0; c0 < hd; c0 += VEC * lanes) {
      const int ch = c0 + VEC * lane;
      const bool in = ch < hd;
      float sum[VEC], l = 0.f, top = -INFINITY;
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
      for (int i0 = part; i0 < mg.count; i0 += split * kMergeBatch) {
        float2 ml[kMergeBatch];
        float x[kMergeBatch][VEC];
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j) {
          const int i = i0 + j * split;
          const int64_t at = first + int64_t(i < mg.count ? i : i0) * rows;
          ml[j] = float2{a.part_ml[2 * at], a.part_ml[2 * at + 1]};  // (an odd head_dim: at any 4 bytes)
          const float* po = a.part_o + at * hd + (in ? ch : 0);
          if constexpr (VEC == 4) {
            const float4 v = *reinterpret_cast<const float4*>(po);
            x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
          } else {
            x[j][0] = *po;
          }
        }
        float high = top;
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j) high = fmaxf(high, ml[j].x);  // (a repeated result changes no maximum)
        const float mu = high == -INFINITY ? 0.f : high;
        if (high > top) {
          const float f = __builtin_amdgcn_exp2f(top - mu);
          l = top == -INFINITY ? 0.f : l * f;
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] = top == -INFINITY ? sum[k] : sum[k] * f;
          top = high;
        }
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j) {
          if (j > 0 && i0 + j * split >= mg.count) break;
          const float w = __builtin_amdgcn_exp2f(ml[j].x - mu);
          l = fmaf(w, ml[j].y, l);
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] = fmaf(w, x[j][k], sum[k]);
        }
      }
      if (many) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) joined[VEC * tid + k] = sum[k];
        sums[tid] = l;
        tops[tid] = top;
        __syncthreads();
        if (part == 0) {
          float high = top;
          for (int p = 1; p < split; ++p) high = fmaxf(high, tops[tid + p * lanes]);
          const float mu = high == -INFINITY ? 0.f : high, f = __builtin_amdgcn_exp2f(top - mu);
          l *= f;
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] *= f;
          for (int p = 1; p < split; ++p) {
            const int t = tid + p * lanes;
            const float w = __builtin_amdgcn_exp2f(tops[t] - mu);
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] = fmaf(w, joined[VEC * t + k], sum[k]);
            l = fmaf(w, sums[t], l);
          }
        }
      }
      if (!has || !in || part != 0) continue;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int k = 0; k < VEC; ++k) store_value(a.out, a.dtype, off + ch + k, sum[k] * inv);
    }
  }
}

// `rows`: of a merge at most.
static int launch_merge_chunk(const ChunkArgs& a, const dc_chunk_merge* merges, int32_t n_merges, int32_t rows, hipStream_t stream) {
  const int hd = a.kpool.geometry.head_dim;
  const bool vec = hd % 4 == 0;
  const int lanes = vec && hd <= 64 ? 16 : vec && hd <= 128 ? 32 : 64;
  const dim3 grid(uint32_t(n_merges), uint32_t(rows < kMergeBlocks ? rows : kMergeBlocks));
  if (vec)
    hipLaunchKernelGGL((merge_chunk_kernel<4>), grid, dim3(256), 0, stream, a, merges, lanes);
  else
    hipLaunchKernelGGL((merge_chunk_kernel<1>), grid, dim3(256), 0, stream, a, merges, lanes);
  return check_hip(hipGetLastError(), "merge_chunk_kernel launch");
}

// Whether a thread's 32 channels share a scale and lie at 16-byte multiples,
// with offsets in a blob that fit 32 bits, in the formats that load_unit takes.
static bool units32(const dc_pool& p) {
  const dc_page_geometry& g = p.geometry;
  uint64_t takes = uint64_t(1) << (DC_FMT_M3_F16 * 9);
  for (int f : {DC_FMT_M0_AFFINE, DC_FMT_M0_SYMMETRIC})
    for (int bits : {4, 8}) takes |= uint64_t(1) << (f * 9 + bits);
  return p.format_mask != 0 && (p.format_mask & ~takes) == 0 && g.head_dim % 32 == 0 && g.group_size % 32 == 0 && chunk16_geometry(g);
}

// How the checks of both entry points and their launches go; `rule` null: plain causal attention.
static int attend_chunk(const char* who, dc_pool k_pool, dc_pool v_pool, const int32_t* k_table, const int32_t* v_table,
                        int32_t table_stride, const dc_chunk_item* items, int32_t n_items, int32_t n_few, int32_t few_rows,
                        const dc_chunk_merge* merges, int32_t n_merges, int32_t n_partials, int32_t n_seqs, int32_t n_kv_heads,
                        int64_t n_tokens, dc_token_rows q, float query_scale, const dc_score_rule* rule, dc_token_rows out,
                        void* workspace, int64_t workspace_bytes, dc_stream_t stream) {
  if (int rc = validate_geometry(k_pool.geometry)) return rc;
  if (int rc = validate_geometry(v_pool.geometry)) return rc;
  const int hd = k_pool.geometry.head_dim;
  if (v_pool.geometry.head_dim != hd || v_pool.geometry.page_capacity != k_pool.geometry.page_capacity)
    return fail(DC_EINVAL, "%s: key and value pools must share head_dim and page_capacity", who);
  if (hd > 256) return fail(DC_EINVAL, "%s: head_dim above 256", who);
  if (n_few < 0 || n_few > n_items || (n_few && (few_rows <= 0 || few_rows > few_row_limit(hd))))
    return fail(DC_EINVAL, "%s: n_few must lie in [0, n_items], their rows in [1, %d]", who, few_row_limit(hd));
  if (n_items < 0 || n_merges < 0 || n_partials < 0 || n_seqs <= 0 || n_kv_heads <= 0 || n_tokens < 0 || table_stride <= 0)
    return fail(DC_EINVAL, "%s: bad counts", who);
  if (n_items == 0) return DC_OK;
  if (!k_pool.arena || !v_pool.arena || !k_pool.descs || !v_pool.descs || !k_table || !v_table || !items || !q.data || !out.data ||
      (n_merges && !merges))
    return fail(DC_EINVAL, "%s: null pointer", who);
  if (q.dtype != DC_F32 && q.dtype != DC_F16 && q.dtype != DC_BF16) return fail(DC_EINVAL, "%s: queries must be DC_F32, DC_F16 or DC_BF16", who);
  if (out.dtype != q.dtype || out.n_heads != q.n_heads || q.n_heads <= 0 || q.n_heads % n_kv_heads)
    return fail(DC_EINVAL, "%s: the output needs the queries' dtype and heads, a multiple of the KV heads", who);
  if (workspace_bytes < dc_chunk_workspace_bytes(n_partials, hd) || (n_partials && !workspace))
    return fail(DC_ESPACE, "%s: workspace too small", who);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(DC_EINVAL, "%s: workspace must be 16-byte aligned", who);
  if (rule && !(rule->cap >= 0.f)) return fail(DC_EINVAL, "%s: cap must be positive, or 0 for none", who);
  if (rule && (reinterpret_cast<uintptr_t>(rule->ranges) % 16 || reinterpret_cast<uintptr_t>(rule->gaps) % 8))
    return fail(DC_EINVAL, "%s: ranges must be 16-byte aligned, gaps 8-byte", who);
  if (rule && rule->gaps && !rule->ranges) return fail(DC_EINVAL, "%s: gaps are those of ranges", who);
  ChunkArgs a{k_pool, v_pool, k_table, v_table, table_stride, items, n_items, n_seqs, n_kv_heads, q.n_heads / n_kv_heads,
                  n_tokens, n_partials, q.data, q.token_stride, q.head_stride, q.dtype,
                  query_scale == 0.f ? 1.f : fabsf(query_scale), query_scale > 0.f ? 1.f : query_scale < 0.f ? -1.f : 0.f, out.data, out.token_stride,
              out.head_stride, static_cast<float*>(workspace), static_cast<float*>(workspace) + int64_t(n_partials) * hd};
  const hipStream_t st = hipStream_t(stream);
  a.q_vec = reinterpret_cast<uintptr_t>(q.data) % 16 == 0 && q.token_stride % 8 == 0 && q.head_stride % 8 == 0;
  a.o_vec = reinterpret_cast<uintptr_t>(out.data) % 8 == 0 && out.token_stride % 4 == 0 && out.head_stride % 4 == 0;
  // u / page_capacity = u * page_mul >> page_shift for u < 2^31
  const uint32_t P = uint32_t(k_pool.geometry.page_capacity);
  a.page_shift = 31;
  while ((1u << (a.page_shift - 31)) < P) ++a.page_shift;
  a.page_mul = uint32_t(((uint64_t(1) << a.page_shift) + P - 1) / P);
  if (rule) {
    a.cap = rule->cap * kLog2e;
    a.cap_in = rule->cap > 0.f ? float(2.0 * a.scale * kLog2e / rule->cap) : 0.f;
    a.slopes = rule->slopes;
    a.ranges = reinterpret_cast<const int4*>(rule->ranges);
    a.gaps = reinterpret_cast<const int2*>(rule->gaps);
    if (!(a.cap <= 3e38f && a.cap_in <= 3e38f)) return fail(DC_EINVAL, "%s: cap is out of range for the scale", who);
  }
  const bool units = q.dtype != DC_F32 && units32(k_pool) && units32(v_pool);
  const auto launch = !rule ? launch_chunks : rule->cap > 0.f ? launch_chunks_cap : launch_chunks_rule;
  if (int rc = launch(a, n_few, few_rows, units, st)) return rc;
  // (items of few rows alone: blocks for those rows)
  return n_merges ? launch_merge_chunk(a, merges, n_merges, n_few == n_items ? few_rows : kMergeBlocks, st) : DC_OK;
}

int launch_chunks(ChunkArgs a, int32_t n_few, int32_t few_rows, bool units, hipStream_t stream) {
  return launch_all<kCausal>(a, n_few, few_rows, units, stream);
}

}  // namespace dc

extern "C" int dc_attend_chunk(dc_pool k_pool, dc_pool v_pool, const int32_t* k_table, const int32_t* v_table,
                               int32_t table_stride, const dc_chunk_item* items, int32_t n_items, int32_t n_few, int32_t few_rows,
                               const dc_chunk_merge* merges, int32_t n_merges, int32_t n_partials, int32_t n_seqs,
                               int32_t n_kv_heads, int64_t n_tokens, dc_token_rows q, float query_scale, dc_token_rows out,
                               void* workspace, int64_t workspace_bytes, dc_stream_t stream) {
  return dc::attend_chunk("dc_attend_chunk", k_pool, v_pool, k_table, v_table, table_stride, items, n_items, n_few, few_rows, merges,
                          n_merges, n_partials, n_seqs, n_kv_heads, n_tokens, q, query_scale, nullptr, out, workspace, workspace_bytes,
                          stream);
}

extern "C" int dc_attend_chunk_rule(dc_pool k_pool, dc_pool v_pool, const int32_t* k_table, const int32_t* v_table,
                                    int32_t table_stride, const dc_chunk_item* items, int32_t n_items, int32_t n_few, int32_t few_rows,
                                    const dc_chunk_merge* merges, int32_t n_merges, int32_t n_partials, int32_t n_seqs,
                                    int32_t n_kv_heads, int64_t n_tokens, dc_token_rows q, float query_scale, dc_score_rule rule,
                                    dc_token_rows out, void* workspace, int64_t workspace_bytes, dc_stream_t stream) {
  return dc::attend_chunk("dc_attend_chunk_rule", k_pool, v_pool, k_table, v_table, table_stride, items, n_items, n_few, few_rows,
                          merges, n_merges, n_partials, n_seqs, n_kv_heads, n_tokens, q, query_scale, &rule, out, workspace,
                          workspace_bytes, stream);
}
