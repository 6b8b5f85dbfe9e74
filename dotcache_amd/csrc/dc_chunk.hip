// Attention of a chunk of new tokens of every sequence over its compressed
// pages (dc_attend_chunk): prompt chunks, drafted tokens and decodes of one
// batch in one launch, causal among the new tokens.
//
//   o_r = sum_u p_ru v_u / sum_u p_ru,  p_ru = exp(scale q_r . k_u),  u <= last token that row r sees
//
// A work item is a tile of 128 query rows (token-major, the n_q heads of a KV
// head next to each other, so they share every key and value) of one
// (sequence, KV head) against a range of its tokens.  Four wavefronts of 32
// rows each walk the range in tiles of KT tokens: the block turns a tile's
// page rows into dense rows in LDS once, for all 128 query rows, and every
// wavefront then takes
//   S^T = K Q^T   tokens x rows, so a lane holds one row's logits and the
//                 softmax needs one exchange between the two half-wavefronts;
//   O^T += V^T P^T  with P in the registers it was computed in: the matrix
//                 instruction's k index runs over the tokens in the order in
//                 which S^T left them, and V's operand is read in that order.
// The running maximum moves only when a tile's exceeds it by 2^kLazy, so that
// rescaling the output is rare; sums and the output are fp32.
#include "dc_chunk.h"
#include "dc_unpack.h"

namespace dc {

namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLazy = 8.f;  // log2 of how far a weight may pass 1 before the maximum moves

// Byte offset of 16-byte chunk ch of token t's row in an LDS tile whose rows
// have CH chunks.  Chunks are exchanged within a row so that reads of one
// chunk of 16 consecutive tokens (keys), of four chunks of four consecutive
// tokens (values, transposed) and the writes of 16 tokens each touch every
// bank once.
template <int CH>
__device__ __forceinline__ int lds_at(int t, int ch) {
  const int x = CH >= 16 ? ((t & 3) << 2) | ((t >> 2) & 3) : (((t >> 1) & 1) << 2) | ((t >> 2) & 3);
  return (t * CH + (ch ^ x)) * 16;
}

// This lane's value and that of lane ^ 32 (in one order or the other).
__device__ __forceinline__ float2 both_halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t x = r[0], y = r[1];  // (bit casts of vector elements would all take the first)
  return float2{__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float half_max(float v) {
  const float2 b = both_halves(v);
  return fmaxf(b.x, b.y);
}
__device__ __forceinline__ float half_sum(float v) {
  const float2 b = both_halves(v);
  return b.x + b.y;
}

// Sixteen channels from c0 of slot t of a page as fp32 (zeros past head_dim).
__device__ __forceinline__ void page_values16(const dc_pool& pool, const dc_page_desc& d, int t, int c0, bool chunks,
                                              float (&v)[16]) {
  const dc_page_geometry& geo = pool.geometry;
  const uint8_t* blob = blob_ptr(pool.arena, d);
  if (chunks) {  // (uniform)
    const Blob32 L = blob32(d.format, d.bits, geo, num_groups(geo));
    const Chunk16 ck = chunk16_at(d.format, d.bits, geo, L, c0);
    for_chunk_kind(chunk_kind(d.format, d.bits), [&](auto kind) __attribute__((always_inline)) {
      constexpr int K = decltype(kind)::value;
      uint32_t r[16];
      load_chunk16(K, blob + t * ck.word_step + ck.word(), r);
      float s = 1.f, b = 0.f;
      if constexpr (K != CK_F16 && K != CK_F32) {
        constexpr float zp = K == CK_B2 ? -1.f : K == CK_B3 ? -3.f : K == CK_B4 ? -7.f : K == CK_B8 ? -127.f : 0.f;
        s = half_bits(*reinterpret_cast<const uint16_t*>(blob + t * ck.scale_step + ck.scale), 0);
        b = d.format == DC_FMT_M0_AFFINE ? half_bits(*reinterpret_cast<const uint16_t*>(blob + t * ck.scale_step + ck.bias), 0)
            : K == CK_I8                 ? 0.f
                                         : zp * s;
      }
      values16<K>(r, ck.shift(), s, b, v);
    });
    return;
  }
  const BlobLayout L = blob_layout(d.format, d.bits, geo);
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const float x = c0 + i < geo.head_dim ? page_value(blob, d, L, geo, t, c0 + i) : 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = k == i ? x : v[k];
  }
}

}  // namespace

// T: the matrix operands, _Float16 or float.  HDP: head_dim rounded up to the
// operands' rows (channels past head_dim are zeros).  KT: tokens per tile.
template <typename T, int HDP, int KT>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && HDP == 256 ? 1 : 2) attend_chunk_kernel(ChunkArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int CH = HDP * int(sizeof(T)) / 16;  // 16-byte chunks of a row
  constexpr int TB = KT / 32, CB = HDP / 32;     // 32-token and 32-channel blocks
  constexpr int TILE = KT * HDP * int(sizeof(T));
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  uint8_t* const kt = lds;
  uint8_t* const vt = lds + TILE;
  __shared__ uint32_t live[TB];    // one bit per token: it counts
  __shared__ uint32_t poison[TB];  // it has a value that is not finite (in a tile that some row does not see whole)
  __shared__ float odd[HDP];       // such a token's values

  const dc_chunk_item it = a.items[blockIdx.x];
  if (!chunk_item_ok(it, a)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hd = a.kpool.geometry.head_dim, P = a.kpool.geometry.page_capacity;

  // this lane's query row
  const int row = it.row_begin + 32 * wave + col;
  const bool wave_rows = it.row_begin + 32 * wave < it.row_end;  // (uniform)
  const bool has_row = row < it.row_end;
  const int tok = row / a.n_q, head = it.kv_head * a.n_q + (row - tok * a.n_q);
  const int sees = has_row ? it.first + tok : -1;                        // last token this row attends
  const int sees_all = it.first + (it.row_begin + 32 * wave) / a.n_q;    // and the least of the wavefront's rows

  // Q as the B operand: row col, channels 16 ks + 8 half .. + 7 (F32: 8 ks + 4 half .. + 3)
  constexpr int QW = F32 ? HDP / 8 : HDP / 16;
  typedef std::conditional_t<F32, float4, h8v> QV;
  QV q[QW];
  {
    const int64_t off = int64_t(it.q_begin + tok) * a.q_token_stride + int64_t(head) * a.q_head_stride;
#pragma unroll
    for (int i = 0; i < QW; ++i) {
      constexpr int W = F32 ? 4 : 8;
      const int c = 2 * W * i + W * half;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float x = has_row && c + k < hd ? load_value(a.q, a.dtype, off + c + k) : 0.f;
        if constexpr (F32)
          (&q[i].x)[k] = x;
        else
          q[i][k] = _Float16(x);
      }
    }
  }
  const float c = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;  // maximum (of scaled log2 logits), sum of this half's weights
  f32x16 o[CB];
#pragma unroll
  for (int i = 0; i < CB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[i][v] = 0.f;

  const bool k_chunks = chunk16_geometry(a.kpool.geometry), v_chunks = chunk16_geometry(a.vpool.geometry);
  const int64_t table = (int64_t(it.seq) * a.n_kv_heads + it.kv_head) * a.table_stride;
  for (int u0 = it.kv_begin; u0 < it.kv_end; u0 += KT) {
    __syncthreads();
    if (tid < TB) live[tid] = poison[tid] = 0;
    __syncthreads();
    const bool border = u0 + KT - 1 > it.first + it.row_begin / a.n_q;  // (uniform)
    for (int i = tid; i < KT * (HDP / 16); i += 256) {
      const int t = i % KT, c0 = i / KT * 16, u = u0 + t;
      const int page = u / P, slot = u - page * P;
      float kv[16], vv[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) kv[k] = vv[k] = 0.f;
      if (u < it.kv_end && page < a.table_stride) {
        const int32_t kid = a.k_table[table + page], vid = a.v_table[table + page];
        if (uint32_t(kid) < uint32_t(a.kpool.n_descs) && uint32_t(vid) < uint32_t(a.vpool.n_descs)) {
          const dc_page_desc kd = a.kpool.descs[kid], vd = a.vpool.descs[vid];
          const BlobLayout kl = blob_layout(kd.format, kd.bits, a.kpool.geometry);
          const BlobLayout vl = blob_layout(vd.format, vd.bits, a.vpool.geometry);
          if (slot < kd.tokens && slot < vd.tokens && kd.tokens <= P && vd.tokens <= P &&
              (int64_t(kd.block) << 8) + kl.total <= a.kpool.arena_bytes &&
              (int64_t(vd.block) << 8) + vl.total <= a.vpool.arena_bytes) {
            if (c0 < hd) {
              page_values16(a.kpool, kd, slot, c0, k_chunks, kv);
              page_values16(a.vpool, vd, slot, c0, v_chunks, vv);
              if (border) {
                // a weight of 0 times an infinity or NaN would reach rows that do not see the token:
                // such values are left out here, and added to the rows that see it below
                bool bad = false;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const bool fin = __builtin_isfinite(float(T(vv[k])));
                  bad = bad || !fin;
                  vv[k] = fin ? vv[k] : 0.f;
                }
                if (bad) atomicOr(&poison[t >> 5], 1u << (t & 31));
              }
            }
            if (c0 == 0) atomicOr(&live[t >> 5], 1u << (t & 31));
          }
        }
      }
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          *reinterpret_cast<float4*>(kt + lds_at<CH>(t, c0 / 4 + k)) = float4{kv[4 * k], kv[4 * k + 1], kv[4 * k + 2], kv[4 * k + 3]};
          *reinterpret_cast<float4*>(vt + lds_at<CH>(t, c0 / 4 + k)) = float4{vv[4 * k], vv[4 * k + 1], vv[4 * k + 2], vv[4 * k + 3]};
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          h8v x, y;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[j] = _Float16(kv[8 * k + j]);
            y[j] = _Float16(vv[8 * k + j]);
          }
          *reinterpret_cast<h8v*>(kt + lds_at<CH>(t, c0 / 8 + k)) = x;
          *reinterpret_cast<h8v*>(vt + lds_at<CH>(t, c0 / 8 + k)) = y;
        }
      }
    }
    __syncthreads();
    if (border) {
#pragma unroll 1
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll 1
        for (uint32_t bits = poison[tb]; bits != 0; bits &= bits - 1) {
          const int u = u0 + 32 * tb + __builtin_ctz(bits), page = u / P;
          __syncthreads();
          if (tid < HDP / 16) {
            float x[16];
            for (int k = 0; k < 16; ++k) x[k] = 0.f;
            if (16 * tid < hd) page_values16(a.vpool, a.vpool.descs[a.v_table[table + page]], u - page * P, 16 * tid, v_chunks, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) odd[16 * tid + k] = float(T(x[k]));
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < CB; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const float x = odd[32 * i + 8 * (v / 4) + 4 * half + v % 4];
              if (u <= sees && !__builtin_isfinite(x)) o[i][v] += x;
            }
        }
    }
    if (!wave_rows) continue;

    // S^T: block tb's token 8 (v / 4) + 4 half + v % 4 against this lane's row
    f32x16 s[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[tb][v] = 0.f;
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        if constexpr (F32) {
          const float4 x = *reinterpret_cast<const float4*>(kt + lds_at<CH>(32 * tb + col, 2 * i + half));
#pragma unroll
          for (int k = 0; k < 4; ++k) s[tb] = __builtin_amdgcn_mfma_f32_32x32x2f32((&x.x)[k], (&q[i].x)[k], s[tb], 0, 0, 0);
        } else {
          const h8v x = *reinterpret_cast<const h8v*>(kt + lds_at<CH>(32 * tb + col, 2 * i + half));
          s[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[i], s[tb], 0, 0, 0);
        }
      }
    }
    // tokens that do not count, or that this row does not see
    bool masked = u0 + KT - 1 > sees_all;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) masked = masked || live[tb] != ~0u;
    float top = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
      const uint32_t bits = live[tb];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int t = 8 * (v / 4) + 4 * half + v % 4;
        if (masked) s[tb][v] = ((bits >> t) & 1) && u0 + 32 * tb + t <= sees ? s[tb][v] : -INFINITY;
        top = fmaxf(top, s[tb][v]);
      }
    }
    top = half_max(top) * c;
    if (__any(top > m + kLazy || (m == -INFINITY && top > m))) {
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 1.f : exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < CB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] *= f;
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[tb][v] = exp2f(fmaf(s[tb][v], c, -mu));
        l += s[tb][v];
      }
    // O^T: channel block i's channel 8 (v / 4) + 4 half + v % 4 of this lane's row
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < CB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int t = 32 * tb + 8 * (v / 4) + 4 * half + v % 4, ch = 32 * i + col;
            const float x = *reinterpret_cast<const float*>(vt + lds_at<CH>(t, ch / 4) + 4 * (ch % 4));
            o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[tb][v], o[i], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          h8v p;
#pragma unroll
          for (int k = 0; k < 8; ++k) p[k] = _Float16(s[tb][8 * ks + k]);
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            // (a transposed read: 16 lanes read four tokens x 16 channels, and lane n gets channel n's four)
            const int t = 32 * tb + 16 * ks + 4 * half + ((lane & 15) >> 2), ch = 32 * i + (lane & 16) + 4 * (lane & 3);
            s4v x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
              x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) s4v*)(vt + lds_at<CH>(t + 8 * j, ch / 8) + 2 * (ch % 8)));
            const h8v av = __builtin_bit_cast(h8v, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, p, o[i], 0, 0, 0);
          }
        }
      }
    }
  }
  if (!has_row) return;
  l = half_sum(l);
  if (it.partial >= 0) {
    const int64_t r = int64_t(it.partial) * kChunkRows + 32 * wave + col;
    float* po = a.part_o + r * hd;
#pragma unroll
    for (int i = 0; i < CB; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int ch = 32 * i + 8 * (v / 4) + 4 * half + v % 4;
        if (ch < hd) po[ch] = o[i][v];
      }
    if (half == 0) {
      a.part_ml[2 * r] = m;
      a.part_ml[2 * r + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t off = int64_t(it.q_begin + tok) * a.o_token_stride + int64_t(head) * a.o_head_stride;
#pragma unroll
  for (int i = 0; i < CB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int ch = 32 * i + 8 * (v / 4) + 4 * half + v % 4;
      if (ch < hd) store_value(a.out, a.dtype, off + ch, o[i][v] * inv);
    }
}

// Joins the partial results of a tile's token ranges: a wavefront per row,
// channels over its lanes.
__global__ void __launch_bounds__(256) merge_chunk_kernel(ChunkArgs a, const dc_chunk_merge* merges) {
  const dc_chunk_merge mg = merges[blockIdx.x];
  if (!chunk_merge_ok(mg, a)) return;
  const int lane = threadIdx.x & 63, r = int(blockIdx.y) * 4 + int(threadIdx.x >> 6), row = mg.row_begin + r;
  if (row >= mg.row_end) return;
  const int hd = a.kpool.geometry.head_dim;
  const int tok = row / a.n_q, head = mg.kv_head * a.n_q + (row - tok * a.n_q);
  float top = -INFINITY;
  for (int i = 0; i < mg.count; ++i) top = fmaxf(top, a.part_ml[2 * (int64_t(mg.partial_begin + i) * kChunkRows + r)]);
  const float mu = top == -INFINITY ? 0.f : top;
  const int64_t off = int64_t(mg.q_begin + tok) * a.o_token_stride + int64_t(head) * a.o_head_stride;
  for (int ch = lane; ch < hd; ch += 64) {
    float sum = 0.f, l = 0.f;
    for (int i = 0; i < mg.count; ++i) {
      const int64_t at = int64_t(mg.partial_begin + i) * kChunkRows + r;
      const float w = exp2f(a.part_ml[2 * at] - mu);
      l = fmaf(w, a.part_ml[2 * at + 1], l);
      sum = fmaf(w, a.part_o[at * hd + ch], sum);
    }
    store_value(a.out, a.dtype, off + ch, l == 0.f ? 0.f : sum / l);
  }
}

template <typename T, int HDP, int KT>
static int launch_chunk(const ChunkArgs& a, hipStream_t stream) {
  constexpr int bytes = 2 * KT * HDP * int(sizeof(T)) + 16;
  static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(&attend_chunk_kernel<T, HDP, KT>),
                                                    hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (int rc = check_hip(set, "attend_chunk_kernel LDS")) return rc;
  hipLaunchKernelGGL((attend_chunk_kernel<T, HDP, KT>), dim3(a.n_items), dim3(256), bytes, stream, a);
  return check_hip(hipGetLastError(), "attend_chunk_kernel launch");
}

}  // namespace dc

extern "C" int dc_attend_chunk(dc_pool k_pool, dc_pool v_pool, const int32_t* k_table, const int32_t* v_table,
                               int32_t table_stride, const dc_chunk_item* items, int32_t n_items,
                               const dc_chunk_merge* merges, int32_t n_merges, int32_t n_partials, int32_t n_seqs,
                               int32_t n_kv_heads, int64_t n_tokens, dc_token_rows q, float query_scale, dc_token_rows out,
                               void* workspace, int64_t workspace_bytes, dc_stream_t stream) {
  const char* who = "dc_attend_chunk";
  if (int rc = dc::validate_geometry(k_pool.geometry)) return rc;
  if (int rc = dc::validate_geometry(v_pool.geometry)) return rc;
  const int hd = k_pool.geometry.head_dim;
  if (v_pool.geometry.head_dim != hd || v_pool.geometry.page_capacity != k_pool.geometry.page_capacity)
    return dc::fail(DC_EINVAL, "%s: key and value pools must share head_dim and page_capacity", who);
  if (hd > 256) return dc::fail(DC_EINVAL, "%s: head_dim above 256", who);
  if (n_items < 0 || n_merges < 0 || n_partials < 0 || n_seqs <= 0 || n_kv_heads <= 0 || n_tokens < 0 || table_stride <= 0)
    return dc::fail(DC_EINVAL, "%s: bad counts", who);
  if (n_items == 0) return DC_OK;
  if (!k_pool.arena || !v_pool.arena || !k_pool.descs || !v_pool.descs || !k_table || !v_table || !items || !q.data || !out.data ||
      (n_merges && !merges))
    return dc::fail(DC_EINVAL, "%s: null pointer", who);
  if (q.dtype != DC_F32 && q.dtype != DC_F16 && q.dtype != DC_BF16) return dc::fail(DC_EINVAL, "%s: queries must be DC_F32, DC_F16 or DC_BF16", who);
  if (out.dtype != q.dtype || out.n_heads != q.n_heads || q.n_heads <= 0 || q.n_heads % n_kv_heads)
    return dc::fail(DC_EINVAL, "%s: the output needs the queries' dtype and heads, a multiple of the KV heads", who);
  const int64_t rows = int64_t(n_partials) * dc::kChunkRows;
  if (workspace_bytes < dc_chunk_workspace_bytes(n_partials, hd) || (n_partials && !workspace))
    return dc::fail(DC_ESPACE, "%s: workspace too small", who);
  dc::ChunkArgs a{k_pool, v_pool, k_table, v_table, table_stride, items, n_items, n_seqs, n_kv_heads, q.n_heads / n_kv_heads,
                  n_tokens, n_partials, q.data, q.token_stride, q.head_stride, q.dtype, query_scale, out.data, out.token_stride,
                  out.head_stride, static_cast<float*>(workspace), static_cast<float*>(workspace) + rows * hd};
  const hipStream_t st = hipStream_t(stream);
  int rc;
  if (q.dtype == DC_F32)
    rc = hd <= 64 ? dc::launch_chunk<float, 64, 64>(a, st) : hd <= 128 ? dc::launch_chunk<float, 128, 32>(a, st) : dc::launch_chunk<float, 256, 32>(a, st);
  else
    rc = hd <= 64 ? dc::launch_chunk<_Float16, 64, 128>(a, st) : hd <= 128 ? dc::launch_chunk<_Float16, 128, 64>(a, st) : dc::launch_chunk<_Float16, 256, 32>(a, st);
  if (rc != DC_OK || n_merges == 0) return rc;
  hipLaunchKernelGGL(dc::merge_chunk_kernel, dim3(n_merges, dc::kChunkRows / 4), dim3(256), 0, st, a, merges);
  return dc::check_hip(hipGetLastError(), "merge_chunk_kernel launch");
}
