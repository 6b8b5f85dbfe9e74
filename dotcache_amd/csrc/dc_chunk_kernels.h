// Attention of a chunk of new tokens of every sequence over its compressed
// pages (dc_attend_chunk): prompt chunks, drafted tokens and decodes of one
// batch in one launch, causal among the new tokens.
//
//   o_r = sum_u p_ru v_u / sum_u p_ru,  p_ru = exp(scale q_r . k_u),  u <= last token that row r sees
//
// A work item is a tile of up to 256 query rows (token-major, the n_q heads of a KV
// head next to each other, so they share every key and value) of one
// (sequence, KV head) against a range of its tokens.  Wavefronts of 32 rows
// each walk the range in tiles of KT tokens: the block turns a tile's
// page rows into dense rows in LDS once, for all its query rows, and every
// wavefront then takes
//   S^T = K Q^T   tokens x rows, so a lane holds one row's logits and the
//                 softmax needs one exchange between the two half-wavefronts;
//   O^T += V^T P^T  with P in the registers it was computed in: the matrix
//                 instruction's k index runs over the tokens in the order in
//                 which S^T left them, and V's operand is read in that order.
// The running maximum moves only when a tile's exceeds it by 2^kLazy, so that
// rescaling the output is rare; sums and the output are fp32.  The maximum is
// taken of unscaled logits, and a masked one is an infinity before it is
// scaled, which needs a positive scale: the queries carry the scale's sign
// (exactly; with a scale of 0 they are zeros, and the scale 1).
//
// Three kernels, by what the pools hold and by rows: attend_chunk16_kernel
// (16-bit queries, pages of 32-channel units: 2 x 2048 rows of 7 heads a KV head
// over 16384 tokens, fp16 keys and 4-bit values, 1.31 ms with the join, 690
// TFLOP/s of an fp16 library product's 1178; 1.04 ms without the page loads),
// attend_few_kernel (the same pages, few rows against a long range: 5 rows of 7
// heads of four sequences to 131072 tokens, 126 MB, 92 us with the join, where
// the copy rate would take 27; when it was made 170 us, the 256-row kernel 320) and
// attend_chunk_kernel (the rest: 3 x 61 rows of 1001 tokens in fp32 83 us and 7
// for the join; the two calls above, made with 16-bit queries on pools that have
// held a 2-bit page, 4.3 ms and 0.61).
// 16-bit queries' operands are fp16, which the matrix unit takes at eight times
// the fp32 rate: a query, a page's value and a weight are each rounded to it
// once, by 2^-11 relative, or below 2^-14 (a weight: below 2^-21 of the row's
// largest) by 2^-25 (2^-32 of the largest).  All of a row's ranges lift their
// weights alike (kLift), so that joins and the final division cancel it.
//
// RULE, kRuled or kCapped: tokens of any two ranges a row, and shaped scores (dc_attend_chunk_rule),
// instances with a cap apart (its code took registers that those without it need: 4 % at head_dim 64).
// A tile's products are turned into exponents (cap, slope) where they lie, then
// masked; a tile that no row of a wavefront sees is none of its work, one that all see
// whole has no mask.  A cap costs 11 % (2 x 2048 rows at head_dim 256, window
// 4096: 737 -> 822 us), slopes 25 % (1024 rows of 4096 tokens at head_dim 64: 77
// -> 95).
#pragma once

#include <atomic>

#include "dc_chunk.h"
#include "dc_unpack.h"

namespace dc {

namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLazy = 8.f;  // log2 of how far a weight may pass the maximum's before the maximum moves
// log2 of the weight that a row's maximum has as an fp16 operand.  The steps of
// small weights, 2^-24 of 2^7, are then 2^-31 of the maximum's; the largest
// weight, 2^(kLift + kLazy), is half of what fp16 holds.
constexpr float kLift = 7.f;

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

// An address that the compiler takes for a new one here: what is derived from
// it by one exclusive or is then computed where it is used, not kept in a
// register for each use across the loop.  (Chunks are exchanged by exclusive
// or within a row, so a chunk's address is its row's, the chunk's number
// joined in by exclusive or too, where the numbers share no bits.)
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// {a, b} of lanes 0 .. 31 and {a, b} of lanes 32 .. 63, exchanged to {a of the
// first half, b of the first} and {a of the second, b of the second}: x is
// what the first, y what the second half held, a in lanes 0 .. 31, b in 32 .. 63.
__device__ __forceinline__ float2 swap_halves(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t x = r[0], y = r[1];  // (bit casts of vector elements would all take the first)
  return float2{__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float2 both_halves(float v) { return swap_halves(v, v); }
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

// Whether the page d describes lies in the pool and holds token slot `slot`.
__device__ __forceinline__ bool page_holds(const dc_pool& pool, const dc_page_desc& d, int slot) {
  return slot < d.tokens && d.tokens <= pool.geometry.page_capacity &&
         (int64_t(d.block) << 8) + blob_layout(d.format, d.bits, pool.geometry).total <= pool.arena_bytes;
}

// This block's item where each takes `parts` blocks, which run on one die (they
// read the same pages), and which of them the block is.
__device__ __forceinline__ uint32_t block_index(int parts) {
  return blockIdx.x / kChunkXcds / parts * kChunkXcds + blockIdx.x % kChunkXcds;
}
__device__ __forceinline__ dc_chunk_item block_item(const ChunkArgs& a, int parts, int* part) {
  const uint32_t i = block_index(parts);
  *part = int(blockIdx.x / kChunkXcds % parts);
  return i < uint32_t(a.n_items) ? a.items[i] : dc_chunk_item{-1};
}

inline dim3 item_grid(int32_t n_items, int parts) {
  return dim3(parts == 1 ? uint32_t(n_items) : (uint32_t(n_items) + kChunkXcds - 1) / kChunkXcds * kChunkXcds * parts);
}

// Narrows an item to its part of `rows` rows, and its tokens to what they see
// if they are `causal`; false: none left.
__device__ __forceinline__ bool block_rows(dc_chunk_item& it, int part, int rows, int n_q, bool causal = true) {
  const int skip = rows * part;
  if (it.row_begin + skip >= it.row_end) return false;
  it.row_begin += skip;
  if (it.partial >= 0) it.partial += skip;
  it.row_end = min(it.row_end, it.row_begin + rows);
  if (causal) it.kv_end = max(min(it.kv_end, it.first + (it.row_end - 1) / n_q + 1), it.kv_begin);
  return true;
}

// ---- the rule of a call (dc_score_rule) ---------------------------------------

// The tokens that a query row sees, first .. first + len - 1 and first2 ..
// first2 + len2 - 1, its own token and its slope.
struct RowRule {
  int first, len, first2, len2, at;
  float slope;
  __device__ __forceinline__ bool sees(int u) const {
    return uint32_t(u - first) < uint32_t(len) || uint32_t(u - first2) < uint32_t(len2);
  }
};

__device__ __forceinline__ int4 token_range(const ChunkArgs& a, const dc_chunk_item& it, int tok) {
  const int4 r = a.ranges ? a.ranges[int64_t(it.q_begin) + tok] : int4{0, 0, 0, it.first + tok + 1};
  return int4{r.x, max(r.y, r.x), r.z, max(r.w, r.z)};
}

// (a row that does not exist sees nothing)
__device__ __forceinline__ RowRule row_rule(const ChunkArgs& a, const dc_chunk_item& it, bool has_row, int tok, int head) {
  const int4 r = token_range(a, it, has_row ? tok : it.row_begin / a.n_q);
  return RowRule{r.z, has_row ? r.w - r.z : 0, r.x, has_row ? r.y - r.x : 0, it.first + tok,
                 a.slopes && has_row ? a.slopes[head] * kLog2e : 0.f};
}

// What rows [row0, row1) of an item see: all of them the tokens of `all`, and
// none a token outside `any` (two ranges each, as RowRule's).
struct Sight {
  int all0, all1, all20, all21, any0, any1, any20, any21;
  // Whether all rows see all of tokens u .. u + n - 1; whether one sees one.
  __device__ __forceinline__ bool whole(int u, int n) const { return (u >= all0 && u + n <= all1) || (u >= all20 && u + n <= all21); }
  __device__ __forceinline__ bool some(int u, int n) const { return (u < any1 && u + n > any0) || (u < any21 && u + n > any20); }
};

__device__ __forceinline__ Sight sight_of(const ChunkArgs& a, const dc_chunk_item& it, int row0, int row1) {
  Sight s{0, INT32_MAX, 0, INT32_MAX, INT32_MAX, 0, INT32_MAX, 0};
  if (row0 < row1) {
    const int t1 = (row1 - 1) / a.n_q;
    for (int t = row0 / a.n_q + int(threadIdx.x & 63); t <= t1; t += 64) {
      const int4 r = token_range(a, it, t);
      s.all0 = max(s.all0, r.z); s.all1 = min(s.all1, r.w); s.all20 = max(s.all20, r.x); s.all21 = min(s.all21, r.y);
      if (r.z < r.w) s.any0 = min(s.any0, r.z), s.any1 = max(s.any1, r.w);
      if (r.x < r.y) s.any20 = min(s.any20, r.x), s.any21 = max(s.any21, r.y);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    s.all0 = max(s.all0, __shfl_xor(s.all0, d)); s.all1 = min(s.all1, __shfl_xor(s.all1, d));
    s.all20 = max(s.all20, __shfl_xor(s.all20, d)); s.all21 = min(s.all21, __shfl_xor(s.all21, d));
    s.any0 = min(s.any0, __shfl_xor(s.any0, d)); s.any1 = max(s.any1, __shfl_xor(s.any1, d));
    s.any20 = min(s.any20, __shfl_xor(s.any20, d)); s.any21 = max(s.any21, __shfl_xor(s.any21, d));
  }
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return Sight{uni(s.all0), uni(s.all1), uni(s.all20), uni(s.all21), uni(s.any0), uni(s.any1), uni(s.any20), uni(s.any21)};
}

// A product q . k as the exponent of its weight, in log2, before the maximum:
// cap tanh(y), y = scale q.k / cap and x = 2 y log2 e, or (no cap) scale q.k.
// Where |y| < 1/2 it is x times a polynomial of x^2 for tanh(y) / y (fitted to
// 2^-26 there), so that the error is a share of the score, whatever the cap.  Beyond,
// cap (1 - 2 / (exp2(|x|) + 1)) with the sign, which holds at either infinity and cancels little.
__device__ __forceinline__ float capped(const ChunkArgs& a, float x) {
  const float t = x * x;
  float near = a.cap * (x * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.2437525e-06f, -3.1857868e-05f), 6.6630519e-04f), -1.3875948e-02f), 0.34657359f));
  float far = a.cap * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fabsf(x)) + 1.f), 1.f);  // (2 cap may leave fp32)
  asm volatile("" : "+v"(near), "+v"(far));  // (both, and a selection: no branch for each score)
  return fabsf(x) < 1.44269504f ? near : __builtin_copysignf(far, x);
}

// The second form alone, for 16-bit queries and caps to kCoarseCap: off by 2^-21 of the cap
// whatever the score, so a weight by 2^-13, where its own rounding to fp16 and those
// of its logit's operands are 2^-11 each (2 x 2048 rows at head_dim 256, window 4096: 822 us, the other 935).
constexpr float kCoarseCap = 256.f;
__device__ __forceinline__ float capped_coarse(float cap, float x) {
  return fmaf(-2.f * cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.f), cap);
}

// The products of a row with blocks of tokens as such exponents: element v of
// block i is token u + 32 i + 8 (v / 4) + v % 4 (16 elements a block), or token
// u + 16 i + v (4 elements).
template <bool CAP, bool EXACT, typename V, int N>
__device__ __forceinline__ void shape_scores(const ChunkArgs& a, float c, const RowRule& r, int u, V (&s)[N]) {
  constexpr int W = sizeof(V) / 4;
  if constexpr (CAP) {
    // (factors of its own: products common to both branches would be taken ahead of them, into registers)
    float cap = a.cap, cap_in = a.cap_in;
    asm("" : "+s"(cap), "+s"(cap_in));
    if (!EXACT && cap <= kCoarseCap * kLog2e) {  // (uniform)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < W; ++v) s[i][v] = capped_coarse(cap, cap_in * s[i][v]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < W; ++v) {
          s[i][v] = capped(a, a.cap_in * s[i][v]);
          if (N * W > 16 && v % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (four at a time, where the registers are short)
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int v = 0; v < W; ++v) s[i][v] *= c;
  }
  if (a.slopes) {
    const float away = float(r.at - u);  // (the difference of far tokens is exact, they themselves are not)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int v = 0; v < W; ++v) s[i][v] = fmaf(-r.slope, fabsf(away - float((W == 16 ? 32 : 16) * i + 2 * (v & ~3) + v % 4)), s[i][v]);
  }
}

// The item's gap: its tiles leave out tokens [x, y).  One that does not lie inside
// the item is none (a fault guard, as chunk_item_ok: the tiles' loop has to
// end), and costs time only, since ranges say what a row sees.
__device__ __forceinline__ int2 item_gap(const ChunkArgs& a, const dc_chunk_item& it, uint32_t item) {
  const int2 g = a.gaps ? a.gaps[item] : int2{-1, -1};
  return g.x > it.kv_begin && g.y > g.x && g.y < it.kv_end ? g : int2{-1, -1};
}

}  // namespace

// T: the matrix operands, _Float16 or float.  HDP: head_dim rounded up to the
// operands' rows (channels past head_dim are zeros).  KT: tokens per tile.
template <typename T, int HDP, int KT, int RULE>
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

  int of_item;
  dc_chunk_item it = block_item(a, kChunkRows / 128, &of_item);
  if (!chunk_item_ok(it, a) || !block_rows(it, of_item, 128, a.n_q, !RULE || !a.ranges)) return;
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
  RowRule rule;
  Sight mine, all;  // the wavefront's rows' and the block's
  int2 gap{-1, -1};
  if constexpr (RULE) {
    rule = row_rule(a, it, has_row, tok, head);
    mine = sight_of(a, it, it.row_begin + 32 * wave, min(it.row_begin + 32 * wave + 32, it.row_end));
    all = sight_of(a, it, it.row_begin, it.row_end);
    gap = item_gap(a, it, block_index(kChunkRows / 128));
  }
  auto seen = [&](int u) { return RULE ? rule.sees(u) : u <= sees; };

  // Q as the B operand: row col, channels 16 ks + 8 half .. + 7 (F32: 8 ks + 4 half .. + 3)
  constexpr int QW = F32 ? HDP / 8 : HDP / 16;
  typedef std::conditional_t<F32, float4, h8v> QV;
  QV q[QW];
  {
    // (channels past head_dim and rows that do not exist: an element that does, then zero; no branch between the loads)
    constexpr int W = F32 ? 4 : 8;
    typedef std::conditional_t<F32, float, uint16_t> QT;  // (16-bit: bits of either type)
    const int rr = has_row ? row : it.row_begin, rt = rr / a.n_q;
    const QT* const p = reinterpret_cast<const QT*>(a.q) + int64_t(it.q_begin + rt) * a.q_token_stride +
                        int64_t(it.kv_head * a.n_q + rr - rt * a.n_q) * a.q_head_stride;
    QT w[QW][W];
#pragma unroll
    for (int i = 0; i < QW; ++i)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int ch = 2 * W * i + W * half + k;
        w[i][k] = p[ch < hd ? ch : 0];
      }
    const bool f16 = a.dtype == DC_F16;
#pragma unroll
    for (int i = 0; i < QW; ++i)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const bool in = has_row && 2 * W * i + W * half + k < hd;
        if constexpr (F32)
          (&q[i].x)[k] = in ? w[i][k] * a.sign : 0.f;
        else
          q[i][k] = !in   ? _Float16(0)
                    : f16 ? __builtin_bit_cast(_Float16, w[i][k]) * _Float16(a.sign)
                          : _Float16(__uint_as_float(uint32_t(w[i][k]) << 16) * a.sign);
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
    if (RULE && u0 == gap.x) u0 = gap.y;  // (a piece with a gap has tokens behind it)
    __syncthreads();
    if (tid < TB) live[tid] = poison[tid] = 0;
    __syncthreads();
    const bool border = RULE ? !all.whole(u0, KT) : u0 + KT - 1 > it.first + it.row_begin / a.n_q;  // (uniform)
    // (keys first, then values: KT HDP / 16 is a multiple of the block, so the side is uniform)
    for (int i = tid; i < KT * (HDP / 8); i += 256) {
      const bool vals = i >= KT * (HDP / 16);
      const int t = i % KT, c0 = (i / KT - (vals ? HDP / 16 : 0)) * 16, u = u0 + t;
      const int page = u / P, slot = u - page * P;
      const dc_pool& pool = vals ? a.vpool : a.kpool;
      float x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = 0.f;
      if (u < it.kv_end && page < a.table_stride) {
        const int32_t kid = a.k_table[table + page], vid = a.v_table[table + page];
        if (uint32_t(kid) < uint32_t(a.kpool.n_descs) && uint32_t(vid) < uint32_t(a.vpool.n_descs)) {
          const dc_page_desc kd = a.kpool.descs[kid], vd = a.vpool.descs[vid];
          if (page_holds(a.kpool, kd, slot) && page_holds(a.vpool, vd, slot)) {
            if (c0 < hd) page_values16(pool, vals ? vd : kd, slot, c0, vals ? v_chunks : k_chunks, x);
            if (vals && border) {
              // a weight of 0 times an infinity or NaN would reach rows that do not see the token:
              // such values are left out here, and added to the rows that see it below
              bool bad = false;
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const bool fin = __builtin_isfinite(float(T(x[k])));
                bad = bad || !fin;
                x[k] = fin ? x[k] : 0.f;
              }
              if (bad) atomicOr(&poison[t >> 5], 1u << (t & 31));
            }
            if (!vals && c0 == 0) atomicOr(&live[t >> 5], 1u << (t & 31));
          }
        }
      }
      uint8_t* const tile = vals ? vt : kt;
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<float4*>(tile + lds_at<CH>(t, c0 / 4 + k)) = float4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          h8v y;
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = _Float16(x[8 * k + j]);
          *reinterpret_cast<h8v*>(tile + lds_at<CH>(t, c0 / 8 + k)) = y;
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
              if (seen(u) && !__builtin_isfinite(x)) o[i][v] += x;
            }
        }
    }
    if (!wave_rows || (RULE && !mine.some(u0, KT))) continue;

    // S^T: block tb's token 8 (v / 4) + 4 half + v % 4 against this lane's row
    f32x16 s[TB];
    const int k_at = fresh(lds_at<CH>(col, half));
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[tb][v] = 0.f;
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        if constexpr (F32) {
          const float4 x = *reinterpret_cast<const float4*>(kt + (k_at ^ (32 * i)) + 32 * tb * CH * 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) s[tb] = __builtin_amdgcn_mfma_f32_32x32x2f32((&x.x)[k], (&q[i].x)[k], s[tb], 0, 0, 0);
        } else {
          const h8v x = *reinterpret_cast<const h8v*>(kt + (k_at ^ (32 * i)) + 32 * tb * CH * 16);
          s[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[i], s[tb], 0, 0, 0);
        }
      }
    }
    if constexpr (RULE) shape_scores<RULE == kCapped, F32>(a, c, rule, u0 + 4 * half, s);
    // tokens that do not count, or that this row does not see
    bool masked = RULE ? !mine.whole(u0, KT) : u0 + KT - 1 > sees_all;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) masked = masked || live[tb] != ~0u;
    float top = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
      const uint32_t bits = live[tb];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int t = 8 * (v / 4) + 4 * half + v % 4;
        if (masked) s[tb][v] = ((bits >> t) & 1) && seen(u0 + 32 * tb + t) ? s[tb][v] : -INFINITY;
        top = fmaxf(top, s[tb][v]);
      }
    }
    top = half_max(top) * (RULE ? 1.f : c);
    if (__any(top > m + kLazy || (m == -INFINITY && top > m))) {
      const float mn = fmaxf(m, top);
      // (no maximum yet: the output holds zeros, or an infinity or NaN from above)
      const float f = m == -INFINITY ? 1.f : exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < CB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] *= f;
    }
    const float mu = (m == -INFINITY ? 0.f : m) - (F32 ? 0.f : kLift);
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[tb][v] = exp2f(RULE ? s[tb][v] - mu : fmaf(s[tb][v], c, -mu));
        l += s[tb][v];
      }
    // O^T: channel block i's channel 8 (v / 4) + 4 half + v % 4 of this lane's row
    // (F32: the value of token 32 tb + 8 (v / 4) + 4 half + v % 4, channel 32 i + col)
    const int v_at = fresh(4 * half * CH * 16 + ((col / 4) ^ half) * 16 + 4 * (col % 4));
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
      if constexpr (F32) {
        static_assert(!F32 || CH >= 16, "the exchange of chunks that v_at joins in");
#pragma unroll
        for (int i = 0; i < CB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int exchanged = (8 * i) ^ ((v % 4) << 2 | (2 * (v / 4) & 3)), first = (32 * tb + 8 * (v / 4) + v % 4) * CH * 16;
            const float x = *reinterpret_cast<const float*>(vt + (v_at ^ (16 * exchanged)) + first);
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
    const int64_t r = int64_t(it.partial) + 32 * wave + col;
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

// ---- 16-bit queries, 32-channel groups ------------------------------------

namespace {

// Channels of an 8-channel group in the order in which LDS rows hold them: a
// 4-bit word gives the pairs (0, 4), (1, 5), (2, 6), (3, 7) with one mask
// each.  Keys and queries share the order, and the output's is undone at the
// end, so it costs nothing.
constexpr int kAhead = 4;  // matrix operands read ahead
constexpr int kPerm[8] = {0, 4, 1, 5, 2, 6, 3, 7};

__device__ __forceinline__ uint32_t twice(uint32_t h) { return h | (h << 16); }

// Where a thread's 16 channels lie in the pages of a pool: the wavefront's
// part (page layout) and the thread's (its channels, and its token where the
// wavefront's share a page).  Byte offsets are those of 4-bit codes; 8-bit
// ones are twice as far.
struct Side {
  const uint8_t* arena;
  const dc_page_desc* descs;
  const int32_t* table;
  int64_t arena_bytes;
  int32_t n_descs;
  uint32_t token4, scales4, gap, f16_bytes, row2, groups2;
  uint32_t at4, scale_at, f16_at;
};

__device__ __forceinline__ Side make_side(const dc_pool& p, const int32_t* table, uint32_t lt, uint32_t c0) {
  const dc_page_geometry& geo = p.geometry;
  Side x;
  x.arena = reinterpret_cast<const uint8_t*>(p.arena);
  x.descs = p.descs;
  x.table = table;
  x.arena_bytes = p.arena_bytes;
  x.n_descs = p.n_descs;
  const uint32_t C = geo.page_capacity, G = num_groups(geo), gs = geo.group_size, row = gs / 2, g = c0 / gs;
  x.token4 = geo.layout == 0 ? row : G * row;
  x.scales4 = G * C * row;
  x.gap = (C * G * 2 + 15u) & ~15u;
  x.f16_bytes = C * geo.head_dim * 2;
  x.row2 = 2 * geo.head_dim;
  x.groups2 = 2 * G;
  const bool in = int(c0) < geo.head_dim;  // (channels past head_dim: any of the page's)
  x.at4 = lt * x.token4 + (in ? g * (geo.layout == 0 ? C * row : row) + (c0 - g * gs) / 2 : 0);
  x.scale_at = (lt * G + (in ? g : 0)) * 2;
  x.f16_at = (lt * geo.head_dim + (in ? c0 : 0)) * 2;
  return x;
}

enum UnitKind { U_NONE = 0, U_F16, U_B4, U_B8 };

// Kind of a page's units, or U_NONE: no such page in the pool, or its first
// token wanted is not in it.
__device__ __forceinline__ int unit_kind(const Side& x, const dc_page_desc& d, int capacity, int slot) {
  const bool m0 = d.format == DC_FMT_M0_AFFINE || d.format == DC_FMT_M0_SYMMETRIC;
  const bool b8 = d.bits == 8;
  const uint32_t codes = b8 ? 2 * x.scales4 : x.scales4;
  const uint32_t bytes = m0 ? codes + (d.format == DC_FMT_M0_AFFINE ? 2 * x.gap : x.gap) : x.f16_bytes;
  const bool ok = slot < d.tokens && d.tokens <= capacity && (int64_t(d.block) << 8) + bytes <= x.arena_bytes;
  return !ok ? U_NONE : d.format == DC_FMT_M3_F16 ? U_F16 : !m0 ? U_NONE : b8 ? U_B8 : d.bits == 4 ? U_B4 : U_NONE;
}

// Loads from a page: the page's and the wavefront's part of the address in
// scalar registers and the lane's in one vector register where the wavefront
// shares the page (a buffer load; pointers would take two registers for each
// load), or by pointer where each lane has its own.  Every load is made
// whatever the page holds, `ok` false from nowhere (zeros) or from `none`: a
// register that two branches load would be waited for where they meet.
template <bool UNI>
struct PageLoad {
  const uint8_t* base;
  const void* none;
  bool ok;
  __device__ __forceinline__ uint16_t u16(uint32_t off, uint32_t lane) const {
    if constexpr (UNI) return (__builtin_amdgcn_raw_buffer_load_b16(rsrc(), int(lane), int(ok ? off : 0), 0));
    return *static_cast<const uint16_t*>(at(off, lane));
  }
  __device__ __forceinline__ uint32_t u32(uint32_t off, uint32_t lane) const {
    if constexpr (UNI) return __builtin_amdgcn_raw_buffer_load_b32(rsrc(), int(lane), int(ok ? off : 0), 0);
    return *static_cast<const uint32_t*>(at(off, lane));
  }
  __device__ __forceinline__ uint2 u64(uint32_t off, uint32_t lane) const {
    if constexpr (UNI) return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rsrc(), int(lane), int(ok ? off : 0), 0));
    return uint2{static_cast<const uint32_t*>(at(off, lane))[0], static_cast<const uint32_t*>(at(off, lane))[1]};
  }
  __device__ __forceinline__ uint4 u128(uint32_t off, uint32_t lane) const {
    if constexpr (UNI) return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(), int(lane), int(ok ? off : 0), 0));
    const uint32_t* p = static_cast<const uint32_t*>(at(off, lane));
    return uint4{p[0], p[1], p[2], p[3]};
  }

 private:
  __device__ __forceinline__ auto rsrc() const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, ok ? 0x7fffffff : 0, 0x00027000);
  }
  __device__ __forceinline__ const void* at(uint32_t off, uint32_t lane) const { return ok ? base + off + lane : none; }
};

// The unit's bytes: r (a 4-bit unit's are the first two words), scale and bias.  A 4-bit unit's 16-byte read ends in the
// scales at the latest.
template <bool UNI>
__device__ __forceinline__ void load_unit(const Side& x, const uint8_t* blob, const void* none, int kind, bool affine, uint32_t slot,
                                          uint32_t (&r)[8], uint16_t& scale, uint16_t& bias) {
  const PageLoad<UNI> p{blob, none, kind != U_NONE};
  const bool f16 = kind == U_F16;
  const uint32_t sh = kind == U_B8;
  const uint32_t off = f16 ? slot * x.row2 : (slot * x.token4) << sh, lane = f16 ? x.f16_at : x.at4 << sh;
  const uint4 u = p.u128(off, lane), v = p.u128(off + (f16 ? 16 : 0), lane);
  r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
  r[4] = v.x; r[5] = v.y; r[6] = v.z; r[7] = v.w;
  const uint32_t so = f16 ? 0 : (x.scales4 << sh) + slot * x.groups2, sl = f16 ? 0 : x.scale_at;
  scale = p.u16(so, sl);
  bias = p.u16(so + (affine ? x.gap : 0), sl);  // (the scale again where there is none: nothing here may wait for a load)
}

__device__ __forceinline__ uint32_t scaled(uint32_t codes, uint32_t zero, h2v s, h2v b) {
  const h2v h = __builtin_bit_cast(h2v, codes | 0x64006400u) + __builtin_bit_cast(h2v, zero);  // exact
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(h, s, b));
}

// The unit's 16 values as fp16 in LDS order, two chunks of 16 bytes.
__device__ __forceinline__ void unit_values(int kind, bool affine, const uint32_t (&r)[8], uint32_t scale, uint32_t bias,
                                            uint32_t (&y)[8]) {
  if (kind == U_F16) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = __builtin_amdgcn_perm(r[4 * (i / 4) + 2 + (i % 4) / 2], r[4 * (i / 4) + (i % 4) / 2], i & 1 ? 0x07060302u : 0x05040100u);
    return;
  }
  const h2v s = __builtin_bit_cast(h2v, twice(scale)), b = __builtin_bit_cast(h2v, affine ? twice(bias) : 0u);
  // -(1024 + zero point): 0xe400 is -1024, one unit per code
  const uint32_t zero = twice(affine ? 0xe400u : kind == U_B4 ? 0xe407u : 0xe47fu);
  if (kind == U_B4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = scaled((r[i / 4] >> (4 * (i % 4))) & 0x000f000fu, zero, s, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = scaled(__builtin_amdgcn_perm(r[2 * (i / 4) + 1], r[2 * (i / 4)], 0x0c040c00u + 0x00010001u * (i % 4)), zero, s, b);
  }
}

// N groups of eight channels of a query row, from channel c0 in steps of `step`.
template <int N>
__device__ __forceinline__ void load_rows(const ChunkArgs& a, const uint16_t* p, int c0, int step, bool has_row, int hd,
                                          uint32_t (&w)[N][4]) {
  if (a.q_vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int ch = c0 + step * k;
      const uint4 x = *reinterpret_cast<const uint4*>(p + (has_row && ch < hd ? ch : 0));
      w[k][0] = x.x; w[k][1] = x.y; w[k][2] = x.z; w[k][3] = x.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ch = (has_row && c0 + step * k < hd ? c0 + step * k : 0) + 2 * i;
        w[k][i] = p[ch] | uint32_t(p[ch + 1]) << 16;
      }
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[k][i] = has_row && c0 + step * k < hd ? w[k][i] : 0;
}

// Them, times `sign`, as fp16 matrix operands, in LDS order.
template <int N>
__device__ __forceinline__ void to_operands(bool f16, float sign, const uint32_t (&w)[N][4], h8v (&q)[N]) {
  if (f16) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) q[k][i] = __builtin_bit_cast(_Float16, uint16_t(w[k][kPerm[i] / 2] >> (16 * (kPerm[i] % 2)))) * _Float16(sign);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) q[k][i] = _Float16(__builtin_bit_cast(float, kPerm[i] % 2 ? w[k][kPerm[i] / 2] & 0xffff0000u : w[k][kPerm[i] / 2] << 16) * sign);
  }
}

// OR over the wavefront's parts of a token: bit t of the result is token t of
// the wavefront's N tokens (lane t + N part).
template <int N>
__device__ __forceinline__ uint32_t fold_tokens(uint64_t b) {
#pragma unroll
  for (int n = 32; n >= N; n >>= 1) b |= b >> n;
  return uint32_t(b) & ((1u << N) - 1u);
}

}  // namespace

// fp16 operands where head_dim and both group sizes are multiples of 32 and the
// pools hold 4- and 8-bit codes and fp16 rows.  Eight wavefronts of 32 rows
// share a tile; a thread turns 16 channels of one token's key and of its value
// into LDS (unit_values; packed fp16 arithmetic), two tiles in turn: while the
// matrix instructions take tile i, tile i + 1 is written from registers, the
// page rows of the next two are on their way to registers, and the descriptors
// and page ids of the tiles after them likewise.
// UNI: the NT tokens that a wavefront turns always lie in one page, whose id,
// descriptor and addresses are then the wavefront's.
// CS: wavefronts that share 32 rows, each with a part of the output's channels
// (head_dim 256, whose queries and output of 32 rows fill the registers).
// WHOLE: head_dim is HDP, so that no channel is left out and no mask kept for it
// (12 sequences at head_dim 256 608 -> 597 us, five rows of four long sequences 98 -> 95).
template <int HDP, int KT, bool UNI, int CS, bool WHOLE, int RULE>
__global__ void __launch_bounds__(512, 2) attend_chunk16_kernel(ChunkArgs a) {
  constexpr int CH = HDP / 8, TB = KT / 32, CB = HDP / 32 / CS, TILE = KT * HDP * 2, QW = HDP / 16;
  constexpr int NT = KT < 64 ? 8 : KT / 8;  // tokens a wavefront turns
  constexpr int TW = KT / NT, PG = 8 / TW;  // wavefronts to a tile's tokens; parts of the channels that groups of TW take
  static_assert(KT * HDP == 512 * 16, "one key and one value unit per thread");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [2] keys, then [2] values
  __shared__ __attribute__((aligned(4))) uint8_t live[2][KT / 8], poison[2][PG][KT / 8];  // one bit per token, as in attend_chunk_kernel
  __shared__ float odd[HDP];

  int of_item;
  dc_chunk_item it = block_item(a, CS, &of_item);
  if (!chunk_item_ok(it, a) || !block_rows(it, of_item, 256 / CS, a.n_q, !RULE || !a.ranges)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hd = WHOLE ? HDP : a.kpool.geometry.head_dim, P = a.kpool.geometry.page_capacity;

  const int rows_at = 32 * (wave % (8 / CS)), cb0 = CS > 1 ? CB * (wave / (8 / CS)) : 0;  // (cb0: first channel block)
  const int row = it.row_begin + rows_at + col;
  const bool wave_rows = it.row_begin + rows_at < it.row_end;  // (uniform)
  const bool has_row = row < it.row_end;
  const int tok = row / a.n_q, head = it.kv_head * a.n_q + (row - tok * a.n_q);
  const int sees = has_row ? it.first + tok : -1;
  const int sees_all = it.first + (it.row_begin + rows_at) / a.n_q;
  const int sees_block = it.first + it.row_begin / a.n_q;
  RowRule rule;
  Sight mine, all;  // the wavefront's rows' and the block's
  int gap_tile = INT32_MAX, gap_len = 0;
  if constexpr (RULE) {
    const int2 gap = item_gap(a, it, block_index(CS));
    if (gap.x >= 0) gap_tile = (gap.x - it.kv_begin) / KT, gap_len = gap.y - gap.x;
  }
  auto seen = [&](int u) { return RULE ? rule.sees(u) : u <= sees; };
  // tokens from the item's first to a tile's
  auto offset = [&](int tile) { return tile * KT + (RULE && tile >= gap_tile ? gap_len : 0); };

  // ---- the tiles' way from the pages to LDS
  const int tw = wave % TW, pg = wave / TW;
  const int ut = tw * NT + lane % NT, uc = 16 * (lane / NT) + HDP / PG * pg;  // this thread's token of a tile, first channel
  const int lt = UNI ? lane % NT : 0;                           // token within the wavefront's, where they share a page
  const int u_first = it.kv_begin + (UNI ? tw * NT : ut);     // first token of this wavefront's (thread's) of tile 0
  const int64_t table = (int64_t(it.seq) * a.n_kv_heads + it.kv_head) * a.table_stride;
  const int tiles = (it.kv_end - it.kv_begin - gap_len + KT - 1) / KT;
  const bool has = uc < hd;
  const Side ks = make_side(a.kpool, a.k_table + table, lt, uc), vs = make_side(a.vpool, a.v_table + table, lt, uc);
  auto uni = [](int x) { return UNI ? __builtin_amdgcn_readfirstlane(x) : x; };
  auto page_of = [&](int tile) { return uint32_t((uint64_t(uint32_t(u_first + offset(tile))) * a.page_mul) >> a.page_shift); };
  // (a zero in a vector register: ids and descriptors are then read by vector
  // loads, which come back in order; a scalar load in flight would make the next
  // wait for LDS wait for all of LDS and for it)
  const int v0 = fresh(0);
  // (loaded values are taken as they are until they are used: an edit would wait for the load)
  int32_t kid, vid;
  uint2 kd, vd;  // dc_page_desc
  bool named = false, listed = false;  // the table names the pages that kid, vid are for; kd, vd are pages of the pools
  struct Raw {
    uint32_t kr[8], vr[8];
    uint16_t k_scale, k_bias, v_scale, v_bias;
    int k_kind, v_kind;
    bool k_affine, v_affine, counts;
  };
  Raw even, odds;  // (of even and of odd tiles)
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
    const uint32_t page = page_of(tile);
    const bool in = u_first + offset(tile) < it.kv_end && page < uint32_t(a.table_stride);
    kid = ks.table[(in ? int(page) : 0) + v0];
    vid = vs.table[(in ? int(page) : 0) + v0];
    named = in;
  };
  auto load_descs = [&]() __attribute__((always_inline)) {
    const int ki = uni(kid), vi = uni(vid);
    const bool in = named && uint32_t(ki) < uint32_t(ks.n_descs) && uint32_t(vi) < uint32_t(vs.n_descs);
    listed = in;
    kd = reinterpret_cast<const uint2*>(ks.descs)[(in ? ki : 0) + v0];
    vd = reinterpret_cast<const uint2*>(vs.descs)[(in ? vi : 0) + v0];
  };
  // The units of a tile, whose descriptors are at hand, and the descriptors and
  // ids of the next ones: those first, since loads come back in order and
  // waiting for them would wait for units issued ahead of them too.
  auto load_units = [&](int tile, Raw& raw) __attribute__((always_inline)) {
    const int u = u_first + offset(tile), slot = u - int(page_of(tile)) * P;
    const auto k = __builtin_bit_cast(dc_page_desc, uint2{uint32_t(uni(kd.x)), uint32_t(uni(kd.y))});
    const auto v = __builtin_bit_cast(dc_page_desc, uint2{uint32_t(uni(vd.x)), uint32_t(uni(vd.y))});
    raw.k_kind = unit_kind(ks, k, P, slot);
    raw.v_kind = unit_kind(vs, v, P, slot);
    raw.k_affine = k.format == DC_FMT_M0_AFFINE;
    raw.v_affine = v.format == DC_FMT_M0_AFFINE;
    // (tokens of the page behind its last and behind kv_end lie in its blob, but do not count)
    const int end = min(min(int(k.tokens), int(v.tokens)), slot + it.kv_end - u);
    const bool ok = listed && raw.k_kind != U_NONE && raw.v_kind != U_NONE;
    load_descs();
    load_ids(tile + 2);
    raw.counts = ok && slot + lt < end;
    if (!ok) raw.k_kind = raw.v_kind = U_NONE;
    load_unit<UNI>(ks, ks.arena + (uint64_t(k.block) << 8), a.items, raw.k_kind, raw.k_affine, slot, raw.kr, raw.k_scale, raw.k_bias);
    load_unit<UNI>(vs, vs.arena + (uint64_t(v.block) << 8), a.items, raw.v_kind, raw.v_affine, slot, raw.vr, raw.v_scale, raw.v_bias);
  };
  const int w_at[2] = {lds_at<CH>(ut, uc / 8), lds_at<CH>(ut, uc / 8 + 1)};  // of the unit's chunks in a tile
  auto write_tile = [&](int tile, const Raw& raw) __attribute__((always_inline)) {
    const int buf = tile & 1;
    const bool zero = !(raw.counts && has), border = RULE ? !all.whole(it.kv_begin + offset(tile), KT) : it.kv_begin + (tile + 1) * KT - 1 > sees_block;  // (border: uniform)
    uint32_t y[8];
    auto put = [&](uint8_t* to) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = zero ? 0 : y[k];
#pragma unroll
      for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(to + w_at[k]) = uint4{y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]};
    };
    unit_values(raw.k_kind, raw.k_affine, raw.kr, raw.k_scale, raw.k_bias, y);
    put(lds + buf * TILE);
    unit_values(raw.v_kind, raw.v_affine, raw.vr, raw.v_scale, raw.v_bias, y);
    if (border) {
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t e = ((y[k] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;  // sign bits: not finite
        any |= e;
        y[k] &= ~((e >> 15) * 0xffffu);
      }
      const uint32_t bits = fold_tokens<NT>(__ballot(any != 0 && !zero));
      if (lane < NT / 8) poison[buf][pg][tw * (NT / 8) + lane] = uint8_t(bits >> (8 * lane));
    }
    put(lds + (2 + buf) * TILE);
    const uint32_t bits = fold_tokens<NT>(__ballot(raw.counts));
    if (pg == 0 && lane < NT / 8) live[buf][tw * (NT / 8) + lane] = uint8_t(bits >> (8 * lane));
  };
  load_ids(0);
  load_descs();
  load_ids(1);
  load_units(0, even);
  load_units(1, odds);
  if constexpr (RULE) {  // (while the pages' rows are on their way)
    rule = row_rule(a, it, has_row, tok, head);
    mine = sight_of(a, it, it.row_begin + rows_at, min(it.row_begin + rows_at + 32, it.row_end));
    all = sight_of(a, it, it.row_begin, it.row_end);
  }

  // ---- queries: row col, channels 16 k + 8 half .. + 7 in LDS order
  h8v q[QW];
  {
    const int rr = has_row ? row : it.row_begin, rt = rr / a.n_q;  // (rows that do not exist: the first one's, as zeros)
    const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q) + int64_t(it.q_begin + rt) * a.q_token_stride +
                        int64_t(it.kv_head * a.n_q + rr - rt * a.n_q) * a.q_head_stride;
    uint32_t w[QW][4];
    load_rows<QW>(a, p, 8 * half, 16, has_row, hd, w);
    to_operands<QW>(a.dtype == DC_F16, a.sign, w, q);
  }
  const float c = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  f32x16 o[CB];
#pragma unroll
  for (int i = 0; i < CB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[i][v] = 0.f;

  write_tile(0, even);
  load_units(2, even);
  __syncthreads();
  auto step = [&](int i, Raw& next) __attribute__((always_inline)) {  // next: tile i + 1's
    if (i + 1 < tiles) {
      write_tile(i + 1, next);
      load_units(i + 3, next);
    }
    const uint8_t* const kt = lds + (i & 1) * TILE;
    const uint8_t* const vt = lds + (2 + (i & 1)) * TILE;
    const int u0 = it.kv_begin + offset(i);
    if (RULE ? !all.whole(u0, KT) : u0 + KT - 1 > sees_block) {
      const uint32_t* const bad = reinterpret_cast<const uint32_t*>(poison[i & 1][0]);
#pragma unroll 1
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll 1
        for (uint32_t bits = bad[tb] | (PG > 1 ? bad[TB + tb] : 0); bits != 0; bits &= bits - 1) {
          const int u = u0 + 32 * tb + __builtin_ctz(bits), page = u / P;
          __syncthreads();
          if (tid < HDP) {
            const dc_page_desc d = a.vpool.descs[a.v_table[table + page]];
            const BlobLayout L = blob_layout(d.format, d.bits, a.vpool.geometry);
            const float x = tid < hd ? page_value(blob_ptr(a.vpool.arena, d), d, L, a.vpool.geometry, u - page * P, tid) : 0.f;
            odd[tid] = float(_Float16(x));
          }
          __syncthreads();
#pragma unroll
          for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const float x = odd[32 * (cb0 + j) + 8 * (v / 4) + kPerm[4 * half + v % 4]];
              if (seen(u) && !__builtin_isfinite(x)) o[j][v] += x;
            }
        }
    }
    if (wave_rows && (!RULE || mine.some(u0, KT))) {
      const uint32_t* const on = reinterpret_cast<const uint32_t*>(live[i & 1]);
      f32x16 s[TB];
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[tb][v] = 0.f;
      // (operands are read kAhead instructions ahead; the scheduler would read them one ahead)
      const int k_at = fresh(lds_at<CH>(col, half));
      auto key = [&](int n) { return *reinterpret_cast<const h8v*>(kt + (k_at ^ (32 * (n / TB))) + 32 * (n % TB) * CH * 16); };
      h8v ka[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ka[n] = key(n);
#pragma unroll
      for (int n = 0; n < QW * TB; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        s[n % TB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[n % kAhead], q[n / TB], s[n % TB], 0, 0, 0);
        if (n + kAhead < QW * TB) ka[n % kAhead] = key(n + kAhead);
      }
      if constexpr (RULE) shape_scores<RULE == kCapped, false>(a, c, rule, u0 + 4 * half, s);
      bool masked = RULE ? !mine.whole(u0, KT) : u0 + KT - 1 > sees_all;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) masked = masked || on[tb] != ~0u;
      if (masked) {
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) {
          const uint32_t bits = on[tb] >> (4 * half);
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int t = 8 * (v / 4) + v % 4;
            s[tb][v] = ((bits >> t) & 1) && seen(u0 + 32 * tb + t + 4 * half) ? s[tb][v] : -INFINITY;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, s[tb][v]);
      top = half_max(top) * (RULE ? 1.f : c);
      if (__any(top > m + kLazy || (m == -INFINITY && top > m))) {
        const float mn = fmaxf(m, top);
        const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[j][v] *= f;
      }
      const float mu = (m == -INFINITY ? 0.f : m) - kLift;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[tb][v] = __builtin_amdgcn_exp2f(RULE ? s[tb][v] - mu : fmaf(s[tb][v], c, -mu));
      const int v_at = fresh(lds_at<CH>(4 * half + ((lane & 15) >> 2), 4 * cb0 + ((lane & 16) >> 3) + ((lane & 3) >> 1)) + 8 * (lane & 1));
      auto value = [&](int n) {
        // token 16 (n / CB) + 4 half + lane % 16 / 4 (+ 8), channel 32 (cb0 + n % CB) + lane / 16 % 2 * 16 + 4 (lane % 4):
        // eight tokens on, the row's chunks are exchanged by 2 more
        s4v x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s4v*)(vt + (v_at ^ (64 * (n % CB) + 32 * e)) + (16 * (n / CB) + 8 * e) * CH * 16));
        return __builtin_bit_cast(h8v, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
      };
      h8v va[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) va[n] = value(n);
#pragma unroll
      for (int st = 0; st < 2 * TB; ++st) {
        h8v p;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          // (the sum takes the rounded weights, which are those the values get)
          const h2v e = {(_Float16)s[st / 2][8 * (st % 2) + k], (_Float16)s[st / 2][8 * (st % 2) + k + 1]};
          l = __builtin_amdgcn_fdot2(e, h2v{(_Float16)1.f, (_Float16)1.f}, l, false);
          p[k] = e[0];
          p[k + 1] = e[1];
        }
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          const int n = st * CB + j;
          __builtin_amdgcn_sched_barrier(0x6);  // (vector and scalar arithmetic may cross)
          o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[n % kAhead], p, o[j], 0, 0, 0);
          if (n + kAhead < 2 * TB * CB) va[n % kAhead] = value(n + kAhead);
        }
      }
    }
    __syncthreads();
  };
  for (int i = 0; i < tiles; i += 2) {
    step(i, odds);
    if (i + 1 < tiles) step(i + 1, even);
  }
  if (!has_row) return;
  l = half_sum(l);
  const bool part = it.partial >= 0;
  const float inv = part ? 1.f : l == 0.f ? 0.f : 1.f / l;
  const int64_t pr = int64_t(it.partial) + rows_at + col;
  if (part && half == 0 && cb0 == 0) {
    a.part_ml[2 * pr] = m;
    a.part_ml[2 * pr + 1] = l;
  }
  uint16_t* const out = reinterpret_cast<uint16_t*>(a.out) + int64_t(it.q_begin + tok) * a.o_token_stride + int64_t(head) * a.o_head_stride;
#pragma unroll
  for (int j = 0; j < CB; ++j)
#pragma unroll
    for (int v = 0; v < 16; v += 4) {
      // this half's channels 4 half .. + 3 of the group, from the LDS order
      const float2 x = swap_halves(o[j][v], o[j][v + 1]), y = swap_halves(o[j][v + 2], o[j][v + 3]);
      const float r[4] = {x.x * inv, y.x * inv, x.y * inv, y.y * inv};
      const int ch = 32 * (cb0 + j) + 2 * v + 4 * half;
      if (ch >= hd) continue;
      if (part) {
        *reinterpret_cast<float4*>(a.part_o + pr * hd + ch) = float4{r[0], r[1], r[2], r[3]};
        continue;
      }
      uint32_t w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        w[k] = a.dtype == DC_F16 ? __builtin_bit_cast(uint32_t, h2v{(_Float16)r[2 * k], (_Float16)r[2 * k + 1]})
                                 : __builtin_bit_cast(uint32_t, b2v{(__bf16)r[2 * k], (__bf16)r[2 * k + 1]});
      if (a.o_vec) {
        *reinterpret_cast<uint2*>(out + ch) = uint2{w[0], w[1]};
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) out[ch + k] = uint16_t(w[k / 2] >> (16 * (k % 2)));
      }
    }
}

// ---- few rows -----------------------------------------------------------------

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kFewTile = 32;   // tokens a wavefront takes at a time
constexpr int kFewWaves = 4;

// Bytes of the wavefronts' joined rows, and whether each has its own: two blocks
// share a compute unit's 160 KiB.
constexpr bool few_joined_apart(int hdp, int nb) { return kFewWaves * 16 * nb * (hdp + 4) * 4 <= 72 * 1024; }
constexpr int few_joined_bytes(int hdp, int nb) { return (few_joined_apart(hdp, nb) ? kFewWaves : 1) * 16 * nb * (hdp + 4) * 4; }

// As lds_at, for tiles whose reads take two chunks of eight tokens at once.
template <int CH>
__device__ __forceinline__ int few_at(int t, int ch) {
  const int x = CH >= 16 ? ((t & 3) << 2) | (((t >> 2) & 1) << 1) | ((t >> 3) & 1)
                         : (((t >> 1) & 1) << 2) | (((t >> 2) & 1) << 1) | ((t >> 3) & 1);
  return (t * CH + (ch ^ x)) * 16;
}

// Maximum over the four lanes of equal lane % 16, in all of them.
__device__ __forceinline__ float quarter_max(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t x = r[0], y = r[1];
  return half_max(fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)));
}
__device__ __forceinline__ float quarter_sum(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t x = r[0], y = r[1];
  return half_sum(__builtin_bit_cast(float, x) + __builtin_bit_cast(float, y));
}

// Eight values of a 4-bit word, of two 8-bit words or of four fp16 words, in LDS order.
__device__ __forceinline__ void eight4(uint32_t r, uint32_t zero, h2v s, h2v b, uint32_t (&y)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = scaled((r >> (4 * i)) & 0x000f000fu, zero, s, b);
}
__device__ __forceinline__ void eight8(uint32_t r0, uint32_t r1, uint32_t zero, h2v s, h2v b, uint32_t (&y)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = scaled(__builtin_amdgcn_perm(r1, r0, 0x0c040c00u + 0x00010001u * i), zero, s, b);
}
__device__ __forceinline__ void eight_halves(uint4 r, uint32_t (&y)[4]) {
  y[0] = __builtin_amdgcn_perm(r.z, r.x, 0x05040100u);
  y[1] = __builtin_amdgcn_perm(r.z, r.x, 0x07060302u);
  y[2] = __builtin_amdgcn_perm(r.w, r.y, 0x05040100u);
  y[3] = __builtin_amdgcn_perm(r.w, r.y, 0x07060302u);
}
__device__ __forceinline__ uint32_t zero_of(int kind, bool affine) {
  return twice(affine ? 0xe400u : kind == U_B4 ? 0xe407u : 0xe47fu);
}

}  // namespace

// A few query rows (at most 16 NB: a decode's, or drafted tokens') against a
// long range: bound by reading the pages, so the four wavefronts split the
// range among them, 32 tokens at a time, and never wait for each other until
// they join at the end.  Keys go from the page's words to the matrix operand
// in registers (a lane's eight channels are one 4-bit word); values pass
// through the wavefront's own LDS to be read transposed.  While a tile is
// worked on, the next one's words are on their way.  16-row operands: S^T =
// K Q^T leaves a row's logits in four lanes, again in the order in which the
// values' operand is read.
// KW: words of a key operand that are read ahead (4: also fp16 rows; 2: codes
// only, and fp16 rows when they are needed; 1: as 2, 4-bit codes only).  UNI: a tile's tokens lie in one page.
// KW 1 is for pools of 4-bit codes in groups of 32 (and fp16 pages between them):
// a token's scales lie side by side, and are one load.  The loads' issue is half of
// a long range's time, so what counts is how few they are: a decode of 8
// sequences of 32768 tokens at head_dim 256, 336 MB, 172 -> 131 us.  Where such
// pools hold fp16 pages for the most part, those are read where they are used: 8
// sequences of 16384 tokens, keys and values both fp16, 34 -> 38 us at head_dim 64 and 56 -> 60
// at 128, but 151 -> 115 at 256; with one of the two in 4 bits 43 -> 44, 50 -> 48 at 128.
template <int HDP, int NB, int KW, bool UNI, bool WHOLE, int RULE>
__global__ void __launch_bounds__(64 * kFewWaves, 2) attend_few_kernel(ChunkArgs a) {
  constexpr int CH = HDP / 8, KS = HDP / 32, CB = HDP / 16, TILE = kFewTile * HDP * 2;
  constexpr int VC = HDP / 2, VU = VC / 32;  // a lane's value channels, in units of 32
  constexpr int PB = UNI ? 1 : 2;            // pages that a lane follows: its tokens of each 16
  constexpr int COMB = HDP + 4;
  constexpr bool C4 = KW == 1;
  static_assert(!C4 || (UNI && WHOLE), "a page's tile, whole rows of scales");
  constexpr bool QL = NB * HDP >= 256;       // the queries stay in LDS (registers are for the output and the next tile)
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // values of each wavefront, then queries; at the end the joined rows
  __shared__ float ml[kFewWaves][16 * NB][2];
  __shared__ float odd[kFewWaves][HDP];

  const dc_chunk_item it = a.items[blockIdx.x];
  if (!chunk_item_ok(it, a) || it.row_end - it.row_begin > 16 * NB) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int hd = WHOLE ? HDP : a.kpool.geometry.head_dim, P = a.kpool.geometry.page_capacity;
  const int rows = it.row_end - it.row_begin;

  int sees[NB];
  RowRule rule[NB];
  Sight all;
  int gap_tile = INT32_MAX, gap_len = 0;
  if constexpr (RULE) {
    all = sight_of(a, it, it.row_begin, it.row_end);
    const int2 gap = item_gap(a, it, blockIdx.x);
    if (gap.x >= 0) gap_tile = (gap.x - it.kv_begin) / kFewTile, gap_len = gap.y - gap.x;
  }
  h8v q[QL ? 1 : NB][QL ? 1 : KS];
  uint8_t* const ql = lds + kFewWaves * TILE;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = it.row_begin + 16 * n + col;
    const bool has_row = row < it.row_end;
    sees[n] = has_row ? it.first + row / a.n_q : -1;
    if constexpr (RULE) rule[n] = row_rule(a, it, has_row, row / a.n_q, it.kv_head * a.n_q + row % a.n_q);
    const int rr = has_row ? row : it.row_begin, rt = rr / a.n_q;  // (rows that do not exist: the first one's, as zeros)
    const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q) + int64_t(it.q_begin + rt) * a.q_token_stride +
                        int64_t(it.kv_head * a.n_q + rr - rt * a.n_q) * a.q_head_stride;
    uint32_t w[KS][4];
    h8v x[KS];
    load_rows<KS>(a, p, 8 * g, 32, has_row, hd, w);
    to_operands<KS>(a.dtype == DC_F16, a.sign, w, x);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if constexpr (!QL)
        q[n][k] = x[k];
      else if (wave == 0)
        *reinterpret_cast<h8v*>(ql + lds_at<CH>(16 * n + col, 4 * k + g)) = x[k];
    }
  }
  if constexpr (QL) __syncthreads();
  auto query = [&](int n, int k, int q_at) {
    if constexpr (QL)
      return *reinterpret_cast<const h8v*>(ql + (q_at ^ (64 * k)) + 16 * n * CH * 16);
    else
      return q[n][k];
  };
  auto seen = [&](int n, int u) { return RULE ? rule[n].sees(u) : u <= sees[n]; };
  // tokens from the item's first to a tile's
  auto offset = [&](int tile) { return tile * kFewTile + (RULE && tile >= gap_tile ? gap_len : 0); };
  const int sees_first = it.first + it.row_begin / a.n_q;  // the least of the rows'

  // ---- the pages: keys of token 16 b + col, channels 32 k + 8 g .. + 7; values of
  // token lane % 32, channels VC (lane / 32) ..
  const int64_t table = (int64_t(it.seq) * a.n_kv_heads + it.kv_head) * a.table_stride;
  const int kt0 = UNI ? col : 0, vt0 = UNI ? (lane & 31) : 0;
  const Side ks = make_side(a.kpool, a.k_table + table, 0, 0), vs = make_side(a.vpool, a.v_table + table, 0, 0);
  const uint32_t kgs = a.kpool.geometry.group_size, vgs = a.vpool.geometry.group_size;
  const uint32_t k_plane = a.kpool.geometry.layout == 0 ? P * kgs / 2 : kgs / 2;  // from a group's codes to the next one's
  const uint32_t v_plane = a.vpool.geometry.layout == 0 ? P * vgs / 2 : vgs / 2;
  auto uni = [](int x) { return UNI ? __builtin_amdgcn_readfirstlane(x) : x; };
  auto token = [&](int tile, int b) { return it.kv_begin + offset(tile) + (UNI ? 0 : 16 * b + col); };
  auto page_of = [&](int u) { return uint32_t((uint64_t(uint32_t(u)) * a.page_mul) >> a.page_shift); };
  // (a zero in a vector register: ids and descriptors are then read by vector
  // loads, which come back in order; a scalar load in flight would make the next
  // wait for LDS wait for all of LDS and for it)
  const int v0 = fresh(0);
  // (loaded values are taken as they are until they are used: an edit would wait for the load)
  int32_t kid[PB], vid[PB];
  uint2 kd[PB], vd[PB];
  bool named[PB], listed[PB];  // the table names the pages that kid, vid are for; kd, vd are pages of the pools
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      const int u = token(tile, b);
      const uint32_t page = page_of(u);
      const bool in = u < it.kv_end && page < uint32_t(a.table_stride);
      kid[b] = ks.table[(in ? int(page) : 0) + v0];
      vid[b] = vs.table[(in ? int(page) : 0) + v0];
      named[b] = in;
    }
  };
  auto load_descs = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      const int ki = uni(kid[b]), vi = uni(vid[b]);
      const bool in = named[b] && uint32_t(ki) < uint32_t(ks.n_descs) && uint32_t(vi) < uint32_t(vs.n_descs);
      listed[b] = in;
      kd[b] = reinterpret_cast<const uint2*>(ks.descs)[(in ? ki : 0) + v0];
      vd[b] = reinterpret_cast<const uint2*>(vs.descs)[(in ? vi : 0) + v0];
    }
  };
  // The raw tile: where it is and what its pages hold (of the lane's tokens 16 b + col, or of all where UNI) ...
  struct Place { const uint8_t *k, *v; int k_kind, v_kind, slot, end; bool k_affine, v_affine; };
  Place at[PB];
  uint32_t on = 0;  // one bit per token: it counts
  auto locate = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      const int u = token(tile, b);
      const auto k = __builtin_bit_cast(dc_page_desc, uint2{uint32_t(uni(kd[b].x)), uint32_t(uni(kd[b].y))});
      const auto v = __builtin_bit_cast(dc_page_desc, uint2{uint32_t(uni(vd[b].x)), uint32_t(uni(vd[b].y))});
      Place& x = at[b];
      x.slot = u - int(page_of(u)) * P;
      x.k_kind = unit_kind(ks, k, P, x.slot);
      x.v_kind = unit_kind(vs, v, P, x.slot);
      // (tokens of the page behind its last and behind kv_end lie in its blob, but do not count)
      x.end = min(min(int(k.tokens), int(v.tokens)) - x.slot, it.kv_end - u);
      if (!listed[b] || x.k_kind == U_NONE || x.v_kind == U_NONE || x.end <= 0) {
        x.k_kind = x.v_kind = U_NONE;
        x.end = 0;
      }
      x.k_affine = k.format == DC_FMT_M0_AFFINE;
      x.v_affine = v.format == DC_FMT_M0_AFFINE;
      x.k = ks.arena + (uint64_t(k.block) << 8);
      x.v = vs.arena + (uint64_t(v.block) << 8);
    }
    if constexpr (UNI)
      on = at[0].end >= 32 ? ~0u : (1u << at[0].end) - 1u;
    else
      on = uint32_t(__ballot(at[0].end > 0) & 0xffffu) | uint32_t(__ballot(at[PB - 1].end > 0) & 0xffffu) << 16;
  };
  // the place of the lane's value token, which is one of its key tokens: 16 (lane / 16 % 2) + col
  auto value_place = [&]() __attribute__((always_inline)) {
    Place x = at[0];
    if constexpr (!UNI) {
      const bool second = (lane & 16) != 0;
      const Place& y = at[PB - 1];
      x.v = second ? y.v : x.v;
      x.v_kind = second ? y.v_kind : x.v_kind;
      x.slot = second ? y.slot : x.slot;
      x.v_affine = second ? y.v_affine : x.v_affine;
    }
    return x;
  };
  // ... and its words; scales and biases as they are
  uint32_t kr[2][KS][KW], vr[VU][C4 ? 4 : 8];
  uint16_t k_scale[2][KS], k_bias[2][KS], v_scale[VU], v_bias[VU];
  uint32_t ks_row[2][KS / 2], kb_row[2][KS / 2], vs_row[(VU + 1) / 2], vb_row[(VU + 1) / 2];  // (C4: in pairs)
  // N halves side by side, in pairs
  auto halves = [](const PageLoad<UNI>& p, uint32_t off, uint32_t at, auto n, uint32_t* to) __attribute__((always_inline)) {
    constexpr int N = decltype(n)::value;
    if constexpr (N == 1) {
      to[0] = p.u16(off, at);
    } else if constexpr (N == 2) {
      to[0] = p.u32(off, at);
    } else if constexpr (N == 4) {
      const uint2 x = p.u64(off, at);
      to[0] = x.x; to[1] = x.y;
    } else {
      const uint4 x = p.u128(off, at);
      to[0] = x.x; to[1] = x.y; to[2] = x.z; to[3] = x.w;
    }
  };
  // half i of such pairs, twice
  auto half_of = [](const uint32_t* row, int i) { return __builtin_amdgcn_perm(row[i / 2], row[i / 2], i % 2 ? 0x03020302u : 0x01000100u); };
  // the lane's offsets in a page, from its tile's first token (from its own where its tokens lie in several pages)
  const uint32_t k4 = kt0 * ks.token4 + 4 * g, k_sc = kt0 * ks.groups2, k16 = kt0 * ks.row2 + 16 * g;
  const uint32_t vc0 = VC * (lane >> 5), v16 = vt0 * vs.row2 + 2 * vc0;
  uint32_t v4[VU], v_sc[VU];
#pragma unroll
  for (int u = 0; u < VU; ++u) {
    const uint32_t c = int(vc0 + 32 * u) < hd ? vc0 + 32 * u : 0, gr = c / vgs;  // (channels past head_dim: the first ones')
    v4[u] = vt0 * vs.token4 + gr * v_plane + (c - gr * vgs) / 2;
    v_sc[u] = vt0 * vs.groups2 + 2 * gr;
  }
  auto load_keys = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const Place& x = at[UNI ? 0 : b];
      const uint32_t slot = x.slot + (UNI ? 16 * b : 0);
      // (fp16 rows are read here where KW is 4, else where they are used)
      const bool f16 = x.k_kind == U_F16;
      const PageLoad<UNI> p{x.k, a.items, x.k_kind != U_NONE};
      const uint32_t sh = x.k_kind == U_B8, lane_at = f16 ? k16 : k4 << sh, lane_s = f16 ? 0 : k_sc;
      const uint32_t codes = f16 ? slot * ks.row2 : (slot * ks.token4) << sh, scales = f16 ? 0 : (ks.scales4 << sh) + slot * ks.groups2;
      const uint32_t gap = x.k_affine && !f16 ? ks.gap : 0;
      if constexpr (C4) {
#pragma unroll
        for (int k = 0; k < KS; ++k) kr[b][k][0] = p.u32(codes + (f16 ? 0 : k * k_plane), f16 ? 0 : k4);
        halves(p, scales, lane_s, std::integral_constant<int, KS>{}, ks_row[b]);
        halves(p, scales + gap, lane_s, std::integral_constant<int, KS>{}, kb_row[b]);
        continue;
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint32_t c = 32 * k < hd ? 32 * k : 0, gr = c / kgs;  // (channels past head_dim: the first ones')
        const uint32_t o = codes + (f16 ? 2 * c : (gr * k_plane + (c - gr * kgs) / 2) << sh);
        if constexpr (KW == 4) {
          const uint4 r = p.u128(o, lane_at);
          kr[b][k][0] = r.x; kr[b][k][1] = r.y; kr[b][k][2] = r.z; kr[b][k][3] = r.w;
        } else if constexpr (KW == 2) {
          const uint2 r = p.u64(o, lane_at);
          kr[b][k][0] = r.x; kr[b][k][1] = r.y;
        }
        k_scale[b][k] = p.u16(scales + (f16 ? 0 : 2 * gr), lane_s);
        k_bias[b][k] = p.u16(scales + (f16 ? 0 : 2 * gr) + gap, lane_s);
      }
    }
  };
  auto load_values = [&]() __attribute__((always_inline)) {
    const Place x = value_place();
    const bool f16 = x.v_kind == U_F16;  // (read where they are used)
    const PageLoad<UNI> p{x.v, a.items, x.v_kind != U_NONE && !f16};
    const uint32_t sh = x.v_kind == U_B8, codes = (x.slot * vs.token4) << sh, scales = (vs.scales4 << sh) + x.slot * vs.groups2;
    const uint32_t gap = x.v_affine ? vs.gap : 0;
    if constexpr (C4) {
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        const uint4 r = p.u128(codes, v4[u]);
        vr[u][0] = r.x; vr[u][1] = r.y; vr[u][2] = r.z; vr[u][3] = r.w;
      }
      halves(p, scales, v_sc[0], std::integral_constant<int, VU>{}, vs_row);
      halves(p, scales + gap, v_sc[0], std::integral_constant<int, VU>{}, vb_row);
      return;
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const uint4 r = p.u128(codes, v4[u] << sh), t = p.u128(codes + (sh ? 16 : 0), v4[u] << sh);
      vr[u][0] = r.x; vr[u][1] = r.y; vr[u][2] = r.z; vr[u][3] = r.w;
      if constexpr (!C4) vr[u][4] = t.x, vr[u][5] = t.y, vr[u][6] = t.z, vr[u][7] = t.w;
      v_scale[u] = p.u16(scales, v_sc[u]);
      v_bias[u] = p.u16(scales + gap, v_sc[u]);
    }
  };

  const int tiles = (it.kv_end - it.kv_begin - gap_len + kFewTile - 1) / kFewTile;
  uint8_t* const vt = lds + wave * TILE;
  const float c = a.scale * kLog2e;
  float m[NB], l[NB];
  f32x4 o[NB][CB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int j = 0; j < CB; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  load_ids(wave);
  load_descs();
  locate(wave);
  load_values();
  load_keys();
  load_ids(wave + kFewWaves);
  load_descs();
  load_ids(wave + 2 * kFewWaves);
  for (int i = wave; i < tiles; i += kFewWaves) {
    const int u0 = it.kv_begin + offset(i);
    const bool border = RULE ? !all.whole(u0, kFewTile) : u0 + kFewTile - 1 > sees_first;  // (uniform)
    const uint32_t live = on;
    // ---- values to LDS
    uint32_t bad = 0;
    {
      const Place x = value_place();
      const bool counts = ((live >> (lane & 31)) & 1) != 0;
      const uint32_t zero = zero_of(x.v_kind, x.v_affine);
      const int w_at = fresh(few_at<CH>(lane & 31, vc0 / 8));
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        uint32_t y[4][4];
        const bool in = int(vc0 + 32 * u) < hd;
        const h2v s = __builtin_bit_cast(h2v, C4 ? half_of(vs_row, u) : twice(v_scale[u]));
        const h2v b = __builtin_bit_cast(h2v, !x.v_affine ? 0u : C4 ? half_of(vb_row, u) : twice(v_bias[u]));
        if (x.v_kind == U_B4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) eight4(vr[u][e], zero, s, b, y[e]);
        } else if (!C4 && x.v_kind == U_B8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) eight8(vr[u][2 * e % (C4 ? 4 : 8)], vr[u][(2 * e + 1) % (C4 ? 4 : 8)], zero, s, b, y[e]);
        } else if (x.v_kind == U_F16 && in) {
          const PageLoad<UNI> p{x.v, a.items, true};
#pragma unroll
          for (int e = 0; e < 4; ++e) eight_halves(p.u128(x.slot * vs.row2 + 64 * u + 16 * e, v16), y[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e][0] = y[e][1] = y[e][2] = y[e][3] = 0;
        }
        if (live != ~0u || HDP > hd) {
          const bool keep = counts && in;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) y[e][k] = keep ? y[e][k] : 0;
        }
        if (border) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t f = ((y[e][k] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;  // sign bits: not finite
              bad |= f;
              y[e][k] &= ~((f >> 15) * 0xffffu);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(vt + (w_at ^ (64 * u + 16 * e))) = uint4{y[e][0], y[e][1], y[e][2], y[e][3]};
      }
    }
    // ---- S^T
    uint32_t y[2][KS][4];  // the keys' operands
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const Place& x = at[UNI ? 0 : b];
      const uint32_t zero = zero_of(x.k_kind, x.k_affine);
      if (x.k_kind == U_B4) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
          eight4(kr[b][k][0], zero, __builtin_bit_cast(h2v, C4 ? half_of(ks_row[b], k) : twice(k_scale[b][k])),
                 __builtin_bit_cast(h2v, !x.k_affine ? 0u : C4 ? half_of(kb_row[b], k) : twice(k_bias[b][k])), y[b][k]);
      } else if (!C4 && x.k_kind == U_B8) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
          eight8(kr[b][k][0], kr[b][k][1 % KW], zero, __builtin_bit_cast(h2v, twice(k_scale[b][k])),
                 __builtin_bit_cast(h2v, x.k_affine ? twice(k_bias[b][k]) : 0u), y[b][k]);
      } else if (x.k_kind == U_F16) {
        if constexpr (KW == 4) {
#pragma unroll
          for (int k = 0; k < KS; ++k) eight_halves(uint4{kr[b][k][0], kr[b][k][1], kr[b][k][2], kr[b][k][3]}, y[b][k]);
        } else {
          const PageLoad<UNI> p{x.k, a.items, true};
          const uint32_t rows = (x.slot + (UNI ? 16 * b : 0)) * ks.row2;
#pragma unroll
          for (int k = 0; k < KS; ++k) eight_halves(p.u128(rows + (32 * k < hd ? 64 * k : 0), k16), y[b][k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) y[b][k][0] = y[b][k][1] = y[b][k][2] = y[b][k][3] = 0;
      }
    }
    const int q_at = fresh(lds_at<CH>(col, g));
    f32x4 s[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (HDP > 64 && 32 * k >= hd) break;  // (uniform; channels past head_dim)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const h8v x = query(n, k, q_at);
#pragma unroll
        for (int b = 0; b < 2; ++b)
          s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              __builtin_bit_cast(h8v, uint4{y[b][k][0], y[b][k][1], y[b][k][2], y[b][k][3]}), x, s[n][b], 0, 0, 0);
      }
    }
    locate(i + kFewWaves);
    load_descs();  // (ahead of the words: loads come back in order)
    load_ids(i + 3 * kFewWaves);
    load_values();
    load_keys();
    // ---- softmax: tokens 16 b + 4 g + v of row col of each block
    h8v p[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if constexpr (RULE) shape_scores<RULE == kCapped, false>(a, c, rule[n], u0 + 4 * g, s[n]);
      if (border || live != ~0u) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int t = 16 * b + 4 * g + v;
            s[n][b][v] = ((live >> t) & 1) && seen(n, u0 + t) ? s[n][b][v] : -INFINITY;
          }
      }
      float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                        fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      top = quarter_max(top) * (RULE ? 1.f : c);
      if (__any(top > m[n] + kLazy || (m[n] == -INFINITY && top > m[n]))) {
        const float mn = fmaxf(m[n], top);
        const float f = m[n] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= f;
#pragma unroll
        for (int j = 0; j < CB; ++j) o[n][j] *= f;
      }
      const float mu = (m[n] == -INFINITY ? 0.f : m[n]) - kLift;
#pragma unroll
      for (int v = 0; v < 8; v += 2) {
        const h2v e = {(_Float16)__builtin_amdgcn_exp2f(RULE ? s[n][v / 4][v % 4] - mu : fmaf(s[n][v / 4][v % 4], c, -mu)),
                       (_Float16)__builtin_amdgcn_exp2f(RULE ? s[n][v / 4][v % 4 + 1] - mu : fmaf(s[n][v / 4][v % 4 + 1], c, -mu))};
        l[n] = __builtin_amdgcn_fdot2(e, h2v{(_Float16)1.f, (_Float16)1.f}, l[n], false);
        p[n][v] = e[0];
        p[n][v + 1] = e[1];
      }
    }
    // ---- values that are not finite, to the rows that see them
    if (border) {
      uint64_t who = __ballot(bad != 0);
      for (uint32_t bits = uint32_t(who) | uint32_t(who >> 32); bits != 0; bits &= bits - 1) {
        const int u = u0 + __builtin_ctz(bits), page = u / P;
        const dc_page_desc d = a.vpool.descs[vs.table[page]];
        const BlobLayout L = blob_layout(d.format, d.bits, a.vpool.geometry);
        for (int ch = lane; ch < HDP; ch += 64)
          odd[wave][ch] = ch < hd ? float(_Float16(page_value(blob_ptr(a.vpool.arena, d), d, L, a.vpool.geometry, u - page * P, ch))) : 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float x = odd[wave][16 * j + 8 * (g / 2) + kPerm[4 * (g % 2) + v]];
#pragma unroll
            for (int n = 0; n < NB; ++n)
              if (seen(n, u) && !__builtin_isfinite(x)) o[n][j][v] += x;
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
    // ---- O^T
    const int v_at = fresh(few_at<CH>(4 * g + ((lane & 15) >> 2), (lane & 3) >> 1) + 8 * (lane & 1));
    auto value = [&](int j) {  // tokens 4 g .. + 3 and 16 on, channels 16 j ..
      s4v x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(vt + (v_at ^ (32 * j)) + 16 * e * CH * 16));
      return __builtin_bit_cast(h8v, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
    };
    h8v va[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) va[j] = value(j);
#pragma unroll
    for (int j = 0; j < CB; ++j) {
      __builtin_amdgcn_sched_barrier(0x6);  // (vector and scalar arithmetic may cross)
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[j % kAhead], p[n], o[n][j], 0, 0, 0);
      if (j + kAhead < CB) va[j % kAhead] = value(j + kAhead);
    }
  }
  // ---- join the wavefronts, in order
  float* const comb = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] = quarter_sum(l[n]);
    if (g == 0) {
      ml[wave][16 * n + col][0] = m[n];
      ml[wave][16 * n + col][1] = l[n];
    }
  }
  __syncthreads();
  // (each into rows of its own where those of all four fit, else one after another: a turn
  // costs a barrier and a pass over LDS, 2 us of a short range's 20 in all)
  constexpr int APART = few_joined_apart(HDP, NB) ? 16 * NB * COMB : 0;
  for (int w = 0; w < (APART ? 1 : kFewWaves); ++w) {
    if (APART || wave == w) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int r = 16 * n + col;
        const float top = fmaxf(fmaxf(ml[0][r][0], ml[1][r][0]), fmaxf(ml[2][r][0], ml[3][r][0]));
        const float f = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float& x = comb[wave * APART + r * COMB + 16 * j + 8 * (g / 2) + kPerm[4 * (g % 2) + v]];
            // (a wavefront that saw no token holds zeros, or what a value that is not finite left)
            const float y = m[n] == -INFINITY ? o[n][j][v] : o[n][j][v] * f;
            x = APART || w == 0 ? y : x + y;
          }
      }
    }
    __syncthreads();
  }
  const bool part = it.partial >= 0;
  for (int i = tid; i < rows * (HDP / 4); i += 64 * kFewWaves) {
    const int r = i / (HDP / 4), ch = 4 * (i % (HDP / 4));
    if (ch >= hd) continue;
    const float top = fmaxf(fmaxf(ml[0][r][0], ml[1][r][0]), fmaxf(ml[2][r][0], ml[3][r][0]));
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
      sum += ml[w][r][0] == -INFINITY ? ml[w][r][1] : ml[w][r][1] * __builtin_amdgcn_exp2f(ml[w][r][0] - top);
    float4 x = *reinterpret_cast<const float4*>(comb + r * COMB + ch);
    if constexpr (APART != 0) {
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(comb + w * APART + r * COMB + ch);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
    }
    if (part) {
      const int64_t pr = int64_t(it.partial) + r;
      *reinterpret_cast<float4*>(a.part_o + pr * hd + ch) = x;
      if (ch == 0) {
        a.part_ml[2 * pr] = top;
        a.part_ml[2 * pr + 1] = sum;
      }
      continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int row = it.row_begin + r, tok = row / a.n_q, head = it.kv_head * a.n_q + (row - tok * a.n_q);
    uint16_t* const out = reinterpret_cast<uint16_t*>(a.out) + int64_t(it.q_begin + tok) * a.o_token_stride +
                          int64_t(head) * a.o_head_stride + ch;
    const float v[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w[k] = a.dtype == DC_F16 ? __builtin_bit_cast(uint32_t, h2v{(_Float16)v[2 * k], (_Float16)v[2 * k + 1]})
                               : __builtin_bit_cast(uint32_t, b2v{(__bf16)v[2 * k], (__bf16)v[2 * k + 1]});
    if (a.o_vec) {
      *reinterpret_cast<uint2*>(out) = uint2{w[0], w[1]};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = uint16_t(w[k / 2] >> (16 * (k % 2)));
    }
  }
}

// A kernel's dynamic LDS limit, raised once on every device that launches it.
struct LdsLimit {
  std::atomic<uint64_t> raised{0};
  int raise(const void* kernel, int bytes, const char* what) {
    int device = 0;
    if (int rc = check_hip(hipGetDevice(&device), what)) return rc;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (raised.load(std::memory_order_acquire) & bit)) return DC_OK;
    if (int rc = check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), what)) return rc;
    raised.fetch_or(device < 64 ? bit : 0, std::memory_order_release);
    return DC_OK;
  }
};

template <typename T, int HDP, int KT, int RULE>
static int launch_chunk(const ChunkArgs& a, hipStream_t stream) {
  constexpr int bytes = 2 * KT * HDP * int(sizeof(T)) + 16;
  static LdsLimit limit;
  if (int rc = limit.raise(reinterpret_cast<const void*>(&attend_chunk_kernel<T, HDP, KT, RULE>), bytes, "attend_chunk_kernel LDS")) return rc;
  hipLaunchKernelGGL((attend_chunk_kernel<T, HDP, KT, RULE>), item_grid(a.n_items, kChunkRows / 128), dim3(256), bytes, stream, a);
  return check_hip(hipGetLastError(), "attend_chunk_kernel launch");
}

template <int HDP, int KT, bool UNI, int CS, bool WHOLE, int RULE>
static int launch_chunk16_as(const ChunkArgs& a, hipStream_t stream) {
  constexpr int bytes = 4 * KT * HDP * 2;
  static LdsLimit limit;
  if (int rc = limit.raise(reinterpret_cast<const void*>(&attend_chunk16_kernel<HDP, KT, UNI, CS, WHOLE, RULE>), bytes, "attend_chunk16_kernel LDS")) return rc;
  hipLaunchKernelGGL((attend_chunk16_kernel<HDP, KT, UNI, CS, WHOLE, RULE>), item_grid(a.n_items, CS), dim3(512), bytes, stream, a);
  return check_hip(hipGetLastError(), "attend_chunk16_kernel launch");
}

template <int HDP, int KT, int CS, int RULE>
static int launch_chunk16(const ChunkArgs& a, hipStream_t stream) {
  if (a.kpool.geometry.page_capacity % (KT < 64 ? 8 : KT / 8) != 0) return launch_chunk16_as<HDP, KT, false, CS, false, RULE>(a, stream);
  return a.kpool.geometry.head_dim == HDP ? launch_chunk16_as<HDP, KT, true, CS, true, RULE>(a, stream)
                                          : launch_chunk16_as<HDP, KT, true, CS, false, RULE>(a, stream);
}

template <int HDP, int NB, int KW, bool UNI, bool WHOLE, int RULE>
static int launch_few_as(const ChunkArgs& a, hipStream_t stream) {
  constexpr int tiles = kFewWaves * kFewTile * HDP * 2 + (NB * HDP >= 256 ? 16 * NB * HDP * 2 : 0), joined = few_joined_bytes(HDP, NB), bytes = tiles > joined ? tiles : joined;
  static LdsLimit limit;
  if (int rc = limit.raise(reinterpret_cast<const void*>(&attend_few_kernel<HDP, NB, KW, UNI, WHOLE, RULE>), bytes, "attend_few_kernel LDS")) return rc;
  hipLaunchKernelGGL((attend_few_kernel<HDP, NB, KW, UNI, WHOLE, RULE>), dim3(a.n_items), dim3(64 * kFewWaves), bytes, stream, a);
  return check_hip(hipGetLastError(), "attend_few_kernel launch");
}

// Whether a pool holds 4-bit codes in groups of 32, and no others.
static bool codes4(const dc_pool& p) {
  uint64_t four = 0, others = 0;
  for (int f : {DC_FMT_M0_AFFINE, DC_FMT_M0_SYMMETRIC}) four |= uint64_t(1) << (f * 9 + 4), others |= uint64_t(1) << (f * 9 + 8);
  return p.geometry.group_size == 32 && (p.format_mask & four) != 0 && (p.format_mask & others) == 0;
}

template <int HDP, int NB, int KW, int RULE>
static int launch_few(const ChunkArgs& a, hipStream_t stream) {
  if (a.kpool.geometry.page_capacity % kFewTile == 0 && a.kpool.geometry.head_dim == HDP && codes4(a.kpool) && codes4(a.vpool))
    return launch_few_as<HDP, NB, 1, true, true, RULE>(a, stream);
  if (a.kpool.geometry.page_capacity % kFewTile != 0) return launch_few_as<HDP, NB, KW, false, false, RULE>(a, stream);
  return a.kpool.geometry.head_dim == HDP ? launch_few_as<HDP, NB, KW, true, true, RULE>(a, stream)
                                          : launch_few_as<HDP, NB, KW, true, false, RULE>(a, stream);
}

template <int RULE>
static int launch_all(ChunkArgs a, int32_t n_few, int32_t few_rows, bool units, hipStream_t st) {
  const int hd = a.kpool.geometry.head_dim;
  if (units && n_few) {
    ChunkArgs f = a;
    f.n_items = n_few;
    const bool one = few_rows <= 16;
    const int rc = hd <= 64    ? (one ? launch_few<64, 1, 4, RULE>(f, st) : launch_few<64, 4, 4, RULE>(f, st))
                   : hd <= 128 ? (one ? launch_few<128, 1, 4, RULE>(f, st) : few_rows <= 32 ? launch_few<128, 2, 4, RULE>(f, st) : launch_few<128, 3, 2, RULE>(f, st))
                               : launch_few<256, 1, 2, RULE>(f, st);
    if (rc != DC_OK) return rc;
    a.items += n_few;
    if (RULE && a.gaps) a.gaps += n_few;
    a.n_items -= n_few;
  }
  if (a.n_items == 0) return DC_OK;
  if (units)
    return hd <= 64 ? launch_chunk16<64, 128, 1, RULE>(a, st) : hd <= 128 ? launch_chunk16<128, 64, 1, RULE>(a, st) : launch_chunk16<256, 32, 2, RULE>(a, st);
  if (a.dtype == DC_F32)
    return hd <= 64 ? launch_chunk<float, 64, 64, RULE>(a, st) : hd <= 128 ? launch_chunk<float, 128, 32, RULE>(a, st) : launch_chunk<float, 256, 32, RULE>(a, st);
  return hd <= 64 ? launch_chunk<_Float16, 64, 128, RULE>(a, st) : hd <= 128 ? launch_chunk<_Float16, 128, 64, RULE>(a, st) : launch_chunk<_Float16, 256, 32, RULE>(a, st);
}

}  // namespace dc
