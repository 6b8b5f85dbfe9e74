// Tokens of cache pages as dense rows (dc_read_tokens): the inverse of the
// page encode, x = s * code + b of every channel, rounded once to the rows'
// dtype.  Bound by memory: a row's compressed bytes in, its dense bytes out.
//
// A lane reads one 16-channel chunk of a row (dc_unpack.h), 32 or 64 bytes of
// it as 16- or 32-bit values.  A block takes consecutive tokens of one head, so
// that a group's words, which a page keeps token by token, are read as whole
// lines.  Four lanes of a row turn their 16-byte units about, so that each
// store of theirs covers 64 bytes in a row, and stores of more than the L2
// holds bypass it (kStreamBytes): 8 x 16384 tokens of 4 heads of 128 channels
// from 4-bit pages as bf16 (352 MB in all) take 65 to 74 us (5 TB/s) where the last
// cache still holds the pages, 97 (3.6) where it does not.  The former: 119 us with
// the units turned alone, 130 us with the bypass alone, 118 us with neither
// (a bypassing store of half a line is written as it is).  Four tokens a lane
// with their loads in flight together were 76 us.  Geometries without such
// chunks take one thread per channel.
#include "dc_unpack.h"

namespace dc {

constexpr int kReadThreads = 256;
constexpr int64_t kStreamBytes = int64_t(32) << 20;  // the L2 of all dies

struct ReadJob {
  const int32_t* pages;
  dc_pool pool;
  dc_token_rows out;
};

struct ReadArgs {
  int64_t n_tokens;
  const int32_t* row;
  const int32_t* token;
  int32_t dest_rows, dest_pages, page_tokens;
};

typedef __bf16 read_bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 read_h2 __attribute__((ext_vector_type(2)));

// The page of a token (row, tok) of head h and its slot; id -1 where the
// table names none.
__device__ __forceinline__ int32_t token_page(const ReadArgs& R, const ReadJob& J, int32_t row, int32_t tok, int32_t h,
                                              int32_t* slot) {
  const uint32_t p = uint32_t(tok) / uint32_t(R.page_tokens);
  *slot = tok - int32_t(p * R.page_tokens);
  if (uint32_t(row) >= uint32_t(R.dest_rows) || tok < 0 || p >= uint32_t(R.dest_pages)) return -1;
  const int32_t id = J.pages[(int64_t(row) * J.out.n_heads + h) * R.dest_pages + p];
  return id < J.pool.n_descs && *slot < J.pool.geometry.page_capacity ? id : -1;
}

__device__ __forceinline__ uint32_t pack2(int32_t dtype, float a, float b) {
  return dtype == DC_F16 ? __builtin_bit_cast(uint32_t, read_h2{(_Float16)a, (_Float16)b})
                         : __builtin_bit_cast(uint32_t, read_bf2{(__bf16)a, (__bf16)b});
}

typedef uint32_t read_u4 __attribute__((ext_vector_type(4)));

template <bool stream>
__device__ __forceinline__ void store16(void* p, const uint32_t (&w)[4]) {
  const read_u4 x{w[0], w[1], w[2], w[3]};
  if constexpr (stream)
    __builtin_nontemporal_store(x, reinterpret_cast<read_u4*>(p));
  else
    *reinterpret_cast<read_u4*>(p) = x;
}

// A lane's N 16-byte units (w) of a row to the row at o.  quads: the row's lanes
// come in aligned fours; store j of lane l is then unit 4 j + l of the four.
template <int N, bool stream>
__device__ __forceinline__ void store_units(uint8_t* o, const uint32_t (&w)[N][4], bool quads) {
  if (!quads) {
#pragma unroll
    for (int j = 0; j < N; ++j) store16<false>(o + 16 * j, w[j]);
    return;
  }
  const int l = threadIdx.x & 3;
  uint8_t* first = o - 16 * N * l;
  auto store = [&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 2) {  // unit 4 j + l: unit l % 2 of lane 2 j + l / 2
        constexpr int from = j ? 0xfa : 0x50;
        const uint32_t a = __builtin_amdgcn_mov_dpp(int(w[0][i]), from, 0xf, 0xf, true);
        const uint32_t b = __builtin_amdgcn_mov_dpp(int(w[1][i]), from, 0xf, 0xf, true);
        x[i] = l & 1 ? b : a;
      } else {  // unit 4 j + l: unit l of lane j
        constexpr int from = 0x55 * j;
        const uint32_t a = __builtin_amdgcn_mov_dpp(int(w[0][i]), from, 0xf, 0xf, true);
        const uint32_t b = __builtin_amdgcn_mov_dpp(int(w[1][i]), from, 0xf, 0xf, true);
        const uint32_t c = __builtin_amdgcn_mov_dpp(int(w[2][i]), from, 0xf, 0xf, true);
        const uint32_t d = __builtin_amdgcn_mov_dpp(int(w[3][i]), from, 0xf, 0xf, true);
        x[i] = l & 2 ? (l & 1 ? d : c) : (l & 1 ? b : a);
      }
    }
    store16<stream>(first + 64 * j + 16 * l, x);
  };
  store(std::integral_constant<int, 0>{});
  store(std::integral_constant<int, 1>{});
  if constexpr (N == 4) {
    store(std::integral_constant<int, 2>{});
    store(std::integral_constant<int, 3>{});
  }
}

// blockIdx.y: keys or values.  Block x takes tokens [tile * tokens, ...) of one
// head, tokens = kReadThreads / (head_dim / 16).
template <bool stream>
__global__ void __launch_bounds__(kReadThreads) read_chunks_kernel(ReadArgs R, ReadJob j0, ReadJob j1) {
  const ReadJob J = blockIdx.y == 0 ? j0 : j1;
  const dc_page_geometry geo = J.pool.geometry;
  const uint32_t cpr = geo.head_dim / 16, tokens = kReadThreads / cpr;
  const uint32_t tile = blockIdx.x / uint32_t(J.out.n_heads), h = blockIdx.x - tile * J.out.n_heads;
  const uint32_t i = threadIdx.x / cpr, chunk = threadIdx.x - i * cpr;
  const int64_t t = int64_t(tile) * tokens + i;
  if (i >= tokens || t >= R.n_tokens) return;  // (a row's lanes together)
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = 0.f;
  int32_t slot;
  const int32_t id = token_page(R, J, R.row[t], R.token[t], h, &slot);
  if (id >= 0) {
    const dc_page_desc d = J.pool.descs[id];
    const Blob32 L = blob32(d.format, d.bits, geo, num_groups(geo));
    if ((int64_t(d.block) << 8) + L.total <= J.pool.arena_bytes) {
      const uint8_t* blob = blob_ptr(J.pool.arena, d);
      const Chunk16 ck = chunk16_at(d.format, d.bits, geo, L, 16 * chunk);
      for_chunk_kind(chunk_kind(d.format, d.bits), [&](auto kind) __attribute__((always_inline)) {
        constexpr int K = decltype(kind)::value;
        uint32_t r[16];
        load_chunk16(K, blob + slot * ck.word_step + ck.word(), r);
        float s = 1.f, b = 0.f;
        if constexpr (K != CK_F16 && K != CK_F32) {
          constexpr float zp = K == CK_B2 ? -1.f : K == CK_B3 ? -3.f : K == CK_B4 ? -7.f : K == CK_B8 ? -127.f : 0.f;
          s = half_bits(*reinterpret_cast<const uint16_t*>(blob + slot * ck.scale_step + ck.scale), 0);
          b = d.format == DC_FMT_M0_AFFINE ? half_bits(*reinterpret_cast<const uint16_t*>(blob + slot * ck.scale_step + ck.bias), 0)
              : K == CK_I8                 ? 0.f
                                           : zp * s;
        }
        values16<K>(r, ck.shift(), s, b, v);
      });
    }
  }
  const int64_t off = t * J.out.token_stride + h * J.out.head_stride + 16 * chunk;
  const bool quads = cpr % 4 == 0;
  if (J.out.dtype == DC_F32) {
    uint32_t w[4][4];
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k / 4][k % 4] = __float_as_uint(v[k]);
    store_units<4, stream>(reinterpret_cast<uint8_t*>(J.out.data) + 4 * off, w, quads);
  } else {
    uint32_t w[2][4];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k / 4][k % 4] = pack2(J.out.dtype, v[2 * k], v[2 * k + 1]);
    store_units<2, stream>(reinterpret_cast<uint8_t*>(J.out.data) + 2 * off, w, quads);
  }
}

__global__ void __launch_bounds__(kReadThreads) read_values_kernel(ReadArgs R, ReadJob j0, ReadJob j1) {
  const ReadJob J = blockIdx.y == 0 ? j0 : j1;
  const dc_page_geometry geo = J.pool.geometry;
  const int64_t i = int64_t(blockIdx.x) * kReadThreads + threadIdx.x;
  const int64_t r = i / geo.head_dim;
  const int32_t c = int32_t(i - r * geo.head_dim);
  const int64_t t = r / J.out.n_heads;
  const int32_t h = int32_t(r - t * J.out.n_heads);
  if (t >= R.n_tokens) return;
  float v = 0.f;
  int32_t slot;
  const int32_t id = token_page(R, J, R.row[t], R.token[t], h, &slot);
  if (id >= 0) {
    const dc_page_desc d = J.pool.descs[id];
    const BlobLayout L = blob_layout(d.format, d.bits, geo);
    if ((int64_t(d.block) << 8) + L.total <= J.pool.arena_bytes) v = page_value(blob_ptr(J.pool.arena, d), d, L, geo, slot, c);
  }
  const int64_t off = t * J.out.token_stride + h * J.out.head_stride + c;
  if (J.out.dtype == DC_F32)
    reinterpret_cast<float*>(J.out.data)[off] = v;
  else if (J.out.dtype == DC_F16)
    reinterpret_cast<_Float16*>(J.out.data)[off] = _Float16(v);
  else
    reinterpret_cast<__bf16*>(J.out.data)[off] = __bf16(v);
}

}  // namespace dc

extern "C" int dc_read_tokens(int64_t n_tokens, dc_token_dest src, dc_pool k_pool, dc_pool v_pool, dc_token_rows k_out,
                              dc_token_rows v_out, dc_stream_t stream) {
  const char* who = "dc_read_tokens";
  if (n_tokens < 0) return dc::fail(DC_EINVAL, "%s: n_tokens must be non-negative", who);
  const dc_pool* pools[2] = {&k_pool, &v_pool};
  const dc_token_rows* outs[2] = {&k_out, &v_out};
  bool chunks = true;
  for (int i = 0; i < 2; ++i) {
    const dc_pool& p = *pools[i];
    const dc_token_rows& o = *outs[i];
    if (int rc = dc::validate_geometry(p.geometry)) return rc;
    if (!p.arena || !p.descs || p.n_descs < 0) return dc::fail(DC_EINVAL, "%s: null pool", who);
    if (!o.data || o.n_heads <= 0 || (o.dtype != DC_F32 && o.dtype != DC_F16 && o.dtype != DC_BF16))
      return dc::fail(DC_EINVAL, "%s: bad output rows", who);
    if (src.page_tokens > p.geometry.page_capacity) return dc::fail(DC_EINVAL, "%s: page_tokens exceeds a pool's page capacity", who);
    const int64_t es = o.dtype == DC_F32 ? 4 : 2;
    chunks = chunks && dc::chunk16_geometry(p.geometry) && p.geometry.head_dim / 16 <= dc::kReadThreads &&
             reinterpret_cast<uintptr_t>(o.data) % 16 == 0 && o.token_stride * es % 16 == 0 && o.head_stride * es % 16 == 0;
  }
  if (k_pool.geometry.head_dim != v_pool.geometry.head_dim || k_out.n_heads != v_out.n_heads)
    return dc::fail(DC_EINVAL, "%s: keys and values must share head_dim and heads", who);
  if (!src.k_pages || !src.v_pages || !src.row || !src.token || src.n_rows <= 0 || src.n_pages <= 0 || src.page_tokens <= 0)
    return dc::fail(DC_EINVAL, "%s: bad token table", who);
  if (n_tokens == 0) return DC_OK;
  const dc::ReadArgs R{n_tokens, src.row, src.token, src.n_rows, src.n_pages, src.page_tokens};
  const dc::ReadJob a{src.k_pages, k_pool, k_out}, b{src.v_pages, v_pool, v_out};
  const int64_t hd = k_pool.geometry.head_dim;
  const int64_t tokens = chunks ? dc::kReadThreads / (hd / 16) : 1;
  const int64_t blocks = chunks ? (n_tokens + tokens - 1) / tokens * k_out.n_heads
                                : (n_tokens * k_out.n_heads * hd + dc::kReadThreads - 1) / dc::kReadThreads;
  if (blocks > 0x7fffffff) return dc::fail(DC_EINVAL, "%s: too many rows", who);
  const dim3 grid(uint32_t(blocks), 2), block(dc::kReadThreads);
  const int64_t bytes = 2 * n_tokens * k_out.n_heads * hd * (k_out.dtype == DC_F32 ? 4 : 2);
  if (!chunks)
    hipLaunchKernelGGL(dc::read_values_kernel, grid, block, 0, hipStream_t(stream), R, a, b);
  else if (bytes > dc::kStreamBytes)
    hipLaunchKernelGGL(dc::read_chunks_kernel<true>, grid, block, 0, hipStream_t(stream), R, a, b);
  else
    hipLaunchKernelGGL(dc::read_chunks_kernel<false>, grid, block, 0, hipStream_t(stream), R, a, b);
  return dc::check_hip(hipGetLastError(), "dc_read_tokens launch");
}
