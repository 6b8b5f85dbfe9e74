// Tokens of cache pages as dense rows (dc_read_tokens): the inverse of the
// page encode, x = s * code + b of every channel, rounded once to the rows'
// dtype.  Bound by memory: a row's compressed bytes in, its dense bytes out.
//
// A lane reads one 16-channel chunk of a row (dc_unpack.h) and stores 32 or 64
// bytes.  A block takes kReadTokens consecutive tokens of one head, so that a
// group's words, which a page keeps token by token, are read as whole lines.
// Geometries without such chunks take one thread per channel.
#include "dc_unpack.h"

namespace dc {

constexpr int kReadThreads = 256;

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

// The page of token t, head h and its slot; false where the table names none.
__device__ __forceinline__ bool token_page(const ReadArgs& R, const ReadJob& J, int64_t t, int32_t h, dc_page_desc* d,
                                           int32_t* slot) {
  const int32_t row = R.row[t], tok = R.token[t];
  if (uint32_t(row) >= uint32_t(R.dest_rows) || tok < 0) return false;
  const uint32_t p = uint32_t(tok) / uint32_t(R.page_tokens);
  if (p >= uint32_t(R.dest_pages)) return false;
  *slot = tok - int32_t(p * R.page_tokens);
  const int32_t id = J.pages[(int64_t(row) * J.out.n_heads + h) * R.dest_pages + p];
  if (id < 0 || id >= J.pool.n_descs || *slot >= J.pool.geometry.page_capacity) return false;
  *d = J.pool.descs[id];
  return true;
}

__device__ __forceinline__ uint32_t pack2(int32_t dtype, float a, float b) {
  return dtype == DC_F16 ? __builtin_bit_cast(uint32_t, read_h2{(_Float16)a, (_Float16)b})
                         : __builtin_bit_cast(uint32_t, read_bf2{(__bf16)a, (__bf16)b});
}

// blockIdx.y: keys or values.  Block x takes tokens [tile * tokens, ...) of one
// head, tokens = kReadThreads / (head_dim / 16).
__global__ void __launch_bounds__(kReadThreads) read_chunks_kernel(ReadArgs R, ReadJob j0, ReadJob j1) {
  const ReadJob J = blockIdx.y == 0 ? j0 : j1;
  const dc_page_geometry geo = J.pool.geometry;
  const uint32_t cpr = geo.head_dim / 16, tokens = kReadThreads / cpr;
  const uint32_t tile = blockIdx.x / uint32_t(J.out.n_heads), h = blockIdx.x - tile * J.out.n_heads;
  const uint32_t i = threadIdx.x / cpr, chunk = threadIdx.x - i * cpr;
  const int64_t t = int64_t(tile) * tokens + i;
  if (i >= tokens || t >= R.n_tokens) return;
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = 0.f;
  dc_page_desc d;
  int32_t slot;
  if (token_page(R, J, t, h, &d, &slot)) {
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
  if (J.out.dtype == DC_F32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(J.out.data) + off);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = float4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
  } else {
    uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(J.out.data) + off);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      o[k] = uint4{pack2(J.out.dtype, v[8 * k], v[8 * k + 1]), pack2(J.out.dtype, v[8 * k + 2], v[8 * k + 3]),
                   pack2(J.out.dtype, v[8 * k + 4], v[8 * k + 5]), pack2(J.out.dtype, v[8 * k + 6], v[8 * k + 7])};
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
  dc_page_desc d;
  int32_t slot;
  if (token_page(R, J, t, h, &d, &slot)) {
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
  const dim3 grid(uint32_t(blocks), 2);
  if (chunks)
    hipLaunchKernelGGL(dc::read_chunks_kernel, grid, dim3(dc::kReadThreads), 0, hipStream_t(stream), R, a, b);
  else
    hipLaunchKernelGGL(dc::read_values_kernel, grid, dim3(dc::kReadThreads), 0, hipStream_t(stream), R, a, b);
  return dc::check_hip(hipGetLastError(), "dc_read_tokens launch");
}
