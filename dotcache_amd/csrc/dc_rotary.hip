// Per-head norms and the position rotation of queries and keys, on their way
// to rows (dc_norm_rotate) or into cache pages (dc_append_rotary).
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head, over head_dim; w optional)
//   z_a = y_a cos - y_b sin,  z_b = y_b cos + y_a sin
//
// for channel pairs (a, b) = (i, i + rd / 2), or (2 i, 2 i + 1) interleaved,
// i < rd / 2; channels past the rotary_dim rd are only normed.  cos and sin of
// a position are one row of an fp32 table.
//
// Rows that go out as rows are computed in fp32 and rounded once.  Keys that
// go into pages are computed in fp64 and rounded to fp32 once: a code is
// decided at a border between two levels, and so does not depend on the order
// a sum was taken in (a page holds what encoding the fp64 formula's rows
// gives).
//
// Two kernels, as in dc_encode.hip: rotary_rows8_kernel (8 channels per lane,
// several rows per wavefront; head_dim a multiple of 8, pairs that start at
// multiples of 8 channels, a row within a wavefront) and
// rotary_rows_kernel (one wavefront per row through LDS) for the rest.
#include <math.h>

#include "dc_encode_row.h"

namespace dc {

constexpr int kRotThreads = 256;

// Rows of one launch: queries out, keys out or into pages, values into pages.
struct RotaryJob {
  dc_token_rows in;
  dc_norm norm;
  dc_token_rows out;     // data null: into pages
  const int32_t* pages;  // [dest_rows][heads][dest_pages] page ids
  dc_pool pool;
  float* keep;
  int32_t rotate;
  // rows out: heads a lane takes; whether the stores bypass the L2
  int32_t heads, stream;
};

struct RotaryArgs {
  int64_t n_tokens;
  int32_t head_dim;
  const int32_t* positions;
  dc_rotary rotary;
  const int32_t* row;  // destinations (dc_token_dest)
  const int32_t* token;
  int32_t dest_rows, dest_pages, page_tokens;
  const int32_t* keep_row;
  int32_t keep_head_stride, keep_rows;
};

typedef uint32_t rot_u4 __attribute__((ext_vector_type(4)));
typedef __bf16 rot_bf2 __attribute__((ext_vector_type(2)));

// Eight values to row elements off .. off + 7, rounded to nearest even, past
// the L2 if stream.
template <bool vec, bool stream>
__device__ __forceinline__ void store8(void* p, int32_t dtype, int64_t off, const float (&z)[8]) {
  if (dtype == DC_F32) {
    float* o = reinterpret_cast<float*>(p) + off;
    if constexpr (vec) {
      *reinterpret_cast<float4*>(o) = float4{z[0], z[1], z[2], z[3]};
      *reinterpret_cast<float4*>(o + 4) = float4{z[4], z[5], z[6], z[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = z[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = dtype == DC_F16 ? __builtin_bit_cast(uint32_t, enc_h2{(_Float16)z[2 * i], (_Float16)z[2 * i + 1]})
                           : __builtin_bit_cast(uint32_t, rot_bf2{(__bf16)z[2 * i], (__bf16)z[2 * i + 1]});
  uint16_t* o = reinterpret_cast<uint16_t*>(p) + off;
  if constexpr (vec) {
    const rot_u4 x{w[0], w[1], w[2], w[3]};
    if constexpr (stream)
      __builtin_nontemporal_store(x, reinterpret_cast<rot_u4*>(o));
    else
      *reinterpret_cast<rot_u4*>(o) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
  }
}

template <bool vec>
__device__ __forceinline__ void load_weight8(const dc_norm& n, int32_t h, int32_t c, float (&w)[8]) {
  const int64_t off = int64_t(h) * n.head_stride + c;
  if (n.dtype == DC_F32)
    load8<DC_F32, vec>(n.weight, off, w);
  else if (n.dtype == DC_F16)
    load8<DC_F16, vec>(n.weight, off, w);
  else
    load8<DC_BF16, vec>(n.weight, off, w);
}

// Sum over a row's lpr lanes, in all of them.
template <typename A>
__device__ __forceinline__ A row_sum(A v, int lpr, int lane, int q) {
  if ((lpr & (lpr - 1)) == 0) {
    for (int o = 1; o < lpr; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
  }
  A s = 0;
  for (int p = 0; p < lpr; ++p) s += __shfl(v, lane - q + p, 64);
  return s;
}

// Rows out: a lane takes two chunks of 8 channels, which in a half-split
// rotation are the two sides of 8 pairs, of `heads` consecutive heads of one
// token, so that the token's cosines and sines (and weights that heads share)
// are loaded once for all of them; kHeadsAhead heads' loads are in flight together.
constexpr int kHeadsAhead = 2;

__host__ __device__ inline int32_t row_lanes(int32_t hd, int32_t split_rd) { return split_rd / 16 + (hd - split_rd + 15) / 16; }

template <int32_t dtype, bool vec, bool vec_out, bool stream>
__device__ __forceinline__ void rows_out(const RotaryArgs& R, const RotaryJob& J, uint32_t b, int wave, int lane) {
  const int32_t hd = R.head_dim, rd = J.rotate ? R.rotary.rotary_dim : 0;
  const bool half = R.rotary.interleaved == 0;
  const int32_t split = half ? rd : 0;
  const int lpr = row_lanes(hd, split), rpw = 64 / lpr, q = lane % lpr, rw = lane / lpr;
  const uint32_t parts = (uint32_t(J.in.n_heads) + J.heads - 1) / J.heads, tile = b / parts;
  const int32_t h0 = int32_t(b - tile * parts) * J.heads, h1 = min(h0 + J.heads, J.in.n_heads);
  const int64_t t = (int64_t(tile) * (kRotThreads / 64) + wave) * rpw + rw;
  const bool in_rows = rw < rpw && t < R.n_tokens;
  const int64_t tt = in_rows ? t : 0;
  const bool paired = q < split / 16;
  const int32_t c0 = paired ? 8 * q : split + 16 * (q - split / 16);
  const int32_t c1 = paired ? c0 + rd / 2 : c0 + 8;
  const bool two = c1 < hd;  // (a lane at the end of an odd number of chunks has one)
  const int32_t cb = two ? c1 : c0;
  const bool turn0 = c0 < rd, turn1 = two && (half ? turn0 : c1 < rd);
  const int32_t pos = rd ? R.positions[tt] : 0;
  const bool known = uint32_t(pos) < uint32_t(rd ? R.rotary.n_positions : 1);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (rd) {  // (uniform; interleaved: four pairs of each chunk)
    const float* row = R.rotary.table + int64_t(known ? pos : 0) * rd;
    const int32_t p0 = half ? (turn0 ? c0 : 0) : (turn0 ? c0 / 2 : 0), p1 = half ? p0 + 4 : (turn1 ? c1 / 2 : 0);
    const float4 a = *reinterpret_cast<const float4*>(row + p0), e = *reinterpret_cast<const float4*>(row + p1);
    const float4 f = *reinterpret_cast<const float4*>(row + rd / 2 + p0), g = *reinterpret_cast<const float4*>(row + rd / 2 + p1);
    if (turn0) {
      cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w;
      sn[0] = f.x; sn[1] = f.y; sn[2] = f.z; sn[3] = f.w;
    }
    if (turn1) {
      cs[4] = e.x; cs[5] = e.y; cs[6] = e.z; cs[7] = e.w;
      sn[4] = g.x; sn[5] = g.y; sn[6] = g.z; sn[7] = g.w;
    }
  }
  const bool norm = J.norm.weight != nullptr;
  float w0[8], w1[8];
  if (norm) {
    load_weight8<vec>(J.norm, h0, c0, w0);
    load_weight8<vec>(J.norm, h0, cb, w1);
  }
  const float inv = 1.f / float(hd);
  for (int32_t h = h0; h < h1; h += kHeadsAhead) {
    float x[kHeadsAhead][8], y[kHeadsAhead][8];
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k) {
      const int64_t base = tt * J.in.token_stride + int64_t(min(h + k, h1 - 1)) * J.in.head_stride;
      load8<dtype, vec>(J.in.data, base + c0, x[k]);
      load8<dtype, vec>(J.in.data, base + cb, y[k]);
    }
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k) {
      if (h + k >= h1) break;  // (uniform)
      if (norm) {
        if (J.norm.head_stride != 0 && h + k > h0) {
          load_weight8<vec>(J.norm, h + k, c0, w0);
          load_weight8<vec>(J.norm, h + k, cb, w1);
        }
        float ss = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = __builtin_fmaf(x[k][i], x[k][i], ss);
          s1 = __builtin_fmaf(y[k][i], y[k][i], s1);
        }
        ss = row_sum<float>(two ? ss + s1 : ss, lpr, lane, q);
        const float r = 1.f / sqrtf(__builtin_fmaf(ss, inv, J.norm.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[k][i] *= r * w0[i];
          y[k][i] *= r * w1[i];
        }
      }
      if (half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x[k][i], v = y[k][i];
          x[k][i] = paired ? __builtin_fmaf(u, cs[i], -v * sn[i]) : u;
          y[k][i] = paired ? __builtin_fmaf(v, cs[i], u * sn[i]) : v;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[k][2 * i], v = x[k][2 * i + 1], u1 = y[k][2 * i], v1 = y[k][2 * i + 1];
          x[k][2 * i] = turn0 ? __builtin_fmaf(u, cs[i], -v * sn[i]) : u;
          x[k][2 * i + 1] = turn0 ? __builtin_fmaf(v, cs[i], u * sn[i]) : v;
          y[k][2 * i] = turn1 ? __builtin_fmaf(u1, cs[i + 4], -v1 * sn[i + 4]) : u1;
          y[k][2 * i + 1] = turn1 ? __builtin_fmaf(v1, cs[i + 4], u1 * sn[i + 4]) : v1;
        }
      }
      if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = y[k][i] = __builtin_nanf("");
      }
      if (in_rows) {
        const int64_t o = t * J.out.token_stride + int64_t(h + k) * J.out.head_stride;
        store8<vec_out, stream>(J.out.data, J.out.dtype, o + c0, x[k]);
        if (two) store8<vec_out, stream>(J.out.data, J.out.dtype, o + c1, y[k]);
      }
    }
  }
}

// Rows into pages: channels c0 .. c0 + 7 of row (t, h) of J, normed and
// rotated in fp64.  Lane q of the row's lpr lanes; every lane of the wavefront
// takes part.  In a half-split rotation the pair's other eight channels are a
// second load (a hit in the cache: cheaper than eight cross-lane moves).
template <int32_t dtype, bool vec>
__device__ __forceinline__ void rotated8(const RotaryArgs& R, const RotaryJob& J, int64_t t, int32_t h, int lpr, int lane,
                                         int q, int32_t c0, float (&z)[8]) {
  const int64_t base = t * J.in.token_stride + h * J.in.head_stride;
  const int32_t hd = R.head_dim;
  const bool has = c0 < hd;  // (lanes past head_dim, where a page pads its groups: zeros)
  const int32_t c = has ? c0 : 0;
  const int32_t rd = J.rotate ? R.rotary.rotary_dim : 0;
  float x[8];
  load8<dtype, vec>(J.in.data, base + c, x);
  if (rd == 0 && J.norm.weight == nullptr) {  // (uniform)
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = has ? x[i] : 0.f;
    return;
  }
  const bool half = R.rotary.interleaved == 0, turns = c < rd;
  const bool second = half && c >= rd / 2;
  const int32_t pc = half && turns ? (second ? c - rd / 2 : c + rd / 2) : c;
  float xp[8];
  if (half && rd) load8<dtype, vec>(J.in.data, base + pc, xp);
  const int32_t pos = rd ? R.positions[t] : 0;
  const bool known = uint32_t(pos) < uint32_t(rd ? R.rotary.n_positions : 1);
  float cs[8], sn[8];
  if (rd) {
    const float* row = R.rotary.table + int64_t(known ? pos : 0) * rd;
    if (half) {
      const float* p = row + (turns ? (second ? pc : c) : 0);
      load8<DC_F32, true>(p, 0, cs);
      load8<DC_F32, true>(p, rd / 2, sn);
    } else {
      const float* p = row + (turns ? c / 2 : 0);
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + rd / 2);
      cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w;
      sn[0] = b.x; sn[1] = b.y; sn[2] = b.z; sn[3] = b.w;
    }
  }
  double y[8], yp[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = x[i];
    yp[i] = half && rd ? double(xp[i]) : 0.0;
  }
  if (J.norm.weight != nullptr) {  // (uniform)
    double ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(y[i], y[i], ss);
    ss = row_sum<double>(has ? ss : 0.0, lpr, lane, q);
    const double r = 1.0 / sqrt(ss / hd + double(J.norm.eps));
    float w[8];
    load_weight8<vec>(J.norm, h, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * (r * double(w[i]));
    if (half && rd) {
      load_weight8<vec>(J.norm, h, pc, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) yp[i] = yp[i] * (r * double(w[i]));
    }
  }
  if (rd) {
    if (half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = fma(y[i], double(cs[i]), (second ? yp[i] : -yp[i]) * double(sn[i]));
        y[i] = turns ? v : y[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double a = y[2 * i], b = y[2 * i + 1], co = cs[i], si = sn[i];
        y[2 * i] = turns ? fma(a, co, -b * si) : a;
        y[2 * i + 1] = turns ? fma(b, co, a * si) : b;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = !has ? 0.f : known ? float(y[i]) : __builtin_nanf("");
}

// Whether token t has a row of cosines and sines (or needs none).
__device__ __forceinline__ bool has_position(const RotaryArgs& R, int64_t t) {
  return R.rotary.rotary_dim == 0 || uint32_t(R.positions[t]) < uint32_t(R.rotary.n_positions);
}

// Page id and slot of token t, head h; -1 where it is not written.
__device__ __forceinline__ void token_dest(const RotaryArgs& R, const RotaryJob& J, int64_t t, int32_t h, int32_t* page,
                                           int32_t* slot) {
  const int32_t row = R.row[t], tok = R.token[t];
  const uint32_t p = uint32_t(tok) / uint32_t(R.page_tokens);
  const bool ok = uint32_t(row) < uint32_t(R.dest_rows) && tok >= 0 && p < uint32_t(R.dest_pages) && has_position(R, t);
  *slot = tok - int32_t(p * R.page_tokens);
  *page = -1;
  if (ok) *page = J.pages[(int64_t(row) * J.in.n_heads + h) * R.dest_pages + p];
  if (*page >= J.pool.n_descs) *page = -1;
}

__device__ __forceinline__ int32_t keep_at(const RotaryArgs& R, const RotaryJob& J, int64_t t, int32_t h) {
  if (J.keep == nullptr) return -1;
  const int32_t k = R.keep_row[t];
  const int64_t at = k + int64_t(h) * R.keep_head_stride;
  return k >= 0 && at < R.keep_rows && has_position(R, t) ? int32_t(at) : -1;
}

// Blocks [0, b1) take rows of j0, [b1, b2) rows of j1 and the rest rows of j2.
// A block that writes pages takes consecutive tokens of
// one head: their codes are neighbours in the page, and lines written whole.
template <int32_t dtype, bool vec, bool vec_out>
__global__ void __launch_bounds__(kRotThreads) rotary_rows8_kernel(RotaryArgs R, RotaryJob j0, RotaryJob j1, RotaryJob j2,
                                                                   uint32_t b1, uint32_t b2, int32_t lds_pack) {
  __shared__ uint32_t pack[kRotThreads / 64][kPackWords];
  const uint32_t block = blockIdx.x;
  const RotaryJob J = block < b1 ? j0 : block < b2 ? j1 : j2;
  const uint32_t b = block < b1 ? block : block < b2 ? block - b1 : block - b2;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (J.out.data != nullptr) {  // (uniform)
    if (vec_out && J.stream)
      rows_out<dtype, vec, vec_out, vec_out>(R, J, b, wave, lane);
    else
      rows_out<dtype, vec, vec_out, false>(R, J, b, wave, lane);
    return;
  }
  const dc_page_geometry geo = J.pool.geometry;
  const int32_t G = (geo.head_dim + geo.group_size - 1) / geo.group_size;
  const int lpr = G * geo.group_size / 8, lpg = geo.group_size / 8, rpw = 64 / lpr, q = lane % lpr, rw = lane / lpr;
  const int32_t c0 = 8 * q, g = c0 / geo.group_size, li = (c0 - g * geo.group_size) / 8;
  const int32_t tile = int32_t(b / uint32_t(J.in.n_heads)), h = int32_t(b - uint32_t(tile) * J.in.n_heads);
  const int64_t t = (int64_t(tile) * (kRotThreads / 64) + wave) * rpw + rw;
  const bool in_rows = rw < rpw && t < R.n_tokens;
  const int64_t tt = in_rows ? t : 0;
  int32_t page, slot;
  token_dest(R, J, tt, h, &page, &slot);
  const int32_t kr = keep_at(R, J, tt, h);
  float z[8];
  rotated8<dtype, vec>(R, J, tt, h, lpr, lane, q, c0, z);
  if (in_rows && kr >= 0 && c0 < geo.head_dim) {
    float4* o = reinterpret_cast<float4*>(J.keep + int64_t(kr) * geo.head_dim + c0);
    o[0] = float4{z[0], z[1], z[2], z[3]};
    o[1] = float4{z[4], z[5], z[6], z[7]};
  }
  const bool live = in_rows && page >= 0 && slot < geo.page_capacity;
  const dc_page_desc d = J.pool.descs[live ? page : 0];
  encode_row(J.pool, z, slot, d, live, pack, lds_pack, lane, wave, q, rw, c0, g, li, lpr, lpg);
}

// One wavefront per row, the row in LDS: any head_dim, group size and pairing.
__global__ void __launch_bounds__(64) rotary_rows_kernel(RotaryArgs R, RotaryJob j0, RotaryJob j1, RotaryJob j2,
                                                         uint32_t b1, uint32_t b2) {
  extern __shared__ float lds[];
  const int32_t hd = R.head_dim, lane = threadIdx.x;
  float *x = lds, *z = lds + hd;
  const uint32_t block = blockIdx.x;
  const RotaryJob J = block < b1 ? j0 : block < b2 ? j1 : j2;
  const uint32_t r = block < b1 ? block : block < b2 ? block - b1 : block - b2;
  const int64_t t = r / uint32_t(J.in.n_heads);
  const int32_t h = int32_t(r - uint32_t(t) * J.in.n_heads);
  const int64_t base = t * J.in.token_stride + h * J.in.head_stride;
  double ss = 0;
  for (int32_t c = lane; c < hd; c += 64) {
    x[c] = load_value(J.in.data, J.in.dtype, base + c);
    ss = fma(double(x[c]), double(x[c]), ss);
  }
  const bool norm = J.norm.weight != nullptr;
  double s = 1.0;
  if (norm) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    s = 1.0 / sqrt(ss / hd + double(J.norm.eps));
  }
  __syncthreads();
  const int32_t rd = J.rotate ? R.rotary.rotary_dim : 0, half = rd / 2;
  const int32_t pos = rd ? R.positions[t] : 0;
  const bool known = rd == 0 || uint32_t(pos) < uint32_t(R.rotary.n_positions);
  const float* row = R.rotary.table + int64_t(known ? pos : 0) * rd;
  auto normed = [&](int32_t c) -> double {
    return norm ? x[c] * (s * double(load_value(J.norm.weight, J.norm.dtype, int64_t(h) * J.norm.head_stride + c))) : double(x[c]);
  };
  for (int32_t c = lane; c < hd; c += 64) {
    double v = normed(c);
    if (c < rd) {
      const bool inter = R.rotary.interleaved != 0;
      const int32_t i = inter ? c / 2 : c % half;
      const bool second = inter ? (c & 1) != 0 : c >= half;
      const double p = normed(inter ? (c ^ 1) : (second ? c - half : c + half));
      const double co = row[i], si = row[half + i];
      v = fma(v, co, (second ? p : -p) * si);
    }
    z[c] = known ? float(v) : __builtin_nanf("");
  }
  __syncthreads();
  if (J.out.data != nullptr) {
    const int64_t o = t * J.out.token_stride + h * J.out.head_stride;
    for (int32_t c = lane; c < hd; c += 64) {
      if (J.out.dtype == DC_F32)
        reinterpret_cast<float*>(J.out.data)[o + c] = z[c];
      else if (J.out.dtype == DC_F16)
        reinterpret_cast<_Float16*>(J.out.data)[o + c] = _Float16(z[c]);
      else
        reinterpret_cast<__bf16*>(J.out.data)[o + c] = __bf16(z[c]);
    }
    return;
  }
  const int32_t kr = keep_at(R, J, t, h);
  if (kr >= 0)
    for (int32_t c = lane; c < hd; c += 64) J.keep[int64_t(kr) * hd + c] = z[c];
  int32_t page, slot;
  token_dest(R, J, t, h, &page, &slot);
  const dc_page_geometry geo = J.pool.geometry;
  if (page < 0 || slot >= geo.page_capacity) return;
  const dc_page_desc d = J.pool.descs[page];
  const BlobLayout L = blob_layout(d.format, d.bits, geo);
  if ((int64_t(d.block) << 8) + L.total > J.pool.arena_bytes) return;
  uint8_t* blob = reinterpret_cast<uint8_t*>(J.pool.arena) + (uint64_t(d.block) << 8);
  const int32_t G = L.groups;
  for (int32_t g = lane; g < G; g += 64) encode_group(geo, d, L, blob, slot, g, G, [&](int32_t c) { return z[c]; });
}

static bool known_dtype(int32_t d) { return d == DC_F32 || d == DC_F16 || d == DC_BF16; }
static int64_t esize(int32_t dtype) { return dtype == DC_F32 ? 4 : 2; }

// Whether every row of x starts on a 16-byte boundary.
static bool aligned_rows(const dc_token_rows& x) {
  return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.token_stride * esize(x.dtype) % 16 == 0 &&
         x.head_stride * esize(x.dtype) % 16 == 0;
}

static int check_rows(const dc_token_rows& x, int64_t n_tokens, const char* who, const char* name) {
  if (!x.data) return fail(DC_EINVAL, "%s: null %s", who, name);
  if (!known_dtype(x.dtype)) return fail(DC_EINVAL, "%s: %s dtype must be DC_F32, DC_F16 or DC_BF16", who, name);
  if (x.n_heads <= 0) return fail(DC_EINVAL, "%s: %s needs at least one head", who, name);
  if (n_tokens * x.n_heads > 0x7fffffff) return fail(DC_EINVAL, "%s: too many %s rows", who, name);
  return DC_OK;
}

static int check_norm(const dc_norm& n, const char* who) {
  if (!n.weight) return DC_OK;
  if (!known_dtype(n.dtype)) return fail(DC_EINVAL, "%s: norm weight dtype must be DC_F32, DC_F16 or DC_BF16", who);
  if (!(n.eps >= 0.f) || n.head_stride < 0) return fail(DC_EINVAL, "%s: bad norm eps or head stride", who);
  return DC_OK;
}

static int check_rotary(const RotaryArgs& R, const char* who) {
  const dc_rotary& r = R.rotary;
  if (R.head_dim <= 0 || R.head_dim > 8192) return fail(DC_EINVAL, "%s: head_dim must lie in [1, 8192]", who);
  if (r.rotary_dim < 0 || r.rotary_dim > R.head_dim || r.rotary_dim % 2)
    return fail(DC_EINVAL, "%s: rotary_dim must be even and at most head_dim", who);
  if (r.rotary_dim && (!r.table || !R.positions || r.n_positions <= 0)) return fail(DC_EINVAL, "%s: null rotary table or positions", who);
  if (reinterpret_cast<uintptr_t>(r.table) % 16 != 0) return fail(DC_EINVAL, "%s: the rotary table must be 16-byte aligned", who);
  return DC_OK;
}

// A lane takes several heads of a token as long as that leaves kRowBlocks
// blocks, and rows that the L2 would not hold bypass it.  16384 tokens of 28 + 4
// heads of 128 channels, bf16 (277 MB): 46 us (6.0 TB/s) on rows that the last
// cache still holds in part, 60 (4.6) on others.  The former with at most 8 heads
// a lane, four of them in flight, 53 us; without the bypass 59; with 2048 / 4096
// blocks asked for 61 / 67 (all with four in flight).
constexpr int64_t kRowBlocks = 1024;
constexpr int32_t kMaxHeads = 16;
constexpr int64_t kStreamBytes = int64_t(32) << 20;  // the L2 of all dies

static int launch_rotary(const RotaryArgs& R, RotaryJob* jobs, int n_jobs, hipStream_t stream) {
  // the 8-channel kernel where every row and pair fits it
  const int32_t hd = R.head_dim, rd = R.rotary.rotary_dim;
  bool fast = hd % 8 == 0 && hd <= 512 && rd % (R.rotary.interleaved ? 8 : 16) == 0;
  bool vec = true, vec_out = true, narrow = false;
  for (int i = 0; i < n_jobs; ++i) {
    const RotaryJob& j = jobs[i];
    vec = vec && aligned_rows(j.in);
    if (j.norm.weight)
      vec = vec && reinterpret_cast<uintptr_t>(j.norm.weight) % 16 == 0 && j.norm.head_stride * esize(j.norm.dtype) % 16 == 0;
    if (j.out.data) {
      vec_out = vec_out && aligned_rows(j.out);
    } else {
      fast = fast && fits_rows8(j.pool.geometry);
      narrow = narrow || has_narrow(j.pool);
    }
  }
  int64_t first[4] = {0, 0, 0, 0};
  for (int i = 0; i < 3; ++i) {
    int64_t blocks = 0;
    if (i < n_jobs) {
      RotaryJob& j = jobs[i];
      const int64_t rows = R.n_tokens * j.in.n_heads;
      if (!fast) {
        blocks = rows;
      } else if (j.out.data) {
        // as many heads a lane as leave kRowBlocks blocks
        const int64_t per = kRotThreads / 64 * (64 / row_lanes(hd, R.rotary.interleaved || !j.rotate ? 0 : rd));
        const int64_t tiles = (R.n_tokens + per - 1) / per;
        auto parts = [&](int32_t heads) { return int64_t((j.in.n_heads + heads - 1) / heads); };
        j.stream = rows * hd * esize(j.out.dtype) > kStreamBytes;
        j.heads = 1;
        while (j.heads < kMaxHeads && j.heads < j.in.n_heads && tiles * parts(2 * j.heads) >= kRowBlocks) j.heads *= 2;
        blocks = tiles * parts(j.heads);
      } else {
        const int64_t per = kRotThreads / 64 * (64 / (num_groups(j.pool.geometry) * j.pool.geometry.group_size / 8));
        blocks = (R.n_tokens + per - 1) / per * j.in.n_heads;
      }
    }
    first[i + 1] = first[i] + blocks;
  }
  if (first[3] > 0x7fffffff) return fail(DC_EINVAL, "too many rows");
  const RotaryJob &a = jobs[0], &b = jobs[n_jobs > 1 ? 1 : 0], &c = jobs[n_jobs > 2 ? 2 : 0];
  const dim3 grid{uint32_t(first[3])};
  const uint32_t b1 = uint32_t(first[1]), b2 = uint32_t(first[2]);
  if (!fast) {
    hipLaunchKernelGGL(rotary_rows_kernel, grid, dim3(64), 2 * size_t(hd) * sizeof(float), stream, R, a, b, c, b1, b2);
    return check_hip(hipGetLastError(), "rotary_rows_kernel launch");
  }
#define DC_ROT_X(DT_, V_, O_) \
  hipLaunchKernelGGL((rotary_rows8_kernel<DT_, V_, O_>), grid, dim3(kRotThreads), 0, stream, R, a, b, c, b1, b2, int32_t(narrow))
#define DC_ROT(DT_)                    \
  do {                                 \
    if (vec && vec_out)                \
      DC_ROT_X(DT_, true, true);       \
    else                               \
      DC_ROT_X(DT_, false, false);     \
  } while (0)
  if (a.in.dtype == DC_F32)
    DC_ROT(DC_F32);
  else if (a.in.dtype == DC_F16)
    DC_ROT(DC_F16);
  else
    DC_ROT(DC_BF16);
#undef DC_ROT
#undef DC_ROT_X
  return check_hip(hipGetLastError(), "rotary_rows8_kernel launch");
}

}  // namespace dc

extern "C" int dc_norm_rotate(int64_t n_tokens, int32_t head_dim, const int32_t* positions, dc_rotary rotary,
                              dc_token_rows q, dc_norm q_norm, dc_token_rows q_out, dc_token_rows k, dc_norm k_norm,
                              dc_token_rows k_out, dc_stream_t stream) {
  const char* who = "dc_norm_rotate";
  dc::RotaryArgs R{};
  R.n_tokens = n_tokens;
  R.head_dim = head_dim;
  R.positions = positions;
  R.rotary = rotary;
  if (n_tokens < 0) return dc::fail(DC_EINVAL, "%s: n_tokens must be non-negative", who);
  if (int rc = dc::check_rotary(R, who)) return rc;
  dc::RotaryJob jobs[3]{};
  int n = 0;
  for (int i = 0; i < 2; ++i) {
    const dc_token_rows &in = i ? k : q, &out = i ? k_out : q_out;
    if (in.n_heads == 0) continue;  // (keys or queries alone)
    const dc_norm& norm = i ? k_norm : q_norm;
    if (int rc = dc::check_rows(in, n_tokens, who, i ? "keys" : "queries")) return rc;
    if (int rc = dc::check_rows(out, n_tokens, who, i ? "keys out" : "queries out")) return rc;
    if (int rc = dc::check_norm(norm, who)) return rc;
    if (out.n_heads != in.n_heads) return dc::fail(DC_EINVAL, "%s: rows in and out must have the same heads", who);
    if (n && in.dtype != jobs[0].in.dtype) return dc::fail(DC_EINVAL, "%s: queries and keys must have one dtype", who);
    jobs[n].in = in;
    jobs[n].norm = norm;
    jobs[n].out = out;
    jobs[n].rotate = 1;
    ++n;
  }
  if (n == 0) return dc::fail(DC_EINVAL, "%s: neither queries nor keys", who);
  if (n_tokens == 0) return DC_OK;
  return dc::launch_rotary(R, jobs, n, hipStream_t(stream));
}

extern "C" int dc_append_rotary(int64_t n_tokens, const int32_t* positions, dc_rotary rotary, dc_token_rows q,
                                dc_norm q_norm, dc_token_rows q_out, dc_token_rows k, dc_norm k_norm, dc_token_rows v,
                                dc_token_dest dest, dc_pool k_pool, dc_pool v_pool, float* k_keep, float* v_keep,
                                const int32_t* keep_row, int32_t keep_head_stride, int32_t keep_rows, dc_stream_t stream) {
  const char* who = "dc_append_rotary";
  if (n_tokens < 0) return dc::fail(DC_EINVAL, "%s: n_tokens must be non-negative", who);
  for (const dc_pool* p : {&k_pool, &v_pool}) {
    if (int rc = dc::validate_geometry(p->geometry)) return rc;
    if (!p->arena || !p->descs) return dc::fail(DC_EINVAL, "%s: null pool", who);
    if (p->n_descs <= 0) return dc::fail(DC_EINVAL, "%s: a pool has no pages to write rows into", who);
  }
  if (v_pool.geometry.head_dim != k_pool.geometry.head_dim) return dc::fail(DC_EINVAL, "%s: key and value pools must share head_dim", who);
  if (!dest.k_pages || !dest.v_pages || !dest.row || !dest.token) return dc::fail(DC_EINVAL, "%s: null destinations", who);
  if (dest.n_rows <= 0 || dest.n_pages <= 0 || dest.page_tokens <= 0 || dest.page_tokens > k_pool.geometry.page_capacity ||
      dest.page_tokens > v_pool.geometry.page_capacity)
    return dc::fail(DC_EINVAL, "%s: bad destination table shape", who);
  dc::RotaryArgs R{};
  R.n_tokens = n_tokens;
  R.head_dim = k_pool.geometry.head_dim;
  R.positions = positions;
  R.rotary = rotary;
  R.row = dest.row;
  R.token = dest.token;
  R.dest_rows = dest.n_rows;
  R.dest_pages = dest.n_pages;
  R.page_tokens = dest.page_tokens;
  if (int rc = dc::check_rotary(R, who)) return rc;
  if ((k_keep == nullptr) != (v_keep == nullptr) || (k_keep && (!keep_row || keep_rows < 0 || keep_head_stride < 0)))
    return dc::fail(DC_EINVAL, "%s: kept rows need two buffers and a row per token", who);
  if (reinterpret_cast<uintptr_t>(k_keep) % 16 != 0 || reinterpret_cast<uintptr_t>(v_keep) % 16 != 0)
    return dc::fail(DC_EINVAL, "%s: kept rows must be 16-byte aligned", who);
  R.keep_row = keep_row;
  R.keep_head_stride = keep_head_stride;
  R.keep_rows = keep_rows;
  if (int rc = dc::check_rows(k, n_tokens, who, "keys")) return rc;
  if (int rc = dc::check_rows(v, n_tokens, who, "values")) return rc;
  if (int rc = dc::check_norm(k_norm, who)) return rc;
  if (k.n_heads != v.n_heads || k.dtype != v.dtype) return dc::fail(DC_EINVAL, "%s: keys and values must have one dtype and the same heads", who);
  dc::RotaryJob jobs[3]{};
  int n = 0;
  if (q.n_heads != 0) {  // (0: keys and values alone)
    if (int rc = dc::check_rows(q, n_tokens, who, "queries")) return rc;
    if (int rc = dc::check_rows(q_out, n_tokens, who, "queries out")) return rc;
    if (int rc = dc::check_norm(q_norm, who)) return rc;
    if (q_out.n_heads != q.n_heads) return dc::fail(DC_EINVAL, "%s: queries in and out must have the same heads", who);
    if (q.dtype != k.dtype) return dc::fail(DC_EINVAL, "%s: queries and keys must have one dtype", who);
    jobs[n].in = q;
    jobs[n].norm = q_norm;
    jobs[n].out = q_out;
    jobs[n].rotate = 1;
    ++n;
  }
  for (int i = 0; i < 2; ++i, ++n) {
    jobs[n].in = i ? v : k;
    if (!i) jobs[n].norm = k_norm;
    jobs[n].pages = i ? dest.v_pages : dest.k_pages;
    jobs[n].pool = i ? v_pool : k_pool;
    jobs[n].keep = i ? v_keep : k_keep;
    jobs[n].rotate = !i;
  }
  if (n_tokens == 0) return DC_OK;
  return dc::launch_rotary(R, jobs, n, hipStream_t(stream));
}
