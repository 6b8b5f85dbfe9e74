// Rows times a weight matrix of grouped 4-bit codes (dc_project):
//
//   y_mn = sum_k x_mk W_nk,   W_nk = s_ng c_nk + b_ng   (group g of k)
//        = sum_g s_ng sum_k x_mk (16 + c_nk) + (b_ng - 16 s_ng) sum_k x_mk
//
// 16 + c is exact in bf16 and in fp16, and one shift and one bit operation away
// from two codes of a word (the exponent of 16 joined to the codes in the top
// mantissa bits), so the matrix instructions multiply x as it is by whole
// numbers, exactly, with fp32 sums; scales and offsets act on the groups' sums
// in fp32.  Nothing is rounded before the output.  fp32 rows are three bf16
// parts each, whose sum they are.
//
// By rows: project_few_kernel to 16 (one row of 3584 x 4608, 9.3 MB, 5.9 us; a launch
// with no work 4.2), project_mid_kernel beyond (48 rows of 4096 x 16384, 38 MB, 21
// us; with the few rows' kernel 59), project_tile_kernel (dc_project_tile.hip)
// where its rounds of blocks end first.
#include "dc_project.h"

namespace dc {

namespace {

// Inputs k .. k + 7 of a row, at any alignment, or the row's last eight where
// those end behind it: one load whatever the row, with no branch (a register that
// two branches load would be waited for where they meet).  Rows have eight inputs
// at least.
template <int DT>
struct Eight {
  static constexpr int W = DT == DC_F32 ? 8 : 4;
  uint32_t w[W];
};
template <int DT>
__device__ __forceinline__ void load_x(const ProjectArgs& a, const char* row, int k, Eight<DT>& x) {
  constexpr int item = DT == DC_F32 ? 4 : 2;
  __builtin_memcpy(x.w, __builtin_assume_aligned(row + int64_t(min(k, a.k - 8)) * item, item), sizeof(x.w));
}

// What load_x read, moved to its place, with zeros behind the row's end (for a last tile
// that the row does not fill).
template <int DT>
__device__ __forceinline__ void cut_x(const ProjectArgs& a, int k, Eight<DT>& x) {
  constexpr int W = Eight<DT>::W, per = DT == DC_F32 ? 1 : 2;  // inputs a word
  const int n = a.k - k, d = n >= 8 ? 0 : 8 - n;               // inputs left; how far the load began before k
#pragma unroll
  for (int by = 4; by >= per; by >>= 1)
#pragma unroll
    for (int i = 0; i < W; ++i) x.w[i] = d & by ? (i + by / per < W ? x.w[(i + by / per) % W] : 0) : x.w[i];
  if constexpr (per == 2) {
#pragma unroll
    for (int i = 0; i < W; ++i) x.w[i] = d & 1 ? x.w[i] >> 16 | (i + 1 < W ? x.w[(i + 1) % W] << 16 : 0) : x.w[i];
  }
#pragma unroll
  for (int i = 0; i < W; ++i) x.w[i] = n > 0 ? x.w[i] : 0;
}

// Part `part` of them as a matrix operand (fp32 rows have three bf16 parts: the
// top 16 bits, those of what is left, and the rest).
template <int DT>
__device__ __forceinline__ uint4 x_operand(const Eight<DT>& x, int part) {
  if constexpr (DT != DC_F32) return uint4{x.w[0], x.w[1], x.w[2], x.w[3]};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t top[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // (a register of its own: built in place, over the loaded ones, the operand
      // overwrote words that it still needed, as hipcc 7.2 ordered it)
      uint32_t w = x.w[(2 * i + e) % Eight<DT>::W];
      asm volatile("" : "+v"(w));
      float v = __builtin_bit_cast(float, w);
#pragma unroll
      for (int j = 0; j < part; ++j) v -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u);  // exact
      top[e] = __builtin_bit_cast(uint32_t, v);
    }
    out[i] = __builtin_amdgcn_perm(top[1], top[0], 0x07060302u);
  }
  return uint4{out[0], out[1], out[2], out[3]};
}

constexpr int kFewWaves = 8;

}  // namespace

// Up to 16 rows by 16 outputs per block.  Bound by reading the weights (few
// bytes: by the time from a launch to its first word), so its wavefronts split
// the inputs' tiles among them, a few tiles each in a round whose loads are all
// made first, and join in order at the end.
template <int DT, int GS, bool AFFINE>
__global__ void __launch_bounds__(64 * kFewWaves) project_few_kernel(ProjectArgs a) {
  constexpr int PARTS = DT == DC_F32 ? 3 : 1, OT = DT == DC_F32 ? DC_BF16 : DT, SC = kTileK / GS * (AFFINE ? 2 : 1);
  constexpr int T = DT == DC_F32 ? 1 : 2;  // tiles a round (4: the same time, more code)
  constexpr uint32_t kOne = OT == DC_F16 ? 0x3c003c00u : 0x3f803f80u;
  __shared__ f32x4 joined[kFewWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.y) * 16;
  // (rows that do not exist repeat the last one: their sums are not stored)
  const char* const row = static_cast<const char*>(a.x) + (row0 + col < a.rows ? row0 + col : a.rows - 1) * a.x_stride * (DT == DC_F32 ? 4 : 2);
  const int64_t tile0 = int64_t(blockIdx.x) * a.k_tiles;
  const uint4* const words = a.words + tile0 * 64 + lane;
  const uint16_t* const scales = a.scales + (tile0 * 16 + col) * SC;
  struct Stage {
    uint4 w;
    uint16_t s[SC];
    Eight<DT> x[4];
  };
  auto load = [&](int t, Stage& st) __attribute__((always_inline)) {
    st.w = words[int64_t(t) * 64];
    __builtin_memcpy(st.s, __builtin_assume_aligned(scales + int64_t(t) * 16 * SC, 2 * SC), 2 * SC);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_x<DT>(a, row, t * kTileK + 32 * i + 8 * g, st.x[i]);
  };
  const uint4 ones{kOne, kOne, kOne, kOne};
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  auto take = [&](int kt, Stage& st) __attribute__((always_inline)) {
    if (kt == a.k_tiles - 1 && a.k % kTileK != 0) {  // (uniform)
#pragma unroll
      for (int i = 0; i < 4; ++i) cut_x<DT>(a, kt * kTileK + 32 * i + 8 * g, st.x[i]);
    }
    f32x4 sum, xs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i * 32 % GS == 0) sum = xs = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint4 b = operand<OT>((&st.w.x)[i]);
#pragma unroll
      for (int j = 0; j < PARTS; ++j) {
        const uint4 x = x_operand<DT>(st.x[i], j);
        xs = mfma<OT>(x, ones, xs);
        sum = mfma<OT>(x, b, sum);
      }
      if ((i + 1) * 32 % GS) continue;
      const int gr = i * 32 / GS;
      const float s = half_of(st.s[gr * (AFFINE ? 2 : 1)]);
      const float off = AFFINE ? half_of(st.s[(2 * gr + 1) % SC]) - 16.f * s : -23.f * s;
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v] = fmaf(s, sum[v], fmaf(off, xs[v], acc[v]));
    }
  };
  // All of a round's loads are under way before its first product; the card's
  // other wavefronts fill the wait between rounds.
  for (int kt = wave; kt < a.k_tiles; kt += T * waves) {  // (uniform)
    Stage st[T];
#pragma unroll
    for (int j = 0; j < T; ++j) load(min(kt + j * waves, a.k_tiles - 1), st[j]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < T; ++j)
      if (kt + j * waves < a.k_tiles) take(kt + j * waves, st[j]);
  }
  joined[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < waves; ++w) acc += joined[w][lane];
  const int out = int(blockIdx.x) * kTileN + col;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int64_t r = row0 + 4 * g + v;
    if (r < a.rows && out < a.n) store_y<DT>(a.y, r * a.y_stride + out, acc[v]);
  }
}

// Sum of a row's eight 16-bit inputs (products with 1, which are exact; fp32 sums).
template <int DT>
__device__ __forceinline__ float sum8(const uint4& x) {
  typedef _Float16 h2v __attribute__((ext_vector_type(2)));
  typedef __bf16 b2v __attribute__((ext_vector_type(2)));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (&x.x)[i];
    if constexpr (DT == DC_F16)
      s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2v, w), __builtin_bit_cast(h2v, 0x3c003c00u), s, false);
    else
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, w), __builtin_bit_cast(b2v, 0x3f803f80u), s, false);
  }
  return s;
}

// 16 MB rows by 64 outputs per block, 16-bit rows: four wavefronts, a tile of
// outputs each, on each half of the inputs' tiles.  A half's rows lie in LDS as
// the matrix operands that all four read, with their groups' sums, two tiles in
// turn: while one is worked on the next is written from registers, and the one
// after it is on its way.
template <int DT, int GS, bool AFFINE, int MB>
__global__ void __launch_bounds__(512, 2) project_mid_kernel(ProjectArgs a) {
  constexpr int NG = kTileK / GS, SC = NG * (AFFINE ? 2 : 1);
  static_assert(MB <= 4, "a wavefront brings one row block");
  __shared__ uint4 xt[2][2][MB][4][64];    // [half][turn][row block][32 inputs][lane]
  __shared__ f32x4 xsum[2][2][MB][NG][4];  // sums of the groups' inputs of four rows
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2, mine = wave & 3;
  const int col = lane & 15, g = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.y) * (16 * MB);
  const int n_tile = int(blockIdx.x) * 4 + mine;
  const int64_t r = row0 + 16 * min(mine, MB - 1) + col;  // the row that this lane brings
  const char* const row = static_cast<const char*>(a.x) + (r < a.rows ? r : a.rows - 1) * a.x_stride * 2;
  const int64_t tile0 = int64_t(min(n_tile, a.n_tiles - 1)) * a.k_tiles;
  const uint4* const words = a.words + tile0 * 64 + lane;
  const uint16_t* const scales = a.scales + (tile0 * 16 + col) * SC;
  struct Weights {
    uint4 w;
    uint16_t s[SC];
  };
  Eight<DT> x[4];
  auto load_rows = [&](int kt) __attribute__((always_inline)) {
    const int t = min(kt, a.k_tiles - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_x<DT>(a, row, t * kTileK + 32 * i + 8 * g, x[i]);
  };
  auto load_weights = [&](int kt, Weights& w) __attribute__((always_inline)) {
    const int t = min(kt, a.k_tiles - 1);
    w.w = words[int64_t(t) * 64];
    __builtin_memcpy(w.s, __builtin_assume_aligned(scales + int64_t(t) * 16 * SC, 2 * SC), 2 * SC);
  };
  auto write_rows = [&](int kt, int turn) __attribute__((always_inline)) {
    if (mine >= MB) return;
    if (kt >= a.k_tiles - 1 && a.k % kTileK != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) cut_x<DT>(a, kt * kTileK + 32 * i + 8 * g, x[i]);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = x_operand<DT>(x[i], 0);
      xt[half][turn][mine][i][lane] = v;
      s = (i * 32 % GS == 0 ? 0.f : s) + sum8<DT>(v);
      if ((i + 1) * 32 % GS) continue;
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (g == 0) reinterpret_cast<float*>(&xsum[half][turn][mine][i * 32 / GS][0])[col] = s;
    }
  };
  f32x4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto take = [&](const Weights& w, int turn) __attribute__((always_inline)) {
    f32x4 sum[MB];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 b = operand<DT>((&w.w.x)[i]);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if (i * 32 % GS == 0) sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
        sum[m] = mfma<DT>(xt[half][turn][m][i][lane], b, sum[m]);
      }
      if ((i + 1) * 32 % GS) continue;
      const int gr = i * 32 / GS;
      const float s = half_of(w.s[gr * (AFFINE ? 2 : 1)]);
      const float off = AFFINE ? half_of(w.s[(2 * gr + 1) % SC]) - 16.f * s : -23.f * s;
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const f32x4 xs = xsum[half][turn][m][gr][g];
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[m][v] = fmaf(s, sum[m][v], fmaf(off, xs[v], acc[m][v]));
      }
    }
  };
  // half h takes tiles h, h + 2, ...; both run as many turns (the second's last
  // may be past the end: rows of the last tile, and no sums taken)
  Weights even, odd;
  load_rows(half);
  load_weights(half, even);
  write_rows(half, 0);
  load_rows(half + 2);
  const int turns = (a.k_tiles + 1) / 2;
  __syncthreads();
  auto step = [&](int t, const Weights& now, Weights& next) __attribute__((always_inline)) {
    const int kt = 2 * t + half;
    load_weights(kt + 2, next);
    write_rows(kt + 2, (t + 1) & 1);  // (behind the last: not read)
    load_rows(kt + 4);
    __builtin_amdgcn_sched_barrier(0);  // (loads stay ahead of the products)
    if (kt < a.k_tiles) take(now, t & 1);
    __syncthreads();
  };
  for (int t = 0;; t += 2) {
    step(t, even, odd);
    if (t + 1 >= turns) break;
    step(t + 1, odd, even);
    if (t + 2 >= turns) break;
  }
  f32x4* const joined = reinterpret_cast<f32x4*>(xt);  // [4][MB][64]
  if (half == 1) {
#pragma unroll
    for (int m = 0; m < MB; ++m) joined[(mine * MB + m) * 64 + lane] = acc[m];
  }
  __syncthreads();
  if (half == 1) return;
  const int out = n_tile * kTileN + col;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const f32x4 y = acc[m] + joined[(mine * MB + m) * 64 + lane];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t at = row0 + 16 * m + 4 * g + v;
      if (at < a.rows && out < a.n) store_y<DT>(a.y, at * a.y_stride + out, y[v]);
    }
  }
}

// Rows of fewer than eight inputs: a thread per output.
template <int DT>
__global__ void __launch_bounds__(256) project_short_kernel(ProjectArgs a, int32_t group_size, int32_t affine) {
  const int out = int(blockIdx.x) * 256 + int(threadIdx.x);
  const int64_t r = blockIdx.y;
  if (out >= a.n) return;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.words + int64_t(out / kTileN) * a.k_tiles * 64 + out % kTileN);
  const uint16_t* sc = a.scales + (int64_t(out / kTileN) * a.k_tiles * 16 + out % kTileN) * (kTileK / group_size) * (affine ? 2 : 1);
  const float s = half_of(sc[0]), b = affine ? half_of(sc[1]) : -7.f * s;
  float sum = 0.f, xs = 0.f;
  for (int k = 0; k < a.k; ++k) {
    const float x = load_value(a.x, DT, r * a.x_stride + k);
    sum = fmaf(float(w[0] >> (4 * (k / 2 + 4 * (k % 2))) & 15u), x, sum);
    xs += x;
  }
  store_y<DT>(a.y, r * a.y_stride + out, fmaf(s, sum, b * xs));
}

// Wavefronts per block of project_few_kernel: kFewWaves where blocks of four leave
// the card's 1024 SIMDs less than four wavefronts each and there is a tile for each, else
// four (16 leave a compute unit one block: one row of 3584 x 4608 7.4 us, 8 5.9).
static int waves_of(int64_t blocks, int k_tiles) {
  return blocks * 4 < 4096 && kFewWaves <= k_tiles ? kFewWaves : 4;
}

// launch(args, grid) for portions of the rows and outputs, blocks of `rows` x
// `outputs` of them: a launch holds 2^16 - 1 blocks in its second dimension, and fewer
// than 2^32 threads in its first (2^22 blocks of 512).  side: scales and biases of an output in a tile.
template <typename F>
static int by_blocks(const ProjectArgs& a, int item, int side, int outputs, int rows, const char* what, F launch) {
  const int64_t most = int64_t(rows) * 65535, wide = int64_t(outputs) << 22;
  for (int64_t n = 0; n < a.n; n += wide) {
    for (int64_t r = 0; r < a.rows; r += most) {
      ProjectArgs b = a;
      b.n = int32_t(a.n - n < wide ? a.n - n : wide);
      b.n_tiles = (b.n + kTileN - 1) / kTileN;
      b.words = a.words + n / kTileN * a.k_tiles * 64;
      b.scales = a.scales + n / kTileN * a.k_tiles * 16 * side;
      b.x = static_cast<const char*>(a.x) + r * a.x_stride * item;
      b.y = static_cast<char*>(a.y) + (r * a.y_stride + n) * item;
      b.rows = a.rows - r < most ? a.rows - r : most;
      launch(b, dim3(uint32_t((b.n + outputs - 1) / outputs), uint32_t((b.rows + rows - 1) / rows)));
      if (int rc = check_hip(hipGetLastError(), what)) return rc;
    }
  }
  return DC_OK;
}

template <int DT>
static int launch_short(const ProjectArgs& a, int group_size, bool affine, hipStream_t stream) {
  return by_blocks(a, DT == DC_F32 ? 4 : 2, kTileK / group_size * (affine ? 2 : 1), 256, 1, "project_short_kernel launch", [&](const ProjectArgs& b, dim3 grid) {
    hipLaunchKernelGGL((project_short_kernel<DT>), grid, dim3(256), 0, stream, b, group_size, int32_t(affine));
  });
}

template <int DT, int GS, bool AFFINE>
static int launch_project(const ProjectArgs& a, hipStream_t stream) {
  constexpr int side = kTileK / GS * (AFFINE ? 2 : 1);
  if constexpr (DT != DC_F32) {
    auto mid = [&](auto blocks) {
      constexpr int MB = decltype(blocks)::value;
      return by_blocks(a, 2, side, 64, 16 * MB, "project_mid_kernel launch", [&](const ProjectArgs& b, dim3 grid) {
        hipLaunchKernelGGL((project_mid_kernel<DT, GS, AFFINE, MB>), grid, dim3(512), 0, stream, b);
      });
    };
    if (a.rows > 48) return mid(std::integral_constant<int, 4>{});
    if (a.rows > 32) return mid(std::integral_constant<int, 3>{});
    if (a.rows > 16) return mid(std::integral_constant<int, 2>{});
  }
  return by_blocks(a, DT == DC_F32 ? 4 : 2, side, 16, 16, "project_few_kernel launch", [&](const ProjectArgs& b, dim3 grid) {
    hipLaunchKernelGGL((project_few_kernel<DT, GS, AFFINE>), grid, dim3(64 * waves_of(int64_t(grid.x) * grid.y, a.k_tiles)), 0, stream, b);
  });
}

template <int DT>
static int launch_groups(const ProjectArgs& a, int group_size, bool affine, hipStream_t stream) {
  if (a.k < 8) return launch_short<DT>(a, group_size, affine, stream);
  if (affine)
    return group_size == 32   ? launch_project<DT, 32, true>(a, stream)
           : group_size == 64 ? launch_project<DT, 64, true>(a, stream)
                              : launch_project<DT, 128, true>(a, stream);
  return group_size == 32   ? launch_project<DT, 32, false>(a, stream)
         : group_size == 64 ? launch_project<DT, 64, false>(a, stream)
                            : launch_project<DT, 128, false>(a, stream);
}

}  // namespace dc

extern "C" int64_t dc_grouped_weight_bytes(int32_t outputs, int32_t inputs, int32_t group_size, int32_t affine, int64_t* scales_offset) {
  if (outputs <= 0 || inputs <= 0 || outputs > 1 << 30 || inputs > 1 << 30 || (group_size != 32 && group_size != 64 && group_size != 128)) return -1;
  const int64_t tiles = ((int64_t(outputs) + dc::kTileN - 1) / dc::kTileN) * ((int64_t(inputs) + dc::kTileK - 1) / dc::kTileK);
  if (scales_offset) *scales_offset = tiles * 1024;
  return tiles * (1024 + dc::kTileN * (dc::kTileK / group_size) * (affine ? 4 : 2));
}

extern "C" int64_t dc_project_workspace_bytes(dc_grouped_weight weight, int32_t dtype, int64_t rows) {
  return dc::project_is_tiled(dtype, rows, weight.outputs, weight.inputs) ? dc::project_tile_workspace(dtype, rows, weight.inputs) : 0;
}

extern "C" int dc_project(dc_grouped_weight weight, dc_matrix_rows x, dc_matrix_rows y, int64_t rows, void* workspace, int64_t workspace_bytes,
                          dc_stream_t stream) {
  const char* who = "dc_project";
  int64_t scales = 0;
  if (dc_grouped_weight_bytes(weight.outputs, weight.inputs, weight.group_size, weight.affine, &scales) < 0)
    return dc::fail(DC_EINVAL, "%s: a weight needs outputs, inputs and groups of 32, 64 or 128", who);
  if (rows < 0) return dc::fail(DC_EINVAL, "%s: bad counts", who);
  if (rows == 0) return DC_OK;
  if (!weight.data || !x.data || !y.data) return dc::fail(DC_EINVAL, "%s: null pointer", who);
  if (x.dtype != DC_F32 && x.dtype != DC_F16 && x.dtype != DC_BF16) return dc::fail(DC_EINVAL, "%s: rows must be DC_F32, DC_F16 or DC_BF16", who);
  if (y.dtype != x.dtype) return dc::fail(DC_EINVAL, "%s: the output needs the rows' dtype", who);
  if (reinterpret_cast<uintptr_t>(weight.data) % 16) return dc::fail(DC_EINVAL, "%s: a weight must be 16-byte aligned", who);
  const int item = x.dtype == DC_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x.data) % item || reinterpret_cast<uintptr_t>(y.data) % item)
    return dc::fail(DC_EINVAL, "%s: rows must be aligned to their type", who);
  if (rows > 1 && (y.stride > -int64_t(weight.outputs) && y.stride < int64_t(weight.outputs)))
    return dc::fail(DC_EINVAL, "%s: the output's rows must not overlap", who);
  const bool tiled = dc::project_is_tiled(x.dtype, rows, weight.outputs, weight.inputs);
  const int64_t need = tiled ? dc::project_tile_workspace(x.dtype, rows, weight.inputs) : 0;
  if (workspace_bytes < need || (need && !workspace)) return dc::fail(DC_ESPACE, "%s: workspace too small", who);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return dc::fail(DC_EINVAL, "%s: workspace must be 16-byte aligned", who);
  const dc::ProjectArgs a{static_cast<const uint4*>(weight.data), reinterpret_cast<const uint16_t*>(static_cast<const char*>(weight.data) + scales),
                    weight.outputs, weight.inputs, (weight.outputs + dc::kTileN - 1) / dc::kTileN,
                    (weight.inputs + dc::kTileK - 1) / dc::kTileK, x.data, y.data, rows, x.stride, y.stride};
  const hipStream_t st = hipStream_t(stream);
  if (tiled) return dc::launch_project_tile(a, x.dtype, weight.group_size, weight.affine, workspace, st);
  return x.dtype == DC_F32   ? dc::launch_groups<DC_F32>(a, weight.group_size, weight.affine, st)
         : x.dtype == DC_F16 ? dc::launch_groups<DC_F16>(a, weight.group_size, weight.affine, st)
                             : dc::launch_groups<DC_BF16>(a, weight.group_size, weight.affine, st);
}
