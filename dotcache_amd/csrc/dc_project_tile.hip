// The largest calls of dc_project with 16-bit rows: products of tiles of up to
// 96 rows by 128 outputs.  Bound by the matrix instructions, so weights are
// fp16 operands, scale and bias in them (one rounding, 2^-11 of a weight at
// most, below 2^-14 2^-25), and no sum is touched until the end: 2048 bf16 rows of 3584 x 4608 in 107
// us, 10 of them the rows' preparation (a library product of dense matrices 66,
// project_mid_kernel 154).
#include "dc_project.h"

namespace dc {

namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));

constexpr int kAhead = 3;
constexpr int kTilesN = 2;                  // tiles of outputs that a wavefront takes ...
constexpr int kOutputs = 4 * 16 * kTilesN;  // ... and outputs of a block
constexpr int kOutRow = 16 * kTilesN + 8;   // a wavefront's outputs and a pad that spreads rows over the banks

struct TileArgs {
  ProjectArgs p;      // x: fp16 rows of k_tiles * 128 inputs
  const int32_t* exps;  // [rows]: log2 of what a row of x was divided by; null: nothing
  int32_t y_vec;        // rows of y start at multiples of 16 bytes
};

__device__ __forceinline__ uint32_t twice(uint32_t h) { return h | (h << 16); }

// Eight weights of a word in packed fp16 arithmetic: code s + bias, or (code - 7) s.
// Codes are 16 + code first and whole numbers then, both exact, so that a weight
// is rounded once, where it is made.
template <bool AFFINE>
__device__ __forceinline__ uint4 weights(uint32_t r, h2v s, h2v bias) {
  uint4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t sh = i == 0 ? r << 6 : i == 1 ? r << 2 : i == 2 ? r >> 2 : r >> 6;
    const h2v c = __builtin_bit_cast(h2v, (sh & 0x03c003c0u) | 0x4c004c00u);
    constexpr _Float16 zero = AFFINE ? -16.f : -23.f;
    const h2v d = c + h2v{zero, zero};
    (&out.x)[i] = __builtin_bit_cast(uint32_t, AFFINE ? __builtin_elementwise_fma(d, s, bias) : d * s);
  }
  return out;
}

}  // namespace

// Rows as the tiles' kernel takes them: fp16, whole tiles long, bf16 rows
// divided by the power of two that brings their largest finite value to 2^14 .. 2^15 (what
// fp16 then drops is below 2^-39 of it).
constexpr int64_t kPrepareBlocks = 1 << 20;  // (a launch has fewer than 2^32 threads in a dimension)
template <int DT>
__global__ void __launch_bounds__(256) project_prepare_kernel(ProjectArgs a, uint16_t* out, int32_t* exps) {
  // a block per row (and further ones in turn), eight inputs a thread, up to kRounds loads under way at once
  constexpr int kRounds = 4;
  __shared__ float tops[4];
  const int width = a.k_tiles * kTileK;
  struct Inputs {
    uint16_t h[8];
  };
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {  // (uniform)
    const uint16_t* const row = static_cast<const uint16_t*>(a.x) + r * a.x_stride;
    auto load = [&](int k) {  // (of the row's last ones where it ends sooner)
      Inputs x;
      __builtin_memcpy(x.h, __builtin_assume_aligned(row + min(k, a.k - 8), 2), 16);
      return x;
    };
    int e = 0;
    if constexpr (DT == DC_BF16) {
      float top = 0.f;
      for (int k = 8 * int(threadIdx.x); k < a.k; k += kRounds * 2048) {
        Inputs x[kRounds];
#pragma unroll
        for (int j = 0; j < kRounds; ++j) x[j] = load(k + 2048 * j);
#pragma unroll
        for (int j = 0; j < kRounds; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = fabsf(__builtin_bit_cast(float, uint32_t(x[j].h[i]) << 16));
            top = __builtin_isfinite(v) ? fmaxf(top, v) : top;
          }
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
      if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
      __syncthreads();
      top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;  // (frexp: top in [2^(e - 1), 2^e))
      if (threadIdx.x == 0) exps[r] = e;
    }
    for (int k = 8 * int(threadIdx.x); k < width; k += kRounds * 2048) {
      Inputs x[kRounds];
#pragma unroll
      for (int j = 0; j < kRounds; ++j) x[j] = load(k + 2048 * j);
#pragma unroll
      for (int j = 0; j < kRounds; ++j) {
        const int at = k + 2048 * j;
        if (at >= width) break;
        Inputs y = x[j];
        if (at + 8 > a.k) {  // (moved to their place, those behind the row's end 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y.h[i] = 0;
#pragma unroll
            for (int l = i; l < 8; ++l) y.h[i] = at + i == a.k - 8 + l ? x[j].h[l] : y.h[i];
          }
        }
        if constexpr (DT == DC_BF16) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y.h[i] = __builtin_bit_cast(uint16_t, _Float16(__builtin_amdgcn_ldexpf(__builtin_bit_cast(float, uint32_t(y.h[i]) << 16), -e)));
        }
        *reinterpret_cast<uint4*>(out + r * width + at) = __builtin_bit_cast(uint4, y);
      }
    }
    if (r + gridDim.x < a.rows) __syncthreads();  // (the next row writes tops)
  }
}

// 16 MB rows by kOutputs per block: four wavefronts of 32 outputs.  The rows
// lie in LDS as the operands that all four read, two tiles of inputs in turn;
// weights go from their words to the operands in registers, once each.  (64
// outputs a wavefront read LDS half as often but leave one wavefront to a SIMD:
// 148 us.)
template <int DT, int GS, bool AFFINE, int MB>
__global__ void __launch_bounds__(256, 2) project_tile_kernel(TileArgs t) {
  constexpr int NT = kTilesN, NG = kTileK / GS, SC = NG * (AFFINE ? 2 : 1);
  __shared__ uint4 xt[2][MB][4][64];  // [turn][row block][32 inputs][lane]
  const ProjectArgs& a = t.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.y) * (16 * MB);
  const int n0 = (int(blockIdx.x) * 4 + wave) * NT;
  struct Operand {
    uint32_t w[4];
  };
  Operand x[MB];
  // This wavefront brings the operands of inputs 32 wave .. of a tile.  (Addresses
  // are made where they are used: kept, they would take registers that the sums need.)
  const uint16_t* const base = static_cast<const uint16_t*>(a.x) + row0 * a.x_stride + 32 * wave + 8 * g;
  const int last = int(min(a.rows - row0, int64_t(16 * MB)) - 1);
  auto load_rows = [&](int kt) __attribute__((always_inline)) {
    int at = last;
    asm volatile("" : "+v"(at));
    const uint16_t* const p = base + int64_t(min(kt, a.k_tiles - 1)) * kTileK;
#pragma unroll
    for (int j = 0; j < MB; ++j) __builtin_memcpy(x[j].w, __builtin_assume_aligned(p + min(16 * j + col, at) * a.x_stride, 2), 16);
  };
  auto write_rows = [&](int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < MB; ++j) xt[turn][j][wave][lane] = uint4{x[j].w[0], x[j].w[1], x[j].w[2], x[j].w[3]};
  };
  struct Weights {
    uint4 w[NT];
    uint16_t s[NT][SC];
  };
  auto load_weights = [&](int kt, Weights& w) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t tile = int64_t(min(n0 + n, a.n_tiles - 1)) * a.k_tiles + min(kt, a.k_tiles - 1);  // (uniform)
      w.w[n] = (a.words + tile * 64)[lane];
      __builtin_memcpy(w.s[n], __builtin_assume_aligned(a.scales + tile * 16 * SC + col * SC, 2 * SC), 2 * SC);
    }
  };
  f32x4 acc[MB][NT];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // (a row operand is read kAhead groups of products ahead, a step's weights are
  // made one by one among the products of the step before: the scheduler, left
  // alone, reads one ahead and makes all weights first)
  auto make = [&](const Weights& w, int i, int n) __attribute__((always_inline)) {
    const int gr = i * 32 / GS;
    const h2v s = __builtin_bit_cast(h2v, twice(w.s[n][gr * (AFFINE ? 2 : 1)]));
    const h2v bias = __builtin_bit_cast(h2v, twice(w.s[n][AFFINE ? 2 * gr + 1 : 0]));
    return weights<AFFINE>((&w.w[n].x)[i], s, bias);
  };
  auto take = [&](const Weights& w, int turn) __attribute__((always_inline)) {
    auto rows_of = [&](int k) { return xt[turn][k % MB][k / MB][lane]; };
    uint4 b[2][NT], v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = rows_of(k);
#pragma unroll
    for (int n = 0; n < NT; ++n) b[0][n] = make(w, 0, n);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const int k = i * MB + m, every = MB / NT;
        __builtin_amdgcn_sched_barrier(0);
        if (i < 3 && m % every == 0 && m / every < NT) b[(i + 1) % 2][m / every] = make(w, i + 1, m / every);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = mfma<DC_F16>(v[k % kAhead], b[i % 2][n], acc[m][n]);
        if (k + kAhead < 4 * MB) v[k % kAhead] = rows_of(k + kAhead);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  Weights even, odd;
  load_rows(0);
  load_weights(0, even);
  write_rows(0);
  load_rows(1);
  __syncthreads();
  auto step = [&](int kt, const Weights& now, Weights& next) __attribute__((always_inline)) {
    load_weights(kt + 1, next);
    write_rows((kt + 1) & 1);  // (behind the last: not read)
    load_rows(kt + 2);
    __builtin_amdgcn_sched_barrier(0);  // (loads stay ahead of the products)
    take(now, kt & 1);
    __syncthreads();
  };
  for (int kt = 0;; kt += 2) {
    step(kt, even, odd);
    if (kt + 1 >= a.k_tiles) break;
    step(kt + 1, odd, even);
    if (kt + 2 >= a.k_tiles) break;
  }
  // Out by LDS, so that a wavefront's 32 outputs of a row leave in one piece.
  uint16_t* const turned = reinterpret_cast<uint16_t*>(&xt[0][0][0][0]) + wave * (16 * kOutRow);
  const int out0 = n0 * kTileN;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int e = DT == DC_BF16 ? t.exps[min(row0 + 16 * m + 4 * g + v, a.rows - 1)] : 0;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        store_y<DT>(turned, (4 * g + v) * kOutRow + 16 * n + col, DT == DC_BF16 ? __builtin_amdgcn_ldexpf(acc[m][n][v], e) : acc[m][n][v]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wavefront's own part)
#pragma unroll
    for (int h = 0; h < kTilesN / 2; ++h) {
      constexpr int per = 2 * kTilesN;  // lanes a row, eight outputs each
      const int at = 64 / per * h + lane / per, ch = 8 * (lane % per);
      const int64_t r = row0 + 16 * m + at;
      if (r >= a.rows) continue;
      const uint16_t* const from = turned + at * kOutRow + ch;
      uint16_t* const to = static_cast<uint16_t*>(a.y) + r * a.y_stride + out0 + ch;
      if (t.y_vec && out0 + ch + 8 <= a.n) {
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
      } else {
        for (int i = 0; i < 8 && out0 + ch + i < a.n; ++i) to[i] = from[i];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Time of a call in tiles of 16 mb rows by kOutputs, or (mb 0) in the 64 x 64
// blocks of project_mid_kernel: rounds of 256 blocks times a block's work, in
// units of 16 rows by kOutputs (2048 rows of 3584 x 4608: 4.9 us a unit, a round
// of the others' blocks 17).
static double rounds(int64_t rows, int32_t n, int mb) {
  const int64_t blocks = mb ? ((rows + 16 * mb - 1) / (16 * mb)) * ((int64_t(n) + kOutputs - 1) / kOutputs)
                            : ((rows + 63) / 64) * ((int64_t(n) + 63) / 64);
  return double((blocks + 255) / 256) * (mb ? mb : 3.5);
}

// Row blocks of a tile: what is done first.  (8 are never done before 4 and take
// as long; 10 need more registers than two wavefronts on a SIMD have: 172 us
// where 4 take 109.)
static int tile_rows(int64_t rows, int32_t n) {
  return rounds(rows, n, 6) < rounds(rows, n, 4) ? 6 : 4;
}

bool project_is_tiled(int32_t dtype, int64_t rows, int32_t n, int32_t k) {
  return (dtype == DC_F16 || dtype == DC_BF16) && rows > 64 && n > 0 && k >= kTileK && rounds(rows, n, tile_rows(rows, n)) < rounds(rows, n, 0);
}

static bool needs_rows(int32_t dtype, int32_t k) { return dtype == DC_BF16 || k % kTileK != 0; }

int64_t project_tile_workspace(int32_t dtype, int64_t rows, int32_t k) {
  if (!needs_rows(dtype, k)) return 0;
  return rows * ((int64_t(k) + kTileK - 1) / kTileK * kTileK) * 2 + (dtype == DC_BF16 ? rows * 4 : 0);
}

template <int DT, int GS, bool AFFINE>
static int launch_tile(const TileArgs& t, hipStream_t stream) {
  auto go = [&](auto blocks) {
    constexpr int MB = decltype(blocks)::value;
    const int64_t most = int64_t(16 * MB) * 65535;
    for (int64_t r = 0; r < t.p.rows; r += most) {
      TileArgs b = t;
      b.p.x = static_cast<const uint16_t*>(t.p.x) + r * t.p.x_stride;
      b.p.y = static_cast<uint16_t*>(t.p.y) + r * t.p.y_stride;
      b.p.rows = t.p.rows - r < most ? t.p.rows - r : most;
      b.exps = t.exps ? t.exps + r : nullptr;
      const dim3 grid(uint32_t((t.p.n + kOutputs - 1) / kOutputs), uint32_t((b.p.rows + 16 * MB - 1) / (16 * MB)));
      hipLaunchKernelGGL((project_tile_kernel<DT, GS, AFFINE, MB>), grid, dim3(256), 0, stream, b);
      if (int rc = check_hip(hipGetLastError(), "project_tile_kernel launch")) return rc;
    }
    return int(DC_OK);
  };
  const int mb = tile_rows(t.p.rows, t.p.n);
  return mb == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 6>{});
}

template <int DT>
static int launch_tile_groups(const TileArgs& t, int group_size, bool affine, hipStream_t stream) {
  if (affine)
    return group_size == 32   ? launch_tile<DT, 32, true>(t, stream)
           : group_size == 64 ? launch_tile<DT, 64, true>(t, stream)
                              : launch_tile<DT, 128, true>(t, stream);
  return group_size == 32   ? launch_tile<DT, 32, false>(t, stream)
         : group_size == 64 ? launch_tile<DT, 64, false>(t, stream)
                            : launch_tile<DT, 128, false>(t, stream);
}

int launch_project_tile(const ProjectArgs& a, int32_t dtype, int group_size, bool affine, void* workspace, hipStream_t stream) {
  TileArgs t{a, nullptr, reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride % 8 == 0};
  if (needs_rows(dtype, a.k)) {
    const int64_t width = int64_t(a.k_tiles) * kTileK;
    uint16_t* const rows = static_cast<uint16_t*>(workspace);
    int32_t* const exps = dtype == DC_BF16 ? reinterpret_cast<int32_t*>(rows + a.rows * width) : nullptr;
    const dim3 grid(uint32_t(a.rows < kPrepareBlocks ? a.rows : kPrepareBlocks));
    if (dtype == DC_BF16)
      hipLaunchKernelGGL((project_prepare_kernel<DC_BF16>), grid, dim3(256), 0, stream, a, rows, exps);
    else
      hipLaunchKernelGGL((project_prepare_kernel<DC_F16>), grid, dim3(256), 0, stream, a, rows, nullptr);
    if (int rc = check_hip(hipGetLastError(), "project_prepare_kernel launch")) return rc;
    t.p.x = rows;
    t.p.x_stride = width;
    t.exps = exps;
  }
  return dtype == DC_F16 ? launch_tile_groups<DC_F16>(t, group_size, affine, stream) : launch_tile_groups<DC_BF16>(t, group_size, affine, stream);
}

}  // namespace dc
