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
#include "dc_common.h"

namespace dc {

namespace {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Weight tiles: 16 outputs x 128 inputs, 1 KiB in the order of the lanes that
// take them: lane l has output l % 16 and, of the tile's inputs, 32 w + 8 (l / 16)
// .. + 7 in its word w.  Input j of a word's eight is nibble j / 2 + 4 (j % 2).
constexpr int kTileN = 16, kTileK = 128;

struct ProjectArgs {
  const uint4* words;     // [N tiles][K tiles][64]
  const uint16_t* scales; // [N tiles][K tiles][16][128 / group] scales, or {scale, bias} pairs
  int32_t n, k, n_tiles, k_tiles;
  const void* x;
  void* y;
  int64_t rows, x_stride, y_stride;
  int32_t x_vec;  // rows of x start at multiples of 16 bytes, and k is a multiple of 8
};

__device__ __forceinline__ float half_of(uint16_t h) { return float(__builtin_bit_cast(_Float16, h)); }

// Eight values 16 + code of a word as a matrix operand.
template <int DT>
__device__ __forceinline__ uint4 operand(uint32_t r) {
  if constexpr (DT == DC_F16) {
    constexpr uint32_t m = 0x03c003c0u, one = 0x4c004c00u;
    return uint4{((r << 6) & m) | one, ((r << 2) & m) | one, ((r >> 2) & m) | one, ((r >> 6) & m) | one};
  } else {
    constexpr uint32_t m = 0x00780078u, one = 0x41804180u;
    return uint4{((r << 3) & m) | one, ((r >> 1) & m) | one, ((r >> 5) & m) | one, ((r >> 9) & m) | one};
  }
}

template <int DT>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (DT == DC_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

// Inputs k .. k + 7 of a row as operands (fp32: three parts), zeros past the
// row's end and for rows that do not exist.
template <int DT, int PARTS>
__device__ __forceinline__ void load_x(const ProjectArgs& a, const void* row, bool has, int k, uint4 (&out)[PARTS]) {
  if constexpr (DT != DC_F32) {
    const uint16_t* p = static_cast<const uint16_t*>(row);
    uint32_t w[4];
    if (a.x_vec) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + (has && k < a.k ? k : 0));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = has && k < a.k ? w[i] : 0;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k0 = k + 2 * i, k1 = k0 + 1;
        const uint32_t lo = p[k0 < a.k ? k0 : 0], hi = p[k1 < a.k ? k1 : 0];
        w[i] = (has && k0 < a.k ? lo : 0) | (has && k1 < a.k ? hi << 16 : 0);
      }
    }
    out[0] = uint4{w[0], w[1], w[2], w[3]};
  } else {
    const float* p = static_cast<const float*>(row);
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = p[k + i < a.k ? k + i : 0];
      v = has && k + i < a.k ? v : 0.f;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t top = __builtin_bit_cast(uint32_t, v) & 0xffff0000u;  // exact: the next part has what is left
        v -= __builtin_bit_cast(float, top);
        w[j][i / 2] = i % 2 ? w[j][i / 2] | top : top >> 16;
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) out[j] = uint4{w[j][0], w[j][1], w[j][2], w[j][3]};
  }
}

template <int DT>
__device__ __forceinline__ void store_y(void* y, int64_t i, float v) {
  if constexpr (DT == DC_F32)
    static_cast<float*>(y)[i] = v;
  else if constexpr (DT == DC_F16)
    static_cast<_Float16*>(y)[i] = _Float16(v);
  else
    static_cast<__bf16*>(y)[i] = __bf16(v);
}

constexpr int kWaves = 4;

}  // namespace

// 16 rows by 16 outputs per block; its wavefronts take the inputs' tiles in turn
// and join in order.
template <int DT, int GS, bool AFFINE>
__global__ void __launch_bounds__(64 * kWaves) project_rows_kernel(ProjectArgs a) {
  constexpr int PARTS = DT == DC_F32 ? 3 : 1, OT = DT == DC_F32 ? DC_BF16 : DT, NG = kTileK / GS;
  constexpr uint32_t kOne = OT == DC_F16 ? 0x3c003c00u : 0x3f803f80u;
  __shared__ f32x4 part_sums[kWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.y) * 16;
  const bool has = row0 + col < a.rows;
  const void* const row = static_cast<const char*>(a.x) + (has ? row0 + col : row0) * a.x_stride * (DT == DC_F32 ? 4 : 2);
  const uint4 ones{kOne, kOne, kOne, kOne};
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  for (int kt = wave; kt < a.k_tiles; kt += kWaves) {
    const int64_t tile = int64_t(blockIdx.x) * a.k_tiles + kt;
    const uint4 r = a.words[tile * 64 + lane];
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    const uint16_t* const sc = a.scales + (tile * 16 + col) * NG * (AFFINE ? 2 : 1);
    f32x4 sum{0.f, 0.f, 0.f, 0.f}, xs{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 x[PARTS];
      load_x<DT, PARTS>(a, row, has, kt * kTileK + 32 * i + 8 * g, x);
      const uint4 b = operand<OT>(w[i]);
#pragma unroll
      for (int j = 0; j < PARTS; ++j) {
        sum = mfma<OT>(x[j], b, sum);
        xs = mfma<OT>(x[j], ones, xs);
      }
      if ((i + 1) * 32 % GS) continue;
      const int gr = i * 32 / GS;
      const float s = half_of(sc[gr * (AFFINE ? 2 : 1)]);
      const float off = AFFINE ? half_of(sc[gr * 2 + 1]) - 16.f * s : -23.f * s;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        acc[v] = fmaf(s, sum[v], fmaf(off, xs[v], acc[v]));
        sum[v] = xs[v] = 0.f;
      }
    }
  }
  part_sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) acc += part_sums[w][lane];
  const int out = int(blockIdx.x) * kTileN + col;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int64_t m = row0 + 4 * g + v;
    if (m < a.rows && out < a.n) store_y<DT>(a.y, m * a.y_stride + out, acc[v]);
  }
}

template <int DT, int GS>
static int launch_project(const ProjectArgs& a, bool affine, hipStream_t stream) {
  // (16 rows a block: at most 2^16 - 1 of them in a launch's second dimension)
  for (int64_t r = 0; r < a.rows; r += 16 * 65535) {
    ProjectArgs b = a;
    b.x = static_cast<const char*>(a.x) + r * a.x_stride * (DT == DC_F32 ? 4 : 2);
    b.y = static_cast<char*>(a.y) + r * a.y_stride * (DT == DC_F32 ? 4 : 2);
    b.rows = a.rows - r < 16 * 65535 ? a.rows - r : 16 * 65535;
    const dim3 grid(uint32_t(a.n_tiles), uint32_t((b.rows + 15) / 16));
    if (affine)
      hipLaunchKernelGGL((project_rows_kernel<DT, GS, true>), grid, dim3(64 * kWaves), 0, stream, b);
    else
      hipLaunchKernelGGL((project_rows_kernel<DT, GS, false>), grid, dim3(64 * kWaves), 0, stream, b);
    if (int rc = check_hip(hipGetLastError(), "project_rows_kernel launch")) return rc;
  }
  return DC_OK;
}

template <int DT>
static int launch_groups(const ProjectArgs& a, int group_size, bool affine, hipStream_t stream) {
  return group_size == 32 ? launch_project<DT, 32>(a, affine, stream)
         : group_size == 64 ? launch_project<DT, 64>(a, affine, stream)
                            : launch_project<DT, 128>(a, affine, stream);
}

}  // namespace dc

extern "C" int64_t dc_grouped_weight_bytes(int32_t outputs, int32_t inputs, int32_t group_size, int32_t affine, int64_t* scales_offset) {
  if (outputs <= 0 || inputs <= 0 || (group_size != 32 && group_size != 64 && group_size != 128)) return -1;
  const int64_t tiles = ((int64_t(outputs) + dc::kTileN - 1) / dc::kTileN) * ((int64_t(inputs) + dc::kTileK - 1) / dc::kTileK);
  if (scales_offset) *scales_offset = tiles * 1024;
  return tiles * (1024 + dc::kTileN * (dc::kTileK / group_size) * (affine ? 4 : 2));
}

extern "C" int dc_project(dc_grouped_weight weight, dc_matrix_rows x, dc_matrix_rows y, int64_t rows, dc_stream_t stream) {
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
  dc::ProjectArgs a{static_cast<const uint4*>(weight.data), reinterpret_cast<const uint16_t*>(static_cast<const char*>(weight.data) + scales),
                    weight.outputs, weight.inputs, (weight.outputs + dc::kTileN - 1) / dc::kTileN,
                    (weight.inputs + dc::kTileK - 1) / dc::kTileK, x.data, y.data, rows, x.stride, y.stride, 0};
  a.x_vec = reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && (x.stride % 8 == 0 || rows == 1) && weight.inputs % 8 == 0;
  const hipStream_t st = hipStream_t(stream);
  return x.dtype == DC_F32   ? dc::launch_groups<DC_F32>(a, weight.group_size, weight.affine, st)
         : x.dtype == DC_F16 ? dc::launch_groups<DC_F16>(a, weight.group_size, weight.affine, st)
                             : dc::launch_groups<DC_BF16>(a, weight.group_size, weight.affine, st);
}
