// Internal interface of the products with grouped 4-bit weights (dc_project.hip,
// dc_project_tile.hip).
#pragma once

#include <type_traits>

#include "dc_common.h"

namespace dc {

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
};

namespace {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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

template <int DT>
__device__ __forceinline__ void store_y(void* y, int64_t i, float v) {
  if constexpr (DT == DC_F32)
    static_cast<float*>(y)[i] = v;
  else if constexpr (DT == DC_F16)
    static_cast<_Float16*>(y)[i] = _Float16(v);
  else
    static_cast<__bf16*>(y)[i] = __bf16(v);
}

}  // namespace

// The largest calls of 16-bit rows (dc_project_tile.hip): workspace bytes that they need,
// and whether a call of these sizes is one of them.
bool project_is_tiled(int32_t dtype, int64_t rows, int32_t n, int32_t k);
int64_t project_tile_workspace(int32_t dtype, int64_t rows, int32_t k);
int launch_project_tile(const ProjectArgs& a, int32_t dtype, int group_size, bool affine, void* workspace, hipStream_t stream);

}  // namespace dc
