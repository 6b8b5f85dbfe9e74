// The chunk attention's kernels with a rule and a cap (dc_attend_chunk_rule).
#include "dc_chunk_kernels.h"

namespace dc {

int launch_chunks_cap(ChunkArgs a, int32_t n_few, int32_t few_rows, bool units, hipStream_t stream) {
  return launch_all<kCapped>(a, n_few, few_rows, units, stream);
}

}  // namespace dc
