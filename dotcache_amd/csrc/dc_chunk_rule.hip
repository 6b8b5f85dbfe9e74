// The chunk attention's kernels with a rule (dc_attend_chunk_rule): no cap; a
// file of its own, so that all sets of instances are compiled at once.
#include "dc_chunk_kernels.h"

namespace dc {

int launch_chunks_rule(ChunkArgs a, int32_t n_few, int32_t few_rows, bool units, hipStream_t stream) {
  return launch_all<kRuled>(a, n_few, few_rows, units, stream);
}

}  // namespace dc
