// Host-callable launchers of the embedding lookup and of its gradient by sorted tokens (embedding.cu).  Each returns 0, or a negative code for sizes
// that it does not take and for a launch that was refused.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tb {

// out[t] = scale * table[ids[t]] (rows of D, `ld` elements apart in the table), rounded once; a row of NaN for an id outside [0, V).
[[nodiscard]] int embedding_rows(const void* ids, bool ids64, const void* table, bool table16, int64_t ld, void* out, bool out16, float scale,
                                 int64_t T, int64_t V, int D, cudaStream_t stream);
// dtable[v] = scale * sum over the t with ids[t] == v of dout[t], all V rows; zeros in row `padding` (-1: none).  Ids outside [0, V) add nothing.
// The order of a row's sum is the tokens', split at fixed places.  scratch: embedding_scratch_bytes, on 16 bytes.
int64_t embedding_scratch_bytes(int64_t T, int64_t V, int D, bool dtable16);
int embedding_grad_kernels(int64_t T, int64_t V, int D, bool dtable16);      // that embedding_grad launches
[[nodiscard]] int embedding_grad(const void* ids, bool ids64, const void* dout, bool dout16, int64_t ld, void* dtable, bool dtable16, float scale,
                                 int64_t padding, int64_t T, int64_t V, int D, void* scratch, cudaStream_t stream);

}  // namespace tb
