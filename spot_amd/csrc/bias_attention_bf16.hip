// The kernels of bias_attention.h for elements of type __bf16.
#include "bias_attention.h"

namespace ba {
int launch_bf16(int what, int D, const Args& a, unsigned grid, hipStream_t stream) { return launch<__bf16>(what, D, a, grid, stream); }
}  // namespace ba
