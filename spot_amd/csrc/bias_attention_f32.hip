// The kernels of bias_attention.h for elements of type float.
#include "bias_attention.h"

namespace ba {
int launch_f32(int what, int D, const Args& a, unsigned grid, hipStream_t stream) { return launch<float>(what, D, a, grid, stream); }
}  // namespace ba
