// The kernels of bias_attention.h for elements of type _Float16.
#include "bias_attention.h"

namespace ba {
int launch_f16(int what, int D, const Args& a, unsigned grid, hipStream_t stream) { return launch<_Float16>(what, D, a, grid, stream); }
}  // namespace ba
