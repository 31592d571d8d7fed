// Norms around a block with rows in registers (norm.hpp): a stream of f16_t and branches of f16_t.
#include "norm_launch.hpp"

template void viola::norm_forward_rows<viola::f16_t, viola::f16_t>(const viola::NormArgs&, int, dim3, hipStream_t);
template void viola::norm_backward_rows<viola::f16_t, viola::f16_t>(const viola::NormArgs&, int, bool, bool, dim3, hipStream_t);
