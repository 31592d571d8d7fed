// Norms around a block with rows in registers (norm.hpp): a stream of float and branches of bf16_t.
#include "norm_launch.hpp"

template void viola::norm_forward_rows<float, viola::bf16_t>(const viola::NormArgs&, int, dim3, hipStream_t);
template void viola::norm_backward_rows<float, viola::bf16_t>(const viola::NormArgs&, int, bool, bool, dim3, hipStream_t);
