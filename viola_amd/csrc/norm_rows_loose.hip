// Norms around a block with rows in registers (norm.hpp): rows of any type that are no whole aligned pieces.
#include "norm_launch.hpp"

template void viola::norm_forward_rows<viola::loose_t, viola::loose_t>(const viola::NormArgs&, int, dim3, hipStream_t);
template void viola::norm_backward_rows<viola::loose_t, viola::loose_t>(const viola::NormArgs&, int, bool, bool, dim3, hipStream_t);
