// Launches of the norm kernels that hold rows in registers, one pair of types in a file of its own.
#pragma once

#include "norm.hpp"

namespace viola {

// a.team threads for a row; as many teams as fit 512 threads
inline int norm_block(const NormArgs& a) { return a.team >= 512 ? a.team : 512 / a.team * a.team; }

template <typename TX, typename TY> void norm_forward_rows(const NormArgs& a, int form, dim3 grid, hipStream_t stream) {
    const int block = norm_block(a);
    if (form == FORM_BEFORE) VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_BEFORE>), grid, block, 0, stream, a);
    else if (form == FORM_AFTER) VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_AFTER>), grid, block, 0, stream, a);
    else VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_BETWEEN>), grid, block, 0, stream, a);
}

template <typename TX, typename TY> void norm_backward_rows(const NormArgs& a, int form, bool bias, bool shift, dim3 grid, hipStream_t stream) {
    const int block = norm_block(a);
    const unsigned lds = (unsigned)((block / a.team - 1) * a.cols * 4);
    if (form == FORM_BEFORE) {
        if (shift) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BEFORE, false, true>), grid, block, lds, stream, a);
        else VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BEFORE, false, false>), grid, block, lds, stream, a);
    } else if (form == FORM_AFTER) {
        if (bias) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_AFTER, true, false>), grid, block, lds, stream, a);
        else VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_AFTER, false, false>), grid, block, lds, stream, a);
    } else if (bias) {
        if (shift) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BETWEEN, true, true>), grid, block, lds, stream, a);
        else VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BETWEEN, true, false>), grid, block, lds, stream, a);
    } else if (shift) {
        VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BETWEEN, false, true>), grid, block, lds, stream, a);
    } else {
        VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BETWEEN, false, false>), grid, block, lds, stream, a);
    }
}

}  // namespace viola
