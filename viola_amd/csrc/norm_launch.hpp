// Launches of the norm kernels that hold rows in registers, one pair of types in a file of its own.
#pragma once

#include "norm.hpp"

#include <type_traits>

namespace viola {

// Threads of a block, of a.team for a row. Backward: as many teams as fit 512 threads (1024: 182 against 168 us for 16384 rows of 4096). Forward: of three
// wavefronts and more as many as fit 1024 (102 against 107 us there, 29 against 34 us for 16384 rows of 1152; rows of 512 and 1024 the other way, 31
// against 29 us), and a row to a block where there are few.
inline int norm_block(const NormArgs& a, bool forward) {
    if (forward && a.rows < 1024) return a.team;
    const int most = a.team >= 512 || (forward && a.team >= 192) ? 1024 : 512;
    return !forward && a.team >= 512 ? a.team : most / a.team * a.team;
}

// f(std::integral_constant of a form, std::bool_constant)
template <typename F> void with_form(int form, bool flag, F&& f) {
    auto second = [&](auto form_constant) { flag ? f(form_constant, std::true_type()) : f(form_constant, std::false_type()); };
    if (form == FORM_BEFORE) second(std::integral_constant<int, FORM_BEFORE>());
    else if (form == FORM_AFTER) second(std::integral_constant<int, FORM_AFTER>());
    else if (form == FORM_BETWEEN) second(std::integral_constant<int, FORM_BETWEEN>());
    else second(std::integral_constant<int, FORM_PLAIN>());
}

inline bool any_layer(const NormArgs& a) { return a.after == VIOLA_NORM_LAYER || a.before == VIOLA_NORM_LAYER; }

template <typename TX, typename TY> void norm_forward_rows(const NormArgs& a, int form, dim3 grid, hipStream_t stream) {
    if constexpr (__is_same(TX, loose_t)) {                                  // one kernel for each form
        if (form == FORM_BEFORE) VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_BEFORE, true>), grid, norm_block(a, true), 0, stream, a);
        else if (form == FORM_AFTER) VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_AFTER, true>), grid, norm_block(a, true), 0, stream, a);
        else VIOLA_LAUNCH((norm_forward_kernel<TX, TY, FORM_BETWEEN, true>), grid, norm_block(a, true), 0, stream, a);
    } else {
        with_form(form, any_layer(a), [&](auto f, auto layer) { VIOLA_LAUNCH((norm_forward_kernel<TX, TY, decltype(f)::value, decltype(layer)::value>), grid, norm_block(a, true), 0, stream, a); });
    }
}

// A form has at most the sums of its own sides. Between two blocks a shift before the one without a bias after the other has a kernel of its own: it keeps none
// of its registers in memory with a 16-bit stream and 2 to 9 with a 32-bit one, where the one that has both keeps 10 to 15, and 18 to 23 beside 16-bit blocks, 56 to 59 beside
// 32-bit ones (16 x 1000 rows of 2048, fp32 and bf16: 125 against 150 us).
template <typename TX, typename TY> void norm_backward_rows(const NormArgs& a, int form, bool bias, bool shift, dim3 grid, hipStream_t stream) {
    const int block = norm_block(a, false);
    const unsigned lds = (unsigned)((block / a.team - 1) * a.cols * 4);
    if constexpr (__is_same(TX, loose_t)) {
        if (form == FORM_BEFORE) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BEFORE, true, false, true>), grid, block, lds, stream, a);
        else if (form == FORM_AFTER) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_AFTER, true, true, false>), grid, block, lds, stream, a);
        else VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM_BETWEEN, true, true, true>), grid, block, lds, stream, a);
    } else {
        with_form(form, any_layer(a), [&](auto f, auto layer) {
            constexpr int FORM = decltype(f)::value;
            constexpr bool LAYER = decltype(layer)::value, WITH_BIAS = FORM == FORM_AFTER || FORM == FORM_BETWEEN, WITH_SHIFT = FORM != FORM_AFTER;
            if (FORM == FORM_BETWEEN && shift && !bias) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM, LAYER, false, WITH_SHIFT>), grid, block, lds, stream, a);
            else if ((WITH_BIAS && bias) || (WITH_SHIFT && shift)) VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM, LAYER, WITH_BIAS, WITH_SHIFT>), grid, block, lds, stream, a);
            else VIOLA_LAUNCH((norm_backward_kernel<TX, TY, FORM, LAYER, false, false>), grid, block, lds, stream, a);
        });
    }
}

}  // namespace viola
