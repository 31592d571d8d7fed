// The norms before and after a block with its gate and residual sum: what the kernels of norm.hip compute.
//
//   n(v) = (v - mu) r,  r = (mean((v - mu)^2) + eps)^-1/2,  mu = mean(v), or 0 for the root mean square
//   after the block   x' = rho x + alpha g (n(y) w_a + b_a)         (or n(y) = y)
//   before the next   h  = (n(x') w_b + b_b) (1 + s) + t
//
// Backward, from D_out = dL/dx' and dh, with x' computed again in 32 bits from x and y (as many bytes as reading x' would be, and
// without its rounding):
//   q = dh w_b (1 + s),  D = D_out + r_x (q - x^ mean(q x^) - mean(q)),  dx = rho D,  p = D alpha g w_a,
//   dy = r_y (p - y^ mean(p y^) - mean(p))
// with x^ = (x' - mu_x) r_x and y^ alike (the means without a product only with mu). Sums over rows: A1 = sum D y^, A0 = sum D, S1 = sum dh x^, S0 = sum dh give every
// vector's gradient: dw_a = alpha sum g A1, db_a = alpha sum g A0, dg = alpha (w_a A1 + b_a A0), dw_b = sum (1 + s) S1,
// db_b = sum (1 + s) S0, ds = w_b S1 + b_b S0, dt = S0.
#pragma once

#include "block_ops.hpp"

namespace viola {

enum { FORM_BEFORE = 0, FORM_AFTER = 1, FORM_BETWEEN = 2 };
enum { SUM_A1 = 1, SUM_A0 = 2, SUM_S1 = 4, SUM_S0 = 8 };

// A vector along the row: one for all rows (pitch 0), or one for each group of rows.
struct NormVector {
    const void* data;
    int64_t pitch;
};

struct NormArgs {
    const void *x, *y;
    int64_t x_pitch, y_pitch, rows, group_rows;
    int cols, x_dtype, branch_dtype, after, before, weight_dtype, vector_dtype;
    const void *after_weight, *after_bias, *weight, *bias;
    NormVector gate, scale, shift;
    float rho, alpha, eps;
    // forward
    void *out, *h;
    float4* stats;                                                           // mu_y, r_y, mu_x, r_x of a row
    int64_t chunk;                                                           // rows of a block
    // backward
    const void *dout, *dh;
    void *dx, *dy;
    float* parts;                                                            // [portions][sums][cols]
    int64_t portions, per_group;                                             // portions in all, and of one group
    int sums;                                                                // which sums over rows are wanted (SUM_*)
};

}  // namespace viola
