// Parameter block of the q / k norm + rotation kernels (qk_norm_rotary.hip).
#pragma once
#include "vfa_kernel_params.h"

namespace vfa {

struct QKNormTensor {
    const void *x, *dy;          // inputs of this side (q or k); dy: backward only
    void *y;                     // forward: output; backward: dx
    const void *w;
    void *dw;                    // backward (same type as w), or null
    int64_t x_bs, x_rs, x_hs, dy_bs, dy_rs, dy_hs, y_bs, y_rs, y_hs;
    int h;
    int toks_sh;                 // a wave's item is the heads of 1 << toks_sh tokens (0: of one token, or a part of them)
};
struct QKNormParams {
    QKNormTensor t[2];           // q, k
    int b, s, d;                 // tokens = b * s
    const int *positions;        // (b, s) with row stride pos_bs, or null: position = index in s
    int64_t pos_bs;
    const void *cos, *sin;       // (table_rows, rd / 2)
    int table_rows, rd, interleaved;
    float eps;
    int is_bf16, table_f32, w_f32;
    float *dw_part;              // backward: (blocks, d) partial sums
    int blocks_q, blocks_k;
};

}  // namespace vfa
