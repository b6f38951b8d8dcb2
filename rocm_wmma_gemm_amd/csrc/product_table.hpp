// Host-side view of the compiled layer-product kernels: entry points by type set, operand
// layouts and form.  Defined in product_slice.hip, one translation unit per type set.
#ifndef ROCM_WMMA_GEMM_PRODUCT_TABLE_HPP
#define ROCM_WMMA_GEMM_PRODUCT_TABLE_HPP

#include "kernel/product_common.hpp"

namespace rocm_wmma_gemm
{
namespace host
{

using product_fn = void (*)(const device::product_args);

// Types of (A and B, C, residual).  The first four are the library's type pairs, in their order;
// the last four are the products of the Newton-Schulz steps.
enum product_types
{
    types_f16_f16 = 0,
    types_f32_f16,
    types_bf16_bf16,
    types_f32_bf16,
    types_steps_square, // f16 -> f16, f16 residual
    types_steps_next, // f16 -> fp32, fp32 residual
    types_steps_f16, // f16 -> f16, fp32 residual
    types_steps_bf16, // f16 -> bf16, fp32 residual
    num_product_types
};

// Operand layouts: which of A and B have the summed dimension contiguous.
enum product_layout
{
    layout_kk = 0, // both
    layout_kn, // A; B is contiguous along N
    layout_mn, // neither
    num_product_layouts
};

enum product_form
{
    form_general_128 = 0, // 128 x 128 tiles, any alignment
    form_general_64, // 64 x 64 tiles, any alignment
    // rows that start on 16 bytes:
    form_tiled_256, // persistent 256 x 256 tiles
    form_tiled_128, // persistent 128 x 128 tiles
    form_tiled_128x256,
    form_tiled_192, // symmetric products of K-contiguous operands only
    form_narrow_128, // 128 x 128 tiles for rows of C that do not start on 16 bytes
    // whole sums of few rows, rows x columns of a tile
    form_skinny_16x32,
    form_skinny_16x64, // B contiguous along N only: a k row of 64 columns is a whole cache line
    form_skinny_32x32,
    form_skinny_32x64, // likewise
    form_skinny_64x32,
    form_skinny_64x64,
    form_skinny_32x16, // B contiguous along K only
    num_product_forms
};

// What happens to a finished tile (tiled forms; the others read it from the arguments).
enum product_finish
{
    finish_plain = 0, // alpha = 1, nothing added
    finish_add, // a residual is added
    finish_layer, // bias, nothing or relu, residual, the sum kept
    finish_logistic, // the same with silu or gelu
    finish_square, // symmetric
    finish_poly, // symmetric, with a residual and the diagonal held apart
    finish_next, // + diagonal times residual, by rows; kept in A's type as well
    finish_last, // the same, not kept
    num_product_finishes
};

struct product_kernel
{
    product_fn fn; // nullptr: not built
    int        block_m, block_n, threads;
    product_fn finish; // adds up and finishes the tiles that the kernel cut along K; nullptr: it cuts none
    product_fn once; // its twin with non-temporal loads of B; nullptr: none
    int        per_cu; // workgroups of a compute unit, for a persistent kernel; 0: a workgroup per tile
};

product_kernel find_product(int types, int layout, int form, int finish);

} // namespace host
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_TABLE_HPP
