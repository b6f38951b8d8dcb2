// Instantiates the tiled layer products for a few types, layouts, tiles and epilogues so that the
// host test can look at the generated assembly (see test_operators_host.py).
#include "kernel/tiled_product.hpp"

using namespace rocm_wmma_gemm;

#define SHAPED(IN, OUT, RES, AK, BK, BM, BN, EPI) \
    template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::IN, OUT, RES, AK, BK, BM, BN, device::EPI>>(device::product_args);
#define CHECKED(IN, OUT, RES, AK, BK, EDGE, EPI) SHAPED(IN, OUT, RES, AK, BK, EDGE, EDGE, EPI)

CHECKED(bf16, __bf16, __bf16, true, true, 256, epilogue_plain)
CHECKED(bf16, __bf16, __bf16, true, true, 256, epilogue_logistic)
CHECKED(f16, float, float, true, false, 256, epilogue_layer)
CHECKED(bf16, float, float, false, false, 256, epilogue_add)
CHECKED(bf16, __bf16, __bf16, true, true, 128, epilogue_logistic)
CHECKED(f16, float, float, true, false, 128, epilogue_logistic)
CHECKED(f16, _Float16, _Float16, false, false, 128, epilogue_add)
CHECKED(f16, _Float16, _Float16, true, true, 256, epilogue_poly)
CHECKED(f16, _Float16, _Float16, true, true, 256, epilogue_square)
CHECKED(f16, _Float16, _Float16, true, true, 128, epilogue_poly)
CHECKED(f16, float, float, true, false, 256, epilogue_next)
CHECKED(f16, float, float, true, false, 128, epilogue_next)
CHECKED(f16, __bf16, float, true, false, 256, epilogue_last)
SHAPED(bf16, __bf16, __bf16, true, true, 128, 256, epilogue_logistic)
CHECKED(f16, _Float16, _Float16, true, true, 192, epilogue_poly)
// rows of C that do not start on 16 bytes
template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::bf16, float, float, true, true, 128, 128, device::epilogue_logistic, true>>(device::product_args);
template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::f16, _Float16, _Float16, false, false, 128, 128, device::epilogue_add, true>>(device::product_args);
