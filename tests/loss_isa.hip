// Instantiates the tiled products behind a loss so that the host test can look at the generated assembly (see
// test_head_loss_host.py).
#include "kernel/tiled_product.hpp"

using namespace rocm_wmma_gemm;

#define SHAPED(IN, OUT, AK, BK, BM, BN, EPI) \
    template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::IN, OUT, OUT, AK, BK, BM, BN, device::EPI>>(device::product_args);

SHAPED(bf16, __bf16, true, true, 256, 256, epilogue_parts)
SHAPED(f16, _Float16, true, false, 256, 256, epilogue_parts)
SHAPED(f16, _Float16, true, true, 128, 128, epilogue_parts)
SHAPED(bf16, __bf16, true, false, 128, 256, epilogue_parts)
SHAPED(bf16, __bf16, true, true, 256, 256, epilogue_slope)
SHAPED(f16, _Float16, true, false, 256, 256, epilogue_slope)
SHAPED(f16, _Float16, true, true, 128, 128, epilogue_slope)
SHAPED(bf16, __bf16, true, false, 128, 256, epilogue_slope)
SHAPED(bf16, __bf16, false, false, 256, 256, epilogue_back)
SHAPED(f16, float, false, false, 128, 256, epilogue_back)
template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::f16, _Float16, _Float16, false, false, 128, 256, device::epilogue_back, true, true>>(device::product_args);
template __global__ void device::tiled_product_entry<device::tiled_product<device::in_kind::bf16, float, float, false, false, 128, 256, device::epilogue_back, true, true>>(device::product_args);
