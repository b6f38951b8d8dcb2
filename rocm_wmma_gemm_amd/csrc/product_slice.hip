// The layer-product kernels of one type set (-DRWG_PRODUCT_TYPES=<product_types>), so that the
// sets build in parallel.
#include "kernel/general_product.hpp"
#include "product_table.hpp"

namespace rocm_wmma_gemm
{
namespace host
{

namespace
{
constexpr int kTypes = RWG_PRODUCT_TYPES;
constexpr device::in_kind kIn
    = kTypes == types_bf16_bf16 || kTypes == types_f32_bf16 ? device::in_kind::bf16 : device::in_kind::f16;
using out_t = std::conditional_t<
    kTypes == types_f16_f16 || kTypes == types_steps_square || kTypes == types_steps_f16, _Float16,
    std::conditional_t<kTypes == types_bf16_bf16 || kTypes == types_steps_bf16, __bf16, float>>;
using res_t = std::conditional_t<kTypes == types_steps_f16 || kTypes == types_steps_bf16, float, out_t>;

template<class Impl>
product_kernel made(int block_m, int block_n)
{
    return {&device::product_entry<Impl>, block_m, block_n, Impl::THREADS};
}

template<int LAYOUT>
product_kernel in_layout(int form)
{
    constexpr bool AK = LAYOUT != layout_mn, BK = LAYOUT == layout_kk;
    switch(form)
    {
        case form_general_128: return made<device::general_product<kIn, out_t, res_t, AK, BK, 128, 128, 32>>(128, 128);
        case form_general_64: return made<device::general_product<kIn, out_t, res_t, AK, BK, 64, 64, 64>>(64, 64);
        default: return {nullptr, 0, 0, 0};
    }
}
} // namespace

template<int TYPES>
product_kernel product_of(int layout, int form);

template<>
product_kernel product_of<kTypes>(int layout, int form)
{
    switch(layout)
    {
        case layout_kk: return in_layout<layout_kk>(form);
        case layout_kn: return in_layout<layout_kn>(form);
        case layout_mn: return in_layout<layout_mn>(form);
        default: return {nullptr, 0, 0, 0};
    }
}

} // namespace host
} // namespace rocm_wmma_gemm
