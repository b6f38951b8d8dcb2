// The layer-product kernels of one type set (-DRWG_PRODUCT_TYPES=<product_types>), so that the
// sets build in parallel.
#include "kernel/general_product.hpp"
#include "kernel/skinny_product.hpp"
#include "kernel/tiled_product.hpp"
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

constexpr product_kernel kNone{nullptr, 0, 0, 0, nullptr, nullptr, 0};
constexpr bool           kSteps = kTypes >= types_steps_square;

template<class Impl>
product_kernel made(int block_m, int block_n, int per_cu)
{
    return {&device::product_entry<Impl>, block_m, block_n, Impl::THREADS, nullptr, nullptr, per_cu};
}

template<int LAYOUT, int BM, int BN, class EPI, bool NARROW = false>
product_kernel tiled()
{
    constexpr bool AK = LAYOUT != layout_mn, BK = LAYOUT == layout_kk;
    using impl        = device::tiled_product<kIn, out_t, res_t, AK, BK, BM, BN, EPI, NARROW>;
    product_fn finish = nullptr;
    if constexpr(!kSteps) // (the steps' products are not cut: their scratch memory holds matrices)
    {
        finish = &device::tiled_finish_entry<impl>;
    }
    return {&device::tiled_product_entry<impl>, BM, BN, impl::THREADS, finish, nullptr, impl::PER_CU};
}

// Only what some call asks for is built.
template<int LAYOUT, int BM, int BN>
product_kernel tiled_finish(int finish)
{
    if constexpr(!kSteps && LAYOUT == layout_mn) // gradients of weights
    {
        switch(finish)
        {
            case finish_plain: return tiled<LAYOUT, BM, BN, device::epilogue_plain>();
            case finish_add: return tiled<LAYOUT, BM, BN, device::epilogue_add>();
            default: return kNone;
        }
    }
    else if constexpr(!kSteps)
    {
        switch(finish)
        {
            case finish_plain: return tiled<LAYOUT, BM, BN, device::epilogue_plain>();
            case finish_layer: return tiled<LAYOUT, BM, BN, device::epilogue_layer>();
            case finish_logistic: return tiled<LAYOUT, BM, BN, device::epilogue_logistic>();
            default: return kNone;
        }
    }
    else if constexpr(kTypes == types_steps_square && LAYOUT == layout_kk)
    {
        switch(finish)
        {
            case finish_square: return tiled<LAYOUT, BM, BN, device::epilogue_square>();
            case finish_poly: return tiled<LAYOUT, BM, BN, device::epilogue_poly>();
            default: return kNone;
        }
    }
    else if constexpr(kTypes != types_steps_square && LAYOUT == layout_kn)
    {
        using epi = std::conditional_t<kTypes == types_steps_next, device::epilogue_next, device::epilogue_last>;
        return tiled<LAYOUT, BM, BN, epi>();
    }
    else
    {
        return kNone;
    }
}

// (an epilogue that finds nothing to add leaves the plain one's result)
template<int LAYOUT>
product_kernel narrow(int finish)
{
    if constexpr(kSteps)
    {
        return kNone;
    }
    else if constexpr(LAYOUT == layout_mn)
    {
        return tiled<LAYOUT, 128, 128, device::epilogue_add, true>();
    }
    else
    {
        return finish == finish_logistic ? tiled<LAYOUT, 128, 128, device::epilogue_logistic, true>()
                                         : tiled<LAYOUT, 128, 128, device::epilogue_layer, true>();
    }
}

template<int LAYOUT, int BM, int BN>
product_kernel skinny()
{
    if constexpr(kSteps && LAYOUT == (kTypes == types_steps_square ? layout_kk : layout_kn) && BM >= 32 && BN >= 32)
    {
        return made<device::skinny_product<kIn, out_t, res_t, BM, BN, LAYOUT == layout_kk, false>>(BM, BN, 0);
    }
    constexpr bool built = (BN == 64 && BM < 64) ? LAYOUT == layout_kn : BN == 16 ? LAYOUT == layout_kk : true;
    if constexpr(!kSteps && LAYOUT != layout_mn && built)
    {
        using impl       = device::skinny_product<kIn, out_t, res_t, BM, BN, LAYOUT == layout_kk, false>;
        using once       = device::skinny_product<kIn, out_t, res_t, BM, BN, LAYOUT == layout_kk, true>;
        product_kernel k = made<impl>(BM, BN, 0);
        k.once           = &device::product_entry<once>;
        return k;
    }
    else
    {
        return kNone;
    }
}

template<int LAYOUT>
product_kernel general(int form)
{
    constexpr bool AK = LAYOUT != layout_mn, BK = LAYOUT == layout_kk;
    if constexpr(kSteps)
    {
        return kNone; // (their operands are the library's own, always aligned)
    }
    else if(form == form_general_128)
    {
        return made<device::general_product<kIn, out_t, res_t, AK, BK, 128, 128, 32>>(128, 128, 8);
    }
    else
    {
        return made<device::general_product<kIn, out_t, res_t, AK, BK, 64, 64, 64>>(64, 64, 8);
    }
}

template<int LAYOUT>
product_kernel in_layout(int form, int finish)
{
    switch(form)
    {
        case form_general_128:
        case form_general_64: return general<LAYOUT>(form);
        case form_tiled_256: return tiled_finish<LAYOUT, 256, 256>(finish);
        case form_tiled_128: return tiled_finish<LAYOUT, 128, 128>(finish);
        case form_tiled_128x256:
            if constexpr(kTypes != types_steps_square) // (a mirrored tile is square)
            {
                return tiled_finish<LAYOUT, 128, 256>(finish);
            }
            return kNone;
        case form_tiled_192:
            if constexpr(kTypes == types_steps_square && LAYOUT == layout_kk)
            {
                return tiled_finish<LAYOUT, 192, 192>(finish);
            }
            return kNone;
        case form_narrow_128: return narrow<LAYOUT>(finish);
        case form_skinny_16x32: return skinny<LAYOUT, 16, 32>();
        case form_skinny_16x64: return skinny<LAYOUT, 16, 64>();
        case form_skinny_32x32: return skinny<LAYOUT, 32, 32>();
        case form_skinny_32x64: return skinny<LAYOUT, 32, 64>();
        case form_skinny_64x32: return skinny<LAYOUT, 64, 32>();
        case form_skinny_64x64: return skinny<LAYOUT, 64, 64>();
        case form_skinny_32x16: return skinny<LAYOUT, 32, 16>();
        default: return kNone;
    }
}
} // namespace

template<int TYPES>
product_kernel product_of(int layout, int form, int finish);

template<>
product_kernel product_of<kTypes>(int layout, int form, int finish)
{
    switch(layout)
    {
        case layout_kk: return in_layout<layout_kk>(form, finish);
        case layout_kn: return in_layout<layout_kn>(form, finish);
        case layout_mn: return in_layout<layout_mn>(form, finish);
        default: return kNone;
    }
}

} // namespace host
} // namespace rocm_wmma_gemm
