// What the host sides of the operators next to the GEMM share: limits, launches that stop behind a failed
// one, statuses, and the choice of a kernel for a product.
#ifndef ROCM_WMMA_GEMM_PRODUCT_HOST_HPP
#define ROCM_WMMA_GEMM_PRODUCT_HOST_HPP

#include <rocm_wmma_gemm_c.h>

#include <algorithm>

#include "host_services.hpp"
#include "product_table.hpp"

namespace rocm_wmma_gemm
{
namespace host
{

// (an extent rounded up to any tile still fits an int)
constexpr size_t most_extent = 0x7fffff00;

// What a launch may have: its threads along x are counted in 32 bits (a kernel with a workgroup for every
// tile may ask for more), its workgroups along y in 16.  most_groups_x: of 256 threads, where they come in parts.
constexpr size_t most_threads_x = 0xffffffff, most_groups_x = size_t{1} << 20, most_groups_y = 65535;

// enqueue(), unless a launch of this call before it was rejected: it would read what that one was to write.
template<class... A>
void follow(A&&... a)
{
    if(launch_failure == hipSuccess)
    {
        enqueue(std::forward<A>(a)...);
    }
}

constexpr size_t ceil_div(size_t a, size_t b)
{
    return (a + b - 1) / b;
}

constexpr size_t round_up8(size_t x)
{
    return (x + 7) / 8 * 8;
}

constexpr size_t whole_lines(size_t bytes)
{
    return (bytes + 255) / 256 * 256;
}

inline hipStream_t stream_of(void* stream)
{
    return stream ? *static_cast<hipStream_t*>(stream) : nullptr;
}

inline size_t out_size(int type_idx)
{
    return type_idx == ROCM_WMMA_GEMM_TYPE_F32_F16 || type_idx == ROCM_WMMA_GEMM_TYPE_F32_BF16 ? 4 : 2;
}

inline bool is_bf16(int type_idx)
{
    return type_idx == ROCM_WMMA_GEMM_TYPE_BF16_BF16 || type_idx == ROCM_WMMA_GEMM_TYPE_F32_BF16;
}

// Runs `body`, a function that returns a status, for an entry point with C linkage: no exception
// leaves it, and a launch that the runtime rejected becomes a status.
template<class Body>
int with_status(Body&& body)
{
    launch_failure = hipSuccess;
    try
    {
        const int rc = body();
        return rc == ROCM_WMMA_GEMM_OK && launch_failure != hipSuccess ? ROCM_WMMA_GEMM_ERR_RUNTIME : rc;
    }
    catch(...)
    {
        return ROCM_WMMA_GEMM_ERR_RUNTIME;
    }
}

// (without a device, for a plan that is only asked for: an MI355X's)
inline size_t compute_units()
{
    const size_t cus = compute_units_of_current_device();
    return cus > 0 ? cus : 256;
}

// Calls f(first, count) for the parts of `all` workgroups that a launch may have along one dimension.
template<class F>
void in_parts(size_t all, size_t most, F&& f)
{
    for(size_t first = 0; first < all; first += most)
    {
        f(static_cast<int>(first), static_cast<unsigned>(std::min(all - first, most)));
    }
}

// Calls f with a null pointer of an element type.
template<class F>
void by_element(int element, F&& f)
{
    switch(element)
    {
        case ROCM_WMMA_GEMM_ELEMENT_F16: f(static_cast<_Float16*>(nullptr)); break;
        case ROCM_WMMA_GEMM_ELEMENT_BF16: f(static_cast<__bf16*>(nullptr)); break;
        default: f(static_cast<float*>(nullptr)); break;
    }
}

// A product's kernel, and how the tiles that would leave compute units idle are cut along K.
struct launch_choice
{
    product_kernel kernel{nullptr, 0, 0, 0, nullptr, nullptr, 0};
    size_t         items = 0; // tiles, or the most there can be (rows: the device knows how many)
    size_t         workgroups = 0;
    size_t         partial_bytes = 0; // room that cutting needs; 0: nothing is cut
    int            k_slices = 1; // workgroups that share a tile of the few-row kernel
    bool           once = false; // B's loads carry the non-temporal hint
    bool           copy_a = false, copy_b = false; // work on padded copies
    size_t         copy_bytes = 0; // room for them
    int            layout = 0, form = 0;
    size_t         scratch() const
    {
        return copy_bytes + partial_bytes;
    }
};

// Which kernel a product runs on: the least estimated time of the forms that can take it.
launch_choice choose(int types, int layout, int finish, const device::product_args& given, size_t cus);

// One product on the kernel chosen for it.  scratch: the room that the choice asked for.  Without it (a
// capture forbids to allocate) nothing is cut, and the general kernel stands in for one that needs copies.
int launch_product(int types, int finish, launch_choice c, device::product_args args, char* scratch, hipStream_t stream);

} // namespace host
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_HOST_HPP
