// Host side of what stands around a layer of experts: the choice of the experts, the rows sorted by expert, the
// weighted sum of their rows, and the gradients of these.  They are additions with no counterpart in the reference.
#include <cmath>

#include "kernel/routing.hpp"
#include "product_host.hpp"

namespace rocm_wmma_gemm
{
namespace host
{
namespace
{

// Tokens of a call, and choices (their places are ints).
constexpr size_t most_tokens = most_extent, most_slots = most_extent;

bool is_element(int code)
{
    return code >= ROCM_WMMA_GEMM_ELEMENT_F16 && code <= ROCM_WMMA_GEMM_ELEMENT_F32;
}

size_t element_size(int code)
{
    return code == ROCM_WMMA_GEMM_ELEMENT_F32 ? 4 : 2;
}

bool is_score(int code)
{
    return code == ROCM_WMMA_GEMM_SCORE_SOFTMAX || code == ROCM_WMMA_GEMM_SCORE_SIGMOID;
}

// Whether an address may be read in pieces of that many bytes (a power of two).
bool starts_on(const void* p, size_t bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Calls f with a number of a lane's experts as a type: the smallest power of two that holds them.
template<class F>
void by_chunk(int chunk, F&& f)
{
    chunk <= 1    ? f(std::integral_constant<int, 1>{})
    : chunk <= 2  ? f(std::integral_constant<int, 2>{})
    : chunk <= 4  ? f(std::integral_constant<int, 4>{})
    : chunk <= 8  ? f(std::integral_constant<int, 8>{})
    : chunk <= 16 ? f(std::integral_constant<int, 16>{})
    : chunk <= 32 ? f(std::integral_constant<int, 32>{})
                  : f(std::integral_constant<int, 64>{});
}

// A run of a lane's elements starts on its pieces: all of `chunk`, in every lane and row.
template<class T, int CHUNK>
bool whole_runs(const void* p, int chunk)
{
    return chunk == CHUNK && starts_on(p, std::min<size_t>(16, CHUNK * sizeof(T)));
}

dim3 token_groups(long long tokens)
{
    return dim3(static_cast<unsigned>(std::min(ceil_div(tokens, 256 / device::route_lanes), most_groups_x)));
}

template<class InT, bool SIGMOID>
void launch_route(const device::route_args& a, hipStream_t stream)
{
    by_chunk(a.chunk, [&](auto c) {
        constexpr int CHUNK = decltype(c)::value;
        const bool    lanes_full = a.spread * a.groups == device::route_lanes && a.size == a.spread * a.chunk;
        const bool    whole = lanes_full && whole_runs<InT, CHUNK>(a.logits, a.chunk) && whole_runs<float, CHUNK>(a.bias, a.chunk);
        auto with = [&](auto kernel) { follow(kernel, token_groups(a.tokens), dim3(256), stream, a); };
        if(a.k <= 8)
        {
            whole ? with(&device::route<InT, CHUNK, SIGMOID, true, 8>) : with(&device::route<InT, CHUNK, SIGMOID, false, 8>);
        }
        else
        {
            with(&device::route<InT, CHUNK, SIGMOID, false, device::most_choices>);
        }
    });
}

template<class InT, bool SIGMOID>
void launch_route_backward(const device::route_back_args& a, hipStream_t stream)
{
    by_chunk(a.chunk, [&](auto c) {
        constexpr int CHUNK = decltype(c)::value;
        if constexpr(CHUNK <= 32) // (512 experts on 16 lanes)
        {
            const bool whole = a.experts == a.chunk * device::route_lanes && whole_runs<InT, CHUNK>(a.logits, a.chunk)
                               && whole_runs<InT, CHUNK>(a.dlogits, a.chunk);
            follow(whole ? &device::route_backward<InT, CHUNK, SIGMOID, true> : &device::route_backward<InT, CHUNK, SIGMOID, false>,
                   token_groups(a.tokens), dim3(256), stream, a);
        }
    });
}

int route(int type, int* chosen, float* weights, const void* logits, const rocm_wmma_gemm_routing& r, size_t M, size_t E,
          size_t k, hipStream_t stream)
{
    if(!is_element(type) || !is_score(r.score) || r.groups < 1 || r.kept_groups < 1 || r.kept_groups > r.groups
       || r.group_best < 1 || r.group_best > 2 || (r.renormalize & ~1) || !std::isfinite(r.scale))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    if(M > most_tokens || E > device::max_groups || k > device::most_choices || r.groups > device::most_parts || M * k > most_slots)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    if(M == 0 || k == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    const size_t groups = r.groups;
    if(E == 0 || E % groups != 0 || k > E / groups * r.kept_groups || chosen == nullptr || weights == nullptr || logits == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    device::route_args a{chosen, weights, logits, r.bias, r.mask, static_cast<long long>(M), static_cast<int>(E),
                         static_cast<int>(k), r.groups, static_cast<int>(E / groups), r.kept_groups, r.group_best, 1, 0,
                         r.renormalize, r.scale};
    // (as many lanes a group as there are, a power of two)
    while(2 * a.spread * a.groups <= device::route_lanes)
    {
        a.spread *= 2;
    }
    a.chunk = static_cast<int>(ceil_div(a.size, a.spread));
    by_element(type, [&](auto* typed) {
        using in_t = std::remove_pointer_t<decltype(typed)>;
        r.score == ROCM_WMMA_GEMM_SCORE_SIGMOID ? launch_route<in_t, true>(a, stream) : launch_route<in_t, false>(a, stream);
    });
    return ROCM_WMMA_GEMM_OK;
}

int route_backward(int type, void* dlogits, const float* dweights, const int* chosen, const void* logits, size_t M, size_t E,
                   size_t k, int score, int renormalize, float scale, hipStream_t stream)
{
    if(!is_element(type) || !is_score(score) || (renormalize & ~1) || !std::isfinite(scale))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    if(M > most_tokens || E > device::max_groups || k > device::most_choices || M * k > most_slots)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    if(M == 0 || E == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if(dlogits == nullptr || logits == nullptr || (k != 0 && (dweights == nullptr || chosen == nullptr)))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    const device::route_back_args a{dlogits, dweights, chosen, logits, static_cast<long long>(M), static_cast<int>(E),
                                    static_cast<int>(k), renormalize, static_cast<int>(ceil_div(E, device::route_lanes)), scale};
    by_element(type, [&](auto* typed) {
        using in_t = std::remove_pointer_t<decltype(typed)>;
        score == ROCM_WMMA_GEMM_SCORE_SIGMOID ? launch_route_backward<in_t, true>(a, stream) : launch_route_backward<in_t, false>(a, stream);
    });
    return ROCM_WMMA_GEMM_OK;
}

// Calls f with a null pointer of a piece of a row: 16 bytes on any element, or an element of a shorter row.
template<class F>
void by_piece(size_t bytes, F&& f)
{
    bytes == 16 ? f(static_cast<device::piece16*>(nullptr)) : f(static_cast<device::piece2*>(nullptr));
}

// Counts that every workgroup adds up for itself rather than wait for a launch that does (8191 tokens of 6 choices
// over 128 experts, 1536 counts: 59 us against 65).
constexpr size_t most_added_up = 8192;

int dispatch(int type, void* rows, int* offsets, int* places, const void* x, const int* chosen, size_t E, size_t M, size_t N,
             size_t k, hipStream_t stream)
{
    if(!is_element(type))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    if(E > device::most_dispatch || M > most_tokens || N > most_extent || k > device::most_choices || M * k > most_slots)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    const size_t slots = M * k;
    const bool   copy  = rows != nullptr && N != 0 && slots != 0;
    if(offsets == nullptr || (slots != 0 && (places == nullptr || chosen == nullptr)) || (copy && x == nullptr))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    device::dispatch_args a{rows, offsets, places, x, chosen, nullptr, static_cast<long long>(slots), static_cast<long long>(M),
                            static_cast<long long>(N * element_size(type)), static_cast<int>(E), static_cast<int>(k), 1, copy};
    const size_t blocks = std::max<size_t>(1, ceil_div(slots, device::sort_block));
    a.blocks            = static_cast<int>(blocks);
    const size_t piece  = a.row_bytes >= 16 ? 16 : 2;
    if(blocks == 1)
    {
        // (a run of 64 pieces a wave, spread over the compute units)
        const size_t runs = M * ceil_div(ceil_div(a.row_bytes, piece), 64);
        const dim3   grid(static_cast<unsigned>(copy ? std::min<size_t>(std::max<size_t>(1, ceil_div(runs, 4)), compute_units()) : 1));
        by_piece(piece, [&](auto* typed) {
            using piece_t = std::remove_pointer_t<decltype(typed)>;
            follow(slots <= device::sort_round ? &device::dispatch_few<1, piece_t> : &device::dispatch_few<device::sort_rounds, piece_t>,
                   grid, dim3(1024), stream, a);
        });
        return ROCM_WMMA_GEMM_OK;
    }
    workspace_lease lease;
    a.counts = reinterpret_cast<int*>(lease.acquire(blocks * std::max<size_t>(1, E) * sizeof(int), stream));
    if(a.counts == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    follow(&device::dispatch_rank, dim3(static_cast<unsigned>(blocks)), dim3(1024), stream, a);
    const bool scanned = blocks * E > most_added_up;
    if(scanned)
    {
        follow(&device::dispatch_scan, dim3(1), dim3(1024), stream, a);
    }
    // (eight workgroups a compute unit where there are so many tokens; their choices end in the next block at the latest)
    const bool   streamed = slots * N * element_size(type) >= device::streamed_bytes;
    const size_t each = std::min(std::max<size_t>(4, ceil_div(M, 8 * compute_units())), device::sort_block / k);
    by_piece(piece, [&](auto* typed) {
        using piece_t = std::remove_pointer_t<decltype(typed)>;
        follow(streamed ? (scanned ? &device::dispatch_rows<piece_t, true, true> : &device::dispatch_rows<piece_t, false, true>)
                        : (scanned ? &device::dispatch_rows<piece_t, true, false> : &device::dispatch_rows<piece_t, false, false>),
               dim3(static_cast<unsigned>(ceil_div(M, each))), dim3(256), stream, a, static_cast<int>(each));
    });
    return ROCM_WMMA_GEMM_OK;
}

// Calls f with null pointers of the rows' and the output's types; false if the two do not go together.
template<class F>
bool by_pair(int rows_type, int out_type, F&& f)
{
    if(!is_element(rows_type) || (out_type != rows_type && out_type != ROCM_WMMA_GEMM_ELEMENT_F32))
    {
        return false;
    }
    by_element(rows_type, [&](auto* in) {
        out_type == rows_type ? f(in, in) : f(in, static_cast<float*>(nullptr));
    });
    return true;
}

int check_rows(size_t M, size_t N, size_t k)
{
    return M > most_tokens || N > most_extent || k > device::most_choices || M * k > most_slots ? ROCM_WMMA_GEMM_ERR_LIMIT
                                                                                                : ROCM_WMMA_GEMM_OK;
}

int combine(int rows_type, int out_type, const device::combine_args& a, hipStream_t stream)
{
    by_pair(rows_type, out_type, [&](auto* in_typed, auto* out_typed) {
        using in_t  = std::remove_pointer_t<decltype(in_typed)>;
        using out_t = std::remove_pointer_t<decltype(out_typed)>;
        in_parts(ceil_div(a.cols, 2048), most_groups_y, [&](int block0, unsigned blocks) {
            follow(&device::combine<in_t, out_t>, dim3(static_cast<unsigned>(std::min<long long>(a.tokens, most_groups_x)), blocks), dim3(256),
                   stream, a, block0);
        });
    });
    return ROCM_WMMA_GEMM_OK;
}

int combine_backward(int rows_type, int out_type, const device::combine_args& a, hipStream_t stream)
{
    const bool streamed = static_cast<size_t>(a.slots) * a.cols * element_size(rows_type) >= device::streamed_bytes;
    by_pair(rows_type, out_type, [&](auto* in_typed, auto* out_typed) {
        using in_t  = std::remove_pointer_t<decltype(in_typed)>;
        using out_t = std::remove_pointer_t<decltype(out_typed)>;
        follow(streamed ? &device::combine_backward<in_t, out_t, true> : &device::combine_backward<in_t, out_t, false>,
               dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(a.slots, 4), most_groups_x))), dim3(256), stream, a);
    });
    return ROCM_WMMA_GEMM_OK;
}

} // namespace
} // namespace host
} // namespace rocm_wmma_gemm

extern "C" {

using namespace rocm_wmma_gemm::host;
namespace device = rocm_wmma_gemm::device;

int rocm_wmma_gemm_route(int logits_type, int* chosen, float* weights, const void* logits,
                         const rocm_wmma_gemm_routing* routing, size_t M, size_t E, size_t k, void* stream)
{
    return with_status([&] {
        return routing == nullptr ? ROCM_WMMA_GEMM_ERR_ARGUMENT
                                  : route(logits_type, chosen, weights, logits, *routing, M, E, k, stream_of(stream));
    });
}

int rocm_wmma_gemm_route_backward(int logits_type, void* dlogits, const float* dweights, const int* chosen,
                                  const void* logits, size_t M, size_t E, size_t k, int score, int renormalize, float scale,
                                  void* stream)
{
    return with_status([&] {
        return route_backward(logits_type, dlogits, dweights, chosen, logits, M, E, k, score, renormalize, scale,
                              stream_of(stream));
    });
}

int rocm_wmma_gemm_dispatch(int rows_type, void* rows, int* offsets, int* places, const void* X, const int* chosen,
                            size_t E, size_t M, size_t N, size_t k, void* stream)
{
    return with_status([&] { return dispatch(rows_type, rows, offsets, places, X, chosen, E, M, N, k, stream_of(stream)); });
}

int rocm_wmma_gemm_combine(int rows_type, int out_type, void* C, const void* rows, const int* places, const float* weights,
                           const void* residual, size_t M, size_t N, size_t k, void* stream)
{
    return with_status([&] {
        if(!by_pair(rows_type, out_type, [](auto*, auto*) {}))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        const int rc = check_rows(M, N, k);
        if(rc != ROCM_WMMA_GEMM_OK || M == 0 || N == 0)
        {
            return rc;
        }
        if(C == nullptr || (k != 0 && (rows == nullptr || places == nullptr)))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return combine(rows_type, out_type,
                       {C, rows, places, weights, residual, static_cast<long long>(M), static_cast<long long>(N),
                        static_cast<long long>(M * k), static_cast<int>(k), nullptr, nullptr, nullptr},
                       stream_of(stream));
    });
}

int rocm_wmma_gemm_combine_backward(int rows_type, int out_type, void* drows, float* dweights, const void* dC,
                                    const void* rows, const int* places, const float* weights, size_t M, size_t N, size_t k,
                                    void* stream)
{
    return with_status([&] {
        if(!by_pair(rows_type, out_type, [](auto*, auto*) {}))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        const int rc = check_rows(M, N, k);
        if(rc != ROCM_WMMA_GEMM_OK || M == 0 || k == 0 || (drows == nullptr && dweights == nullptr))
        {
            return rc;
        }
        if(places == nullptr || (N != 0 && (dC == nullptr || (dweights != nullptr && rows == nullptr))))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return combine_backward(rows_type, out_type,
                                {nullptr, rows, places, weights, nullptr, static_cast<long long>(M), static_cast<long long>(N),
                                 static_cast<long long>(M * k), static_cast<int>(k), drows, dweights, dC},
                                stream_of(stream));
    });
}

} // extern "C"
