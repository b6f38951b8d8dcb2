// Host side of the operators next to the GEMM: a linear layer with its epilogue, the same for
// groups of rows (experts), their backward passes, and Newton-Schulz steps on an update.  They
// are additions with no counterpart in the reference.
#include <rocm_wmma_gemm_c.h>

#include <algorithm>
#include <cmath>
#include <exception>

#include "host_services.hpp"
#include "kernel/product_pointwise.hpp"
#include "product_table.hpp"

namespace rocm_wmma_gemm
{
namespace host
{

template<int TYPES>
product_kernel product_of(int layout, int form, int finish);
#define RWG_TYPES(T) \
    template<>       \
    product_kernel product_of<T>(int layout, int form, int finish);
RWG_TYPES(0)
RWG_TYPES(1)
RWG_TYPES(2)
RWG_TYPES(3)
RWG_TYPES(4)
RWG_TYPES(5)
RWG_TYPES(6)
RWG_TYPES(7)
#undef RWG_TYPES

product_kernel find_product(int types, int layout, int form, int finish)
{
    switch(types)
    {
        case 0: return product_of<0>(layout, form, finish);
        case 1: return product_of<1>(layout, form, finish);
        case 2: return product_of<2>(layout, form, finish);
        case 3: return product_of<3>(layout, form, finish);
        case 4: return product_of<4>(layout, form, finish);
        case 5: return product_of<5>(layout, form, finish);
        case 6: return product_of<6>(layout, form, finish);
        case 7: return product_of<7>(layout, form, finish);
        default: return {nullptr, 0, 0, 0, 0};
    }
}

namespace
{
using device::act_args;
using device::act_kind;
using device::product_args;
using device::product_kind;

constexpr size_t most_extent = 0x7fffffff;

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

hipStream_t stream_of(void* stream)
{
    return stream ? *static_cast<hipStream_t*>(stream) : nullptr;
}

size_t out_size(int type_idx)
{
    return type_idx == ROCM_WMMA_GEMM_TYPE_F32_F16 || type_idx == ROCM_WMMA_GEMM_TYPE_F32_BF16 ? 4 : 2;
}

bool is_bf16(int type_idx)
{
    return type_idx == ROCM_WMMA_GEMM_TYPE_BF16_BF16 || type_idx == ROCM_WMMA_GEMM_TYPE_F32_BF16;
}

// The constants of an activation; false for a code that is none.
bool activation_of(int code, act_args* act)
{
    constexpr float two_root_2_over_pi = 1.5957691216057308f;
    switch(code)
    {
        case ROCM_WMMA_GEMM_ACT_NONE: *act = {act_kind::none, 0.0f, 0.0f}; return true;
        case ROCM_WMMA_GEMM_ACT_RELU: *act = {act_kind::relu, 0.0f, 0.0f}; return true;
        case ROCM_WMMA_GEMM_ACT_SILU: *act = {act_kind::logistic, 1.0f, 0.0f}; return true;
        case ROCM_WMMA_GEMM_ACT_GELU:
            *act = {act_kind::logistic, two_root_2_over_pi, two_root_2_over_pi * 0.044715f};
            return true;
        default: return false;
    }
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
    catch(const std::exception&)
    {
        return ROCM_WMMA_GEMM_ERR_RUNTIME;
    }
}

// Whether the kernels that load 16 bytes at a time, straight to LDS, can take the operands: every row,
// and every group's first, starts on 16 bytes, and a tile's span fits the 31 bits of their offsets.
bool aligned_rows(const product_args& a, int layout)
{
    const bool k_contiguous = layout != layout_mn;
    return a.lda % 8 == 0 && a.ldb % 8 == 0 && a.ldc % 8 == 0 && a.N % 8 == 0 && (k_contiguous ? a.K % 8 == 0 : a.M % 8 == 0)
           && a.stride_a % 8 == 0 && a.stride_b % 8 == 0 && a.stride_c % 8 == 0 && aligned16(a.A) && aligned16(a.B)
           && aligned16(a.C) && aligned16(a.kept) && aligned16(a.residual) && aligned16(a.bias) && a.K > 0
           && std::max({a.lda, a.ldb, a.ldc}) < (1 << 21);
}

// Which kernel a product runs on.
int choose_form(int types, int layout, int finish, const product_args& args, size_t cus)
{
    auto tiles = [&](size_t edge) {
        const size_t n = ceil_div(args.N, edge);
        return args.kind == product_kind::rows ? (args.M / edge + std::min<size_t>(args.groups, args.M)) * n
                                               : args.groups * ceil_div(args.M, edge) * n;
    };
    if(!aligned_rows(args, layout))
    {
        return tiles(128) < cus ? form_general_64 : form_general_128;
    }
    const size_t rows = args.kind == product_kind::rows ? ceil_div(args.M, std::min<size_t>(args.groups, args.M)) : args.M;
    if(args.kind == product_kind::rows && rows <= 64
       && (layout == layout_kk || static_cast<long long>(args.K) * args.ldb < (1ll << 30)))
    {
        return rows <= 16 ? form_skinny_16x32 : rows <= 32 ? form_skinny_32x32 : form_skinny_64x32;
    }
    return rows <= 160 || tiles(256) < cus ? form_tiled_128 : form_tiled_256;
}

// One product: picks the kernel and launches it.
int launch_product(int types, int layout, int finish, product_args args, hipStream_t stream)
{
    if(args.N == 0 || args.M == 0 || args.groups == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    const size_t         cus    = std::max<size_t>(compute_units_of_current_device(), 1);
    const product_kernel kernel = find_product(types, layout, choose_form(types, layout, finish, args, cus), finish);
    if(kernel.fn == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    const size_t grid_m = ceil_div(args.M, kernel.block_m), grid_n = ceil_div(args.N, kernel.block_n);
    // (rows: how many tiles there are is only known on the device; at most this many)
    const size_t items = args.kind == product_kind::rows
                             ? (args.M / kernel.block_m + std::min<size_t>(args.groups, args.M)) * grid_n
                             : args.groups * grid_m * grid_n;
    if(items > most_extent)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    args.grid_m = static_cast<int>(grid_m);
    args.grid_n = static_cast<int>(grid_n);
    const size_t blocks = kernel.per_cu == 0 ? items : std::min(items, kernel.per_cu * cus);
    enqueue(kernel.fn, dim3(static_cast<unsigned>(blocks)), dim3(kernel.threads), stream, args);
    return ROCM_WMMA_GEMM_OK;
}

// A linear layer's problem, for one weight (groups = 1 and no offsets) or one per group of rows.
struct layer
{
    int        type_idx;
    size_t     M, N, K;
    int        layout_b;
    const int* offsets;
    size_t     groups;
    act_args   act;
};

int check_layer(const layer& p)
{
    if(p.type_idx < 0 || p.type_idx > ROCM_WMMA_GEMM_TYPE_F32_BF16 || (p.layout_b & ~1))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    if(p.M > most_extent || p.N > most_extent || p.K > most_extent || p.groups > device::max_groups)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    return ROCM_WMMA_GEMM_OK;
}

product_args arguments(const layer& p)
{
    product_args a{};
    a.offsets = p.offsets;
    a.groups  = static_cast<int>(p.groups);
    a.alpha   = 1.0f;
    a.beta    = 1.0f;
    return a;
}

// C = act(A B + bias) + residual
int forward(const layer& p, void* C, const void* A, const void* B, const rocm_wmma_gemm_epilogue& e,
            hipStream_t stream)
{
    if(p.M == 0 || p.N == 0 || p.groups == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if(C == nullptr || (p.K != 0 && (A == nullptr || B == nullptr)))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    product_args a = arguments(p);
    a.C            = C;
    a.kept         = e.preact;
    a.A            = A;
    a.B            = B;
    a.bias         = e.bias;
    a.residual     = e.residual;
    a.act          = p.act;
    a.kind         = product_kind::rows;
    a.M            = static_cast<int>(p.M);
    a.N            = static_cast<int>(p.N);
    a.K            = static_cast<int>(p.K);
    a.lda          = p.K;
    a.ldb          = p.layout_b == 1 ? p.K : p.N;
    a.ldc          = p.N;
    a.stride_b     = static_cast<long long>(p.N * p.K);
    a.stride_bias  = p.N;
    const int finish = p.act.kind == act_kind::logistic ? finish_logistic
                       : p.act.kind == act_kind::relu || e.bias || e.residual || e.preact ? finish_layer
                                                                                          : finish_plain;
    return launch_product(p.type_idx, p.layout_b == 1 ? layout_kk : layout_kn, finish, a, stream);
}

template<class InT>
void launch_slope(const device::slope_args& s, size_t runs, bool wide, hipStream_t stream)
{
    const unsigned columns = wide ? 512 : 64;
    enqueue(wide ? &device::activation_slope<InT, 8> : &device::activation_slope<InT, 1>,
            dim3(static_cast<unsigned>(runs), static_cast<unsigned>(ceil_div(s.cols, columns))), dim3(256), stream, s);
}

template<class OutT>
void launch_column_sums(const device::slope_args& s, void* dbias, int accumulate, hipStream_t stream)
{
    enqueue(&device::column_sums<OutT>, dim3(static_cast<unsigned>(ceil_div(s.cols, 64)), static_cast<unsigned>(s.groups)),
            dim3(64), stream, s, static_cast<OutT*>(dbias), accumulate);
}

// dZ = dC act'(Z); dA = dZ B^T, dB = A^T dZ, dbias = sum of dZ's rows, group by group
int backward(const layer& p, void* dA, void* dB, void* dbias, const void* dC, const void* A, const void* B,
             const void* preact, int accumulate, hipStream_t stream)
{
    const bool sloped = p.act.kind != act_kind::none;
    if(p.groups == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if((p.M != 0 && p.N != 0 && (dC == nullptr || (sloped && preact == nullptr)))
       || (dA != nullptr && p.N != 0 && p.K != 0 && B == nullptr)
       || (dB != nullptr && p.M != 0 && p.K != 0 && A == nullptr))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    workspace_lease lease;
    const void*     dz = dC;
    if((sloped || dbias != nullptr) && p.N != 0)
    {
        const size_t runs     = p.M / device::slope_rows + std::min(p.groups, p.M);
        const size_t dz_bytes = sloped ? whole_lines(p.M * p.N * 2) : 0;
        const size_t sums     = dbias != nullptr ? runs * p.N * sizeof(float) : 0;
        char*        ws       = nullptr;
        if(dz_bytes + sums != 0)
        {
            ws = lease.acquire(dz_bytes + sums, stream);
            if(ws == nullptr)
            {
                return ROCM_WMMA_GEMM_ERR_SCRATCH;
            }
        }
        device::slope_args s{};
        s.dc      = dC;
        s.z       = sloped ? preact : nullptr;
        s.dz      = sloped ? ws : nullptr;
        s.sums    = dbias != nullptr ? reinterpret_cast<float*>(ws + dz_bytes) : nullptr;
        s.offsets = p.offsets;
        s.groups  = static_cast<int>(p.groups);
        s.rows    = static_cast<int>(p.M);
        s.cols    = static_cast<int>(p.N);
        s.act     = p.act;
        if(runs > most_extent || ceil_div(p.N, 64) > 65535)
        {
            return ROCM_WMMA_GEMM_ERR_LIMIT;
        }
        if(runs != 0)
        {
            const bool wide = p.N % 8 == 0 && aligned16(dC) && (!sloped || aligned16(preact));
            is_bf16(p.type_idx) ? launch_slope<__bf16>(s, runs, wide, stream)
                                : launch_slope<_Float16>(s, runs, wide, stream);
        }
        if(sloped)
        {
            dz = ws;
        }
        if(dbias != nullptr)
        {
            switch(p.type_idx)
            {
                case ROCM_WMMA_GEMM_TYPE_F16_F16: launch_column_sums<_Float16>(s, dbias, accumulate, stream); break;
                case ROCM_WMMA_GEMM_TYPE_BF16_BF16: launch_column_sums<__bf16>(s, dbias, accumulate, stream); break;
                default: launch_column_sums<float>(s, dbias, accumulate, stream); break;
            }
        }
    }
    int rc = ROCM_WMMA_GEMM_OK;
    if(dA != nullptr)
    {
        product_args a = arguments(p);
        a.C            = dA;
        a.A            = dz;
        a.B            = B;
        a.kind         = product_kind::rows;
        a.M            = static_cast<int>(p.M);
        a.N            = static_cast<int>(p.K);
        a.K            = static_cast<int>(p.N);
        a.lda          = p.N;
        a.ldb          = p.layout_b == 1 ? p.K : p.N;
        a.ldc          = p.K;
        a.stride_b     = static_cast<long long>(p.N * p.K);
        rc             = launch_product(p.type_idx, p.layout_b == 1 ? layout_kn : layout_kk, finish_plain, a, stream);
    }
    if(rc == ROCM_WMMA_GEMM_OK && dB != nullptr)
    {
        // stored N x K: dZ^T A; stored K x N: A^T dZ
        const bool   nk = p.layout_b == 1;
        product_args a  = arguments(p);
        a.C             = dB;
        a.A             = nk ? dz : A;
        a.B             = nk ? A : dz;
        a.residual      = accumulate ? dB : nullptr;
        a.kind          = product_kind::sum;
        a.M             = static_cast<int>(nk ? p.N : p.K);
        a.N             = static_cast<int>(nk ? p.K : p.N);
        a.K             = static_cast<int>(p.M);
        a.lda           = a.M;
        a.ldb           = a.N;
        a.ldc           = a.N;
        a.stride_c      = static_cast<long long>(p.N * p.K);
        rc              = launch_product(p.type_idx, layout_mn, accumulate ? finish_add : finish_plain, a, stream);
    }
    return rc;
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

// Newton-Schulz steps X <- a X + (b S + c S^2) X with S = X X^T (X^T X where X is tall, on the
// other side), on X = G / (|G| + epsilon).
//
// What is rounded, and why: products take f16 operands.  Every singular value of X stays below
// 1.3, so f16 holds X (scaled by about the root of its smaller side, a power of two, which
// keeps its elements near 1), S and Q = b S + c S^2 with 11 bits; bf16 would leave 8.  Two terms
// are kept from that rounding, because it is the largest part of the error there:
//   - a X: small singular directions grow 3.4 times a step, and a rounding of the large ones
//     (white noise in all directions) with them, so X is also kept in fp32 and only the products
//     see the f16 copy;
//   - Q's diagonal: near the end Q is about -2.7 I, and rounding that moves whole rows of X by
//     four times as much.  The diagonal stays in fp32 beside Q, whose own is zero, and meets the
//     fp32 X in the epilogue: X = (a + diagonal) X + Q X.
// Against 64 bits, 512 x 1024: 7.5e-4 for noise, 2.4e-4 for a momentum of 16 strong directions (2.1e-2
// with all of it from f16, 1.6e-1 from bf16); 1 x 40: 7.2e-4 (3.7e-3 with the diagonal in f16).
int orthogonalize(int given_type, int out_type, void* O, const void* G, size_t M, size_t N, size_t batch, int steps,
                  const float* coefficients, float epsilon, hipStream_t stream)
{
    if(std::min(M, N) <= device::small_side && std::max(M, N) <= device::small_length)
    {
        const device::steps_args small{G, O, static_cast<int>(M), static_cast<int>(N), steps, coefficients[0],
                                       coefficients[1], coefficients[2], epsilon};
        const bool               f16 = out_type == ROCM_WMMA_GEMM_ELEMENT_F16;
        auto run = [&](auto* typed) {
            using given_t = std::remove_pointer_t<decltype(typed)>;
            enqueue(f16 ? &device::orthogonal_small<given_t, _Float16> : &device::orthogonal_small<given_t, __bf16>,
                    dim3(static_cast<unsigned>(batch)), dim3(256), stream, small);
        };
        by_element(given_type, run);
        return ROCM_WMMA_GEMM_OK;
    }
    const bool   tall = M > N;
    const size_t mp = round_up8(M), np = round_up8(N), lp = std::min(mp, np);
    const size_t each = mp * np, square = lp * lp;
    const bool   direct  = mp == M && np == N && aligned16(O);
    const size_t parts_b = whole_lines(batch * device::square_parts * sizeof(float)),
                 diag_b = whole_lines(batch * lp * sizeof(float)), x32_b = whole_lines(batch * each * 4),
                 x16_b = whole_lines(batch * each * 2), sq_b = whole_lines(batch * square * 2);
    if(batch * each > (size_t{1} << 36))
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    workspace_lease lease;
    char*           ws = lease.acquire(parts_b + diag_b + x32_b + 2 * x16_b + 2 * sq_b, stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    float*    parts = reinterpret_cast<float*>(ws);
    float*    diagonal = reinterpret_cast<float*>(ws + parts_b);
    float*    x32   = reinterpret_cast<float*>(ws + parts_b + diag_b);
    char*     rest  = ws + parts_b + diag_b + x32_b;
    _Float16* x16[2] = {reinterpret_cast<_Float16*>(rest), reinterpret_cast<_Float16*>(rest + x16_b)};
    char*     s = rest + 2 * x16_b;
    char*     q = s + sq_b;
    const float scale = std::exp2(std::round(std::log2(std::sqrt(static_cast<float>(std::min(M, N))))));

    auto start = [&](auto* typed) {
        using given_t = std::remove_pointer_t<decltype(typed)>;
        const given_t* given = static_cast<const given_t*>(G);
        enqueue(&device::sum_squares<given_t>, dim3(device::square_parts, static_cast<unsigned>(batch)), dim3(256), stream,
                given, static_cast<long long>(M * N), parts);
        enqueue(&device::orthogonal_start<given_t>,
                dim3(static_cast<unsigned>(ceil_div(each / 8, 256)), static_cast<unsigned>(batch)), dim3(256), stream, given,
                parts, x32, x16[0], static_cast<int>(M), static_cast<int>(N), static_cast<int>(mp), static_cast<int>(np),
                scale, epsilon);
    };
    by_element(given_type, start);
    const float a = coefficients[0], b = coefficients[1], c = coefficients[2];
    product_args p{};
    p.kind   = product_kind::batch;
    p.groups = static_cast<int>(batch);
    p.diagonal = diagonal, p.stride_diagonal = lp;
    int rc   = ROCM_WMMA_GEMM_OK;
    for(int step = 0; step < steps && rc == ROCM_WMMA_GEMM_OK; ++step)
    {
        _Float16* x    = x16[step & 1];
        const bool last = step + 1 == steps;
        // S = X X^T / scale^2
        p.C = s, p.A = x, p.B = x, p.residual = nullptr, p.kept = nullptr;
        p.M = p.N = static_cast<int>(lp), p.K = static_cast<int>(tall ? mp : np);
        p.lda = p.ldb = np, p.ldc = lp;
        p.stride_a = p.stride_b = each, p.stride_c = square;
        p.alpha = 1.0f / (scale * scale), p.beta = 0.0f, p.diagonal_is = device::diagonal_use::none;
        rc = launch_product(types_steps_square, tall ? layout_mn : layout_kk, finish_square, p, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            break;
        }
        // Q = b S + c S^2 (S is its own transpose)
        p.C = q, p.A = p.B = s, p.residual = s;
        p.K = static_cast<int>(lp), p.lda = p.ldb = lp, p.stride_a = p.stride_b = square;
        p.alpha = c, p.beta = b, p.diagonal_is = device::diagonal_use::split;
        rc = launch_product(types_steps_square, layout_kk, finish_poly, p, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            break;
        }
        // X = (a + diagonal) X + Q X (tall: X (a + diagonal) + X Q, Q its own transpose)
        p.A = tall ? static_cast<void*>(x) : q, p.B = tall ? q : static_cast<char*>(static_cast<void*>(x));
        p.M = static_cast<int>(mp), p.N = static_cast<int>(np), p.K = static_cast<int>(lp);
        p.lda = tall ? np : lp, p.ldb = tall ? lp : np, p.ldc = np;
        p.stride_a = tall ? each : square, p.stride_b = tall ? square : each, p.stride_c = each;
        p.residual = x32, p.alpha = last ? 1.0f / scale : 1.0f, p.beta = last ? a / scale : a;
        p.diagonal_is = tall ? device::diagonal_use::cols : device::diagonal_use::rows;
        p.C = last ? (direct ? O : static_cast<void*>(x16[(step + 1) & 1])) : x32;
        p.kept = last ? nullptr : x16[(step + 1) & 1], p.keep_sum = 1;
        rc = launch_product(!last ? types_steps_next
                            : out_type == ROCM_WMMA_GEMM_ELEMENT_F16 ? types_steps_f16 : types_steps_bf16,
                            tall ? layout_kk : layout_kn,
                            last ? (tall ? finish_last_cols : finish_last_rows) : tall ? finish_next_cols : finish_next_rows,
                            p, stream);
        p.keep_sum = 0;
    }
    if(rc == ROCM_WMMA_GEMM_OK && !direct)
    {
        // (a 16-bit element is a 16-bit element)
        enqueue(&device::orthogonal_end<unsigned short>,
                dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(M * N, 256), 4096)), static_cast<unsigned>(batch)),
                dim3(256), stream, reinterpret_cast<const unsigned short*>(x16[steps & 1]), static_cast<unsigned short*>(O),
                static_cast<int>(M), static_cast<int>(N), static_cast<int>(mp), static_cast<int>(np));
    }
    return rc;
}

} // namespace
} // namespace host
} // namespace rocm_wmma_gemm

extern "C" {

using namespace rocm_wmma_gemm::host;

int rocm_wmma_gemm_grouped(int type_idx, void* C, const void* A, const void* B, const int* offsets, size_t groups,
                           size_t M, size_t N, size_t K, int layout_b, const rocm_wmma_gemm_epilogue* epilogue,
                           void* stream)
{
    return with_status([&] {
        const rocm_wmma_gemm_epilogue none{};
        const rocm_wmma_gemm_epilogue& e = epilogue ? *epilogue : none;
        layer p{type_idx, M, N, K, layout_b, offsets, groups, {}};
        const int rc = check_layer(p);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(!activation_of(e.activation, &p.act) || (groups != 0 && offsets == nullptr))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return forward(p, C, A, B, e, stream_of(stream));
    });
}

int rocm_wmma_gemm_grouped_backward(int type_idx, void* dA, void* dB, void* dbias, const void* dC, const void* A,
                                    const void* B, const void* preact, const int* offsets, size_t groups, size_t M,
                                    size_t N, size_t K, int layout_b, int activation, int accumulate, void* stream)
{
    return with_status([&] {
        layer p{type_idx, M, N, K, layout_b, offsets, groups, {}};
        const int rc = check_layer(p);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(!activation_of(activation, &p.act) || (groups != 0 && offsets == nullptr))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return backward(p, dA, dB, dbias, dC, A, B, preact, accumulate, stream_of(stream));
    });
}

int rocm_wmma_gemm_linear(int type_idx, void* C, const void* A, const void* B, size_t M, size_t N, size_t K,
                          int layout_b, const rocm_wmma_gemm_epilogue* epilogue, void* stream)
{
    return with_status([&] {
        const rocm_wmma_gemm_epilogue none{};
        const rocm_wmma_gemm_epilogue& e = epilogue ? *epilogue : none;
        layer p{type_idx, M, N, K, layout_b, nullptr, 1, {}};
        const int rc = check_layer(p);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(!activation_of(e.activation, &p.act))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return forward(p, C, A, B, e, stream_of(stream));
    });
}

int rocm_wmma_gemm_linear_backward(int type_idx, void* dA, void* dB, void* dbias, const void* dC, const void* A,
                                   const void* B, const void* preact, size_t M, size_t N, size_t K, int layout_b,
                                   int activation, int accumulate, void* stream)
{
    return with_status([&] {
        layer p{type_idx, M, N, K, layout_b, nullptr, 1, {}};
        const int rc = check_layer(p);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(!activation_of(activation, &p.act))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return backward(p, dA, dB, dbias, dC, A, B, preact, accumulate, stream_of(stream));
    });
}

int rocm_wmma_gemm_orthogonalize(int given_type, int out_type, void* O, const void* G, size_t M, size_t N,
                                 size_t batch_count, int steps, const float* coefficients, float epsilon, void* stream)
{
    return with_status([&] {
        if(given_type < ROCM_WMMA_GEMM_ELEMENT_F16 || given_type > ROCM_WMMA_GEMM_ELEMENT_F32
           || (out_type != ROCM_WMMA_GEMM_ELEMENT_F16 && out_type != ROCM_WMMA_GEMM_ELEMENT_BF16) || steps < 1
           || coefficients == nullptr)
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        if(M == 0 || N == 0 || batch_count == 0)
        {
            return ROCM_WMMA_GEMM_OK;
        }
        if(O == nullptr || G == nullptr)
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        if(M > (1u << 20) || N > (1u << 20) || batch_count > 65535)
        {
            return ROCM_WMMA_GEMM_ERR_LIMIT;
        }
        return orthogonalize(given_type, out_type, O, G, M, N, batch_count, steps, coefficients, epsilon,
                             stream_of(stream));
    });
}

} // extern "C"
