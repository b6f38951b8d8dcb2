// Host side of the operators next to the GEMM: a linear layer with its epilogue, the same for
// groups of rows (experts), their backward passes, and Newton-Schulz steps on an update.  They
// are additions with no counterpart in the reference.
#include <rocm_wmma_gemm_c.h>

#include <cmath>

#include "kernel/product_pointwise.hpp"
#include "product_host.hpp"

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
        default: return {nullptr, 0, 0, 0, nullptr, nullptr, 0};
    }
}

namespace
{
using device::act_args;
using device::act_kind;
using device::product_args;
using device::product_kind;

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

// Which operands have rows (and groups) that all start on 16 bytes, as the kernels need them that
// load 16 bytes at a time, straight to LDS, or store pieces of 16.
struct starts_on_16
{
    bool a, b, c;
};

starts_on_16 alignment_of(const product_args& x)
{
    return {x.lda % 8 == 0 && x.stride_a % 8 == 0 && aligned16(x.A), x.ldb % 8 == 0 && x.stride_b % 8 == 0 && aligned16(x.B),
            x.ldc % 8 == 0 && (x.N % 8 == 0 || x.padded_c) && x.stride_c % 8 == 0 && aligned16(x.C) && aligned16(x.kept)
                && aligned16(x.residual) && aligned16(x.bias)};
}

// An operand as a matrix of contiguous rows, groups one after the other.
struct matrix_of_rows
{
    size_t rows, length;
    size_t padded() const
    {
        return round_up8(length);
    }
    size_t bytes() const
    {
        return whole_lines(rows * padded() * 2);
    }
};

matrix_of_rows rows_of_a(const product_args& x, int layout)
{
    // (rows and sum: A's rows are those of all groups)
    return layout == layout_mn ? matrix_of_rows{size_t(x.K), size_t(x.M)} : matrix_of_rows{size_t(x.M), size_t(x.K)};
}

matrix_of_rows rows_of_b(const product_args& x, int layout)
{
    const size_t groups = x.kind == product_kind::rows ? x.groups : 1;
    return layout == layout_kk ? matrix_of_rows{groups * x.N, size_t(x.K)} : matrix_of_rows{groups * x.K, size_t(x.N)};
}

// The product on copies whose rows are padded with zeros to multiples of 8.  (Where K is no multiple
// of 8 both K-contiguous operands are such copies, or dZ, which is written that way, so that the
// columns past K add zeros.)
product_args on_copies(product_args x, int layout, bool copy_a, bool copy_b, char* at)
{
    if(copy_a)
    {
        x.lda = static_cast<long long>(rows_of_a(x, layout).padded());
        x.A   = at;
        at += at != nullptr ? rows_of_a(x, layout).bytes() : 0;
    }
    if(copy_b)
    {
        const matrix_of_rows m = rows_of_b(x, layout);
        x.ldb                  = static_cast<long long>(m.padded());
        x.stride_b             = static_cast<long long>(m.rows / (x.kind == product_kind::rows ? x.groups : 1) * m.padded());
        x.B                    = at;
    }
    return x;
}

// Tiles of a product: at most (`most`), and about (rows of several groups end inside a tile, half
// full on average).
size_t tiles_of(const product_args& a, size_t bm, size_t bn, bool symmetric, bool most)
{
    const size_t n = ceil_div(a.N, bn);
    if(a.kind == product_kind::rows)
    {
        if(a.groups == 1 && a.offsets == nullptr)
        {
            return ceil_div(a.M, bm) * n;
        }
        const size_t used = std::min<size_t>(a.groups, a.M);
        return (a.M / bm + (most || static_cast<size_t>(a.M) < bm * used ? used : (used + 1) / 2)) * n;
    }
    return a.groups * (symmetric ? n * (n + 1) / 2 : ceil_div(a.M, bm) * n);
}

// What a form costs, in microseconds: a round of tiles takes `fixed` plus, per 64 of K, `alone` where
// few compute units work (and where each has one workgroup of the two it holds) up to `full` where
// all do.  Measured in bf16 over 60 shapes from 1 x 1024 x 1024 to 8192 x 8192 x 1024, in the three pairs of
// operand layouts (tiled: within 15 % of the measured time for all but the smallest; `full` is what
// the clock under the power limit leaves).
struct form_cost
{
    int   form;
    float fixed, alone, full;
    float stream; // bytes per us at which a weight comes from memory that no cache holds
};
constexpr form_cost tiled_costs[] = {
    {form_tiled_256, 9.0f, 1.10f, 1.45f, 2.3e6f},
    {form_tiled_128x256, 6.0f, 0.64f, 0.85f, 3.5e6f},
    {form_tiled_128, 4.5f, 0.64f, 1.0f, 2.9e6f},
    {form_tiled_192, 8.0f, 0.70f, 0.90f, 2.9e6f},
};
constexpr form_cost narrow_cost = {form_narrow_128, 6.0f, 0.64f, 1.0f, 2.9e6f};
// (finish_back's, 128 x 256 with pieces that start anywhere; on 256 x 256 the two ways to end a tile spill)
constexpr form_cost narrow_back_cost = {form_narrow_128, 7.0f, 0.64f, 0.85f, 3.5e6f};
// The general kernel, by layout: FLOP per us where there is enough to do (it gathers operands that are contiguous
// along M or N two bytes at a time), and us per 64 of K of a tile on its own.
constexpr float general_flops[num_product_layouts] = {2.0e8f, 8.5e7f, 6.5e7f};
constexpr float general_k64 = 1.5f;
constexpr float copy_bytes_per_us = 4.2e6f; // read and written by the copies
// (both operands K-contiguous)
constexpr form_cost skinny_costs_kk[] = {
    {form_skinny_16x32, 3.5f, 0.09f, 0.20f, 5.2e6f},  {form_skinny_32x16, 3.5f, 0.085f, 0.20f, 5.2e6f},
    {form_skinny_32x32, 3.5f, 0.11f, 0.25f, 5.2e6f},  {form_skinny_64x32, 4.0f, 0.16f, 0.29f, 4.5e6f},
    {form_skinny_64x64, 4.5f, 0.24f, 0.25f, 4.0e6f},
};
// (B contiguous along N: a k row of 32 columns is half a cache line)
constexpr form_cost skinny_costs_kn[] = {
    {form_skinny_16x32, 3.5f, 0.15f, 0.24f, 3.2e6f}, {form_skinny_16x64, 4.0f, 0.15f, 0.26f, 4.5e6f},
    {form_skinny_32x32, 3.5f, 0.16f, 0.24f, 3.0e6f}, {form_skinny_32x64, 4.0f, 0.19f, 0.30f, 4.2e6f},
    {form_skinny_64x32, 4.0f, 0.21f, 0.34f, 2.8e6f}, {form_skinny_64x64, 4.5f, 0.25f, 0.28f, 4.0e6f},
};
// What the end of a tile of a Newton-Schulz step takes beyond a layer's, in us per 128 x 128 elements: it is
// written twice, or reads and writes fp32.  (Against none over 19 sizes from 192 x 3328 to 4096 x 4096: 0.98 of
// their time, 11 x 320 x 768 206 -> 178 us, 1336 x 1064 313 -> 268, none slower by more than 1 %.)
constexpr float steps_finish_us(int finish)
{
    return finish == finish_square                              ? 2.5f
           : finish == finish_poly                              ? 5.0f
           : finish == finish_next || finish == finish_last ? 3.0f
                                                                : 0.0f;
}
constexpr float bytes_per_us = 4.5e6f; // of partial tiles, written and read once each
constexpr float join_us      = 9.0f; // the scratch buffer's lease and a second launch, or the exchange in one
// A weight of this many bytes is not in the 256 MB memory-side cache when it is read again, behind
// the others of its model; non-temporal loads then stream 6..15 % faster (16 x 8192 x 8192: 25.6 -> 23.4 us,
// 16 x 8192 x 28672 79 -> 71), but lose what that cache holds of smaller ones (64 x 4096 x 4096: 10.9 -> 14.0).
constexpr size_t once_bytes = size_t{96} << 20;

// One round's time on `tiles` workgroups of a form.
float round_us(const form_cost& f, size_t tiles, size_t cus, int per_cu, float k64)
{
    const float busy = per_cu > 1 ? (tiles > cus ? std::min(1.0f, float(tiles - cus) / cus * 2.0f) : 0.0f)
                                  : std::min(1.0f, float(tiles) / cus);
    return f.fixed + k64 * (f.alone + (f.full - f.alone) * busy);
}

} // namespace

launch_choice choose(int types, int layout, int finish, const product_args& given, size_t cus)
{
    const bool         logits    = finish == finish_parts || finish == finish_slope; // (whole tiles)
    const bool         symmetric = finish == finish_square || finish == finish_poly;
    const starts_on_16 aligned   = alignment_of(given);
    const bool         copy_a = !aligned.a, copy_b = !aligned.b;
    const product_args args = on_copies(given, layout, copy_a, copy_b, nullptr);
    const matrix_of_rows am = rows_of_a(given, layout), bm = rows_of_b(given, layout);
    auto                 made = [&](int form) {
        launch_choice c;
        c.layout = layout;
        c.form   = form;
        if(form != form_general_64 && form != form_general_128)
        {
            c.copy_a     = copy_a;
            c.copy_b     = copy_b;
            c.copy_bytes = (copy_a ? am.bytes() : 0) + (copy_b ? bm.bytes() : 0);
        }
        c.kernel = find_product(types, layout, form, finish);
        if(c.kernel.fn != nullptr)
        {
            // (the few-row kernel computes all of a symmetric product)
            c.items      = tiles_of(args, c.kernel.block_m, c.kernel.block_n, symmetric && c.kernel.per_cu != 0, true);
            c.workgroups = c.kernel.per_cu == 0 ? c.items : std::min(c.items, c.kernel.per_cu * cus);
        }
        return c;
    };
    auto with_cut = [&](launch_choice c) {
        const size_t all = c.kernel.per_cu * cus, tile_bytes = size_t{4} * c.kernel.block_m * c.kernel.block_n;
        c.workgroups    = all;
        c.partial_bytes = all * tile_bytes;
        return c;
    };
    const size_t stages      = ceil_div(args.K, 128); // of the few-row kernel
    auto         with_slices = [&](launch_choice c, size_t slices) {
        // (every slice has a stage, and the counters have a place for every tile)
        slices = std::max<size_t>(1, std::min(slices, stages));
        slices = ceil_div(stages, ceil_div(stages, slices));
        if(c.kernel.per_cu == 0 && slices > 1 && c.items <= stream_arrival_slots)
        {
            c.k_slices      = static_cast<int>(slices);
            c.partial_bytes = c.items * slices * c.kernel.block_m * c.kernel.block_n * 4;
        }
        return c;
    };
    const int general = tiles_of(args, 128, 128, false, true) < cus ? form_general_64 : form_general_128;
    if(args.K == 0 || std::max({args.lda, args.ldb, args.ldc}) >= (1 << 21))
    {
        // (no K tile to load; or a tile's span beyond the 31 bits of the other kernels' offsets)
        return made(general);
    }
    launch_choice best;
    float         least = 1e30f;
    auto          offer = [&](const launch_choice& c, float us) {
        if(us < least)
        {
            least = us;
            best  = c;
        }
    };
    const bool  several = args.kind == product_kind::sum && args.groups > 1; // sums of different lengths
    const bool  rows_kind = args.kind == product_kind::rows;
    // (rows: a group's weight is read if it has a row)
    const size_t used   = rows_kind ? std::min<size_t>(args.groups, args.M) : args.groups;
    const float  weight = rows_kind ? float(used) * args.N * args.K * 2 : 0.0f;
    const float k64     = std::max(1.0f, (several ? float(args.K) / args.groups : float(args.K)) / 64.0f);
    const float copies = copy_a || copy_b ? 3.0f + 2.0f * ((copy_a ? am.bytes() : 0) + (copy_b ? bm.bytes() : 0)) / copy_bytes_per_us
                                          : 0.0f;
    if(copy_a || copy_b)
    {
        // (the copies pay against a large product only: a few rows read a weight as it is)
        const float flops = 2.0f * tiles_of(args, 64, 64, false, false) * 4096 * k64 * 64;
        offer(made(general), 5.0f + std::max(flops / general_flops[layout], k64 * general_k64));
    }
    auto consider_tiled = [&](form_cost f) {
        const launch_choice c = made(f.form);
        if(c.kernel.fn == nullptr)
        {
            return;
        }
        f.fixed += steps_finish_us(finish) * c.kernel.block_m * c.kernel.block_n / (128 * 128);
        const size_t tiles = tiles_of(args, c.kernel.block_m, c.kernel.block_n, symmetric, false);
        const size_t slots = c.kernel.per_cu * cus, rounds = tiles / slots, rest = tiles % slots;
        const float  whole = rounds * round_us(f, slots, cus, c.kernel.per_cu, k64), least_us = weight / f.stream;
        offer(c, copies + std::max(least_us, whole + (rest ? round_us(f, rest, cus, c.kernel.per_cu, k64) : 0.0f)));
        const device::tail_cut cut = device::cut_tail(static_cast<int>(tiles), static_cast<int>(slots),
                                                      static_cast<int>(std::ceil(k64)), !several && c.kernel.finish != nullptr);
        if(cut.cut != 0)
        {
            const size_t parts = size_t(cut.cut) * cut.slices;
            offer(with_cut(c), copies + std::max(least_us, whole + round_us(f, parts, cus, c.kernel.per_cu, float(cut.each))) + join_us
                                   + 2.0f * parts * 4 * c.kernel.block_m * c.kernel.block_n / bytes_per_us);
        }
    };
    if(aligned.c)
    {
        for(const form_cost& f : tiled_costs)
        {
            consider_tiled(f);
        }
    }
    else
    {
        consider_tiled(finish == finish_back ? narrow_back_cost : narrow_cost);
    }
    // (the few-row kernel's offsets within a weight that is contiguous along N have 31 bits)
    const bool batch = args.kind == product_kind::batch;
    if((rows_kind || batch) && (layout == layout_kk || static_cast<long long>(args.K) * args.ldb < (1ll << 30)))
    {
        const size_t rows = batch ? args.M : ceil_div(args.M, used);
        auto         consider = [&](const form_cost& f) {
            launch_choice c = made(f.form);
            if(c.kernel.fn == nullptr || c.items * c.kernel.threads > most_threads_x)
            {
                return;
            }
            const size_t tiles = tiles_of(args, c.kernel.block_m, c.kernel.block_n, false, false);
            const int    per_cu = f.form == form_skinny_64x64 ? 1 : 2;
            const size_t slots = per_cu * cus;
            const bool   one_high = rows <= static_cast<size_t>(c.kernel.block_m);
            c.once                = one_high && weight >= once_bytes;
            for(const size_t slices : {1, 2, 4})
            {
                const launch_choice s = slices == 1 ? c : with_slices(c, slices);
                if(slices > 1 && (batch || logits || s.k_slices == 1 || tiles * slices > slots))
                {
                    continue;
                }
                const size_t workgroups = tiles * s.k_slices, rounds = workgroups / slots, rest = workgroups % slots;
                const float  k = k64 / s.k_slices;
                float us = rounds * round_us(f, slots, cus, per_cu, k) + (rest ? round_us(f, rest, cus, per_cu, k) : 0.0f);
                // (row tiles that share a weight do not all find it in L2)
                us = std::max(us, weight / (one_high ? f.stream : 0.65f * f.stream));
                offer(s, copies + us + (s.k_slices > 1 ? join_us : 0.0f));
            }
        };
        if(layout == layout_kk)
        {
            for(const form_cost& f : skinny_costs_kk)
            {
                consider(f);
            }
        }
        else
        {
            for(const form_cost& f : skinny_costs_kn)
            {
                consider(f);
            }
        }
    }
    return best;
}

int launch_product(int types, int finish, launch_choice c, product_args args, char* scratch, hipStream_t stream)
{
    if(args.N == 0 || args.M == 0 || args.groups == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if(c.copy_bytes != 0 && scratch == nullptr)
    {
        c.kernel     = find_product(types, c.layout, form_general_128, finish);
        c.copy_bytes = 0;
        c.copy_a = c.copy_b = c.once = false;
        c.items      = tiles_of(args, 128, 128, false, true);
        c.workgroups = std::min(c.items, c.kernel.per_cu * compute_units());
    }
    if(c.kernel.fn == nullptr || c.items > most_extent)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    if(c.copy_bytes != 0)
    {
        const product_args on = on_copies(args, c.layout, c.copy_a, c.copy_b, scratch);
        auto job = [](const matrix_of_rows& m, const void* from, const void* to) {
            return device::pack_job{from, const_cast<void*>(to), static_cast<int>(m.rows), static_cast<int>(m.length),
                                    static_cast<int>(m.rows), static_cast<int>(m.padded()), 0, 0};
        };
        const matrix_of_rows   am = rows_of_a(args, c.layout), bm = rows_of_b(args, c.layout);
        const device::pack_job ja = job(am, args.A, on.A), jb = job(bm, args.B, on.B);
        const size_t pieces = std::max(c.copy_a ? am.rows * am.padded() / 8 : 0, c.copy_b ? bm.rows * bm.padded() / 8 : 0);
        follow(&device::pack_padded<unsigned short>,
               dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(pieces, 256), 8192)), c.copy_a && c.copy_b ? 2 : 1),
               dim3(256), stream, c.copy_a ? ja : jb, c.copy_b ? jb : ja);
        args = on;
        scratch += c.copy_bytes;
    }
    if(args.offsets == nullptr && args.kind != product_kind::batch)
    {
        // (one group of all rows: nothing to look up, 1 us less of a small call)
        args.kind     = product_kind::batch;
        args.stride_a = args.stride_b = args.stride_c = 0;
    }
    const bool cuts = c.partial_bytes != 0 && scratch != nullptr;
    args.grid_m     = static_cast<int>(ceil_div(args.M, c.kernel.block_m));
    args.grid_n     = static_cast<int>(ceil_div(args.N, c.kernel.block_n));
    args.partials   = cuts ? reinterpret_cast<float*>(scratch) : nullptr;
    args.workgroups = static_cast<int>(c.workgroups);
    args.k_slices   = 1;
    args.wide       = alignment_of(args).c;
    if(cuts && c.k_slices > 1)
    {
        args.arrivals = arrivals_of_current_device(false);
        if(args.arrivals == nullptr)
        {
            return ROCM_WMMA_GEMM_ERR_RUNTIME;
        }
        args.arrival_epoch = next_arrival_epoch();
        args.k_slices      = c.k_slices;
    }
    follow(c.once && c.kernel.once != nullptr ? c.kernel.once : c.kernel.fn,
           dim3(static_cast<unsigned>(c.workgroups * args.k_slices)), dim3(c.kernel.threads), stream, args);
    if(cuts && c.kernel.finish != nullptr)
    {
        follow(c.kernel.finish, dim3(static_cast<unsigned>(std::min<size_t>(2048, c.workgroups * 8))),
               dim3(c.kernel.threads), stream, args);
    }
    return ROCM_WMMA_GEMM_OK;
}

namespace
{

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

// The three products of a layer, without their pointers.
struct layer_product
{
    product_args args;
    int          layout, finish;
};

layer_product forward_product(const layer& p, bool extras)
{
    product_args a = arguments(p);
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
    return {a, p.layout_b == 1 ? layout_kk : layout_kn,
            p.act.kind == act_kind::logistic           ? finish_logistic
            : p.act.kind == act_kind::relu || extras ? finish_layer
                                                       : finish_plain};
}

// dA = dZ B^T; pitch: dZ's row length
layer_product gradient_a(const layer& p, size_t pitch)
{
    product_args a = arguments(p);
    a.kind         = product_kind::rows;
    a.M            = static_cast<int>(p.M);
    a.N            = static_cast<int>(p.K);
    a.K            = static_cast<int>(p.N);
    a.lda          = pitch;
    a.ldb          = p.layout_b == 1 ? p.K : p.N;
    a.ldc          = p.K;
    a.stride_b     = static_cast<long long>(p.N * p.K);
    return {a, p.layout_b == 1 ? layout_kn : layout_kk, finish_plain};
}

// dB, stored N x K: dZ^T A; stored K x N: A^T dZ
layer_product gradient_b(const layer& p, size_t pitch, bool accumulate)
{
    const bool   nk = p.layout_b == 1;
    product_args a  = arguments(p);
    a.kind          = product_kind::sum;
    a.M             = static_cast<int>(nk ? p.N : p.K);
    a.N             = static_cast<int>(nk ? p.K : p.N);
    a.K             = static_cast<int>(p.M);
    a.lda           = nk ? pitch : p.K;
    a.ldb           = nk ? p.K : pitch;
    a.ldc           = a.N;
    a.stride_c      = static_cast<long long>(p.N * p.K);
    return {a, layout_mn, accumulate ? finish_add : finish_plain};
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
    layer_product f = forward_product(p, e.bias || e.residual || e.preact);
    f.args.C        = C;
    f.args.kept     = e.preact;
    f.args.A        = A;
    f.args.B        = B;
    f.args.bias     = e.bias;
    f.args.residual = e.residual;
    const launch_choice c = choose(p.type_idx, f.layout, f.finish, f.args, compute_units());
    workspace_lease     lease;
    char*               scratch = c.scratch() != 0 ? lease.acquire(c.scratch(), stream) : nullptr;
    return launch_product(p.type_idx, f.finish, c, f.args, scratch, stream);
}

template<class InT>
void launch_slope(device::slope_args s, size_t runs, bool wide, hipStream_t stream)
{
    in_parts(runs, most_groups_x, [&](int run0, unsigned some_runs) {
        in_parts(ceil_div(s.cols, wide ? 512 : 64), most_groups_y, [&](int block0, unsigned some_blocks) {
            s.run0   = run0;
            s.block0 = block0;
            follow(wide ? &device::activation_slope<InT, 8> : &device::activation_slope<InT, 1>, dim3(some_runs, some_blocks),
                   dim3(256), stream, s);
        });
    });
}

template<class OutT>
void launch_column_sums(device::slope_args s, void* dbias, int accumulate, hipStream_t stream)
{
    in_parts(ceil_div(s.cols, 64), most_groups_x, [&](int block0, unsigned some_blocks) {
        s.block0 = block0;
        follow(&device::column_sums<OutT>, dim3(some_blocks, static_cast<unsigned>(s.groups)), dim3(256), stream, s,
               static_cast<OutT*>(dbias), accumulate);
    });
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
    const size_t       cus = compute_units();
    const void*        dz  = dC;
    layer_product      to_a, to_b;
    launch_choice      on_a, on_b;
    device::slope_args s{};
    // dZ and the sums of its columns live in the scratch buffer, and what the products ask for
    // (a dC whose rows do not start on 16 bytes is copied to rows that do, as dZ is written; for the bias alone
    // there is nobody to read either)
    const bool   wants_a = dA != nullptr && p.M != 0 && p.K != 0, wants_b = dB != nullptr && p.N != 0 && p.K != 0;
    const bool   pitched = (wants_a || wants_b) && (sloped || p.N % 8 != 0 || !aligned16(dC));
    const bool   passes  = (pitched || dbias != nullptr) && p.N != 0;
    const size_t pitch   = pitched ? round_up8(p.N) : p.N;
    const size_t runs   = p.M / device::slope_rows + std::min(p.groups, p.M);
    const size_t dz_bytes = passes && pitched ? whole_lines(p.M * pitch * 2) : 0;
    const size_t sums     = passes && dbias != nullptr ? whole_lines(runs * p.N * sizeof(float)) : 0;
    to_a = gradient_a(p, pitch);
    to_b = gradient_b(p, pitch, accumulate != 0);
    // (where the products find dZ is not known yet; the buffer is aligned for any kernel)
    auto placed = [&](const void* at) {
        to_a.args.A                                   = at;
        (p.layout_b == 1 ? to_b.args.A : to_b.args.B) = at;
    };
    to_a.args.C        = dA;
    to_a.args.B        = B;
    to_b.args.C        = dB;
    to_b.args.residual = accumulate ? dB : nullptr;
    (p.layout_b == 1 ? to_b.args.B : to_b.args.A) = A;
    placed(dz_bytes != 0 ? nullptr : dC);
    if(wants_a)
    {
        on_a = choose(p.type_idx, to_a.layout, to_a.finish, to_a.args, cus);
    }
    if(wants_b)
    {
        on_b = choose(p.type_idx, to_b.layout, to_b.finish, to_b.args, cus);
    }
    workspace_lease lease;
    const size_t    needed = dz_bytes + sums, cuts = std::max(on_a.scratch(), on_b.scratch());
    char*           ws = needed + cuts != 0 ? lease.acquire(needed + cuts, stream) : nullptr;
    char*           scratch = ws != nullptr && cuts != 0 ? ws + needed : nullptr;
    if(ws == nullptr && needed != 0)
    {
        // (a capture forbids to allocate: perhaps there is room without cut tiles and copies)
        ws = cuts != 0 ? lease.acquire(needed, stream) : nullptr;
        if(ws == nullptr)
        {
            return ROCM_WMMA_GEMM_ERR_SCRATCH;
        }
    }
    if(passes)
    {
        s.dc      = dC;
        s.z       = sloped ? preact : nullptr;
        s.dz      = pitched ? ws : nullptr;
        s.dz_pitch = static_cast<int>(pitch);
        s.sums    = dbias != nullptr ? reinterpret_cast<float*>(ws + dz_bytes) : nullptr;
        s.offsets = p.offsets;
        s.groups  = static_cast<int>(p.groups);
        s.rows    = static_cast<int>(p.M);
        s.cols    = static_cast<int>(p.N);
        s.act     = p.act;
        if(runs != 0)
        {
            const bool wide = p.N % 8 == 0 && aligned16(dC) && (!sloped || aligned16(preact));
            is_bf16(p.type_idx) ? launch_slope<__bf16>(s, runs, wide, stream)
                                : launch_slope<_Float16>(s, runs, wide, stream);
        }
        dz = pitched ? ws : dC;
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
    placed(dz);
    int rc = ROCM_WMMA_GEMM_OK;
    if(on_a.kernel.fn != nullptr)
    {
        rc = launch_product(p.type_idx, to_a.finish, on_a, to_a.args, on_a.scratch() != 0 ? scratch : nullptr, stream);
    }
    if(rc == ROCM_WMMA_GEMM_OK && on_b.kernel.fn != nullptr)
    {
        rc = launch_product(p.type_idx, to_b.finish, on_b, to_b.args, on_b.scratch() != 0 ? scratch : nullptr, stream);
    }
    return rc;
}

struct update
{
    int          given_type, out_type;
    void*        O;
    const void*  G;
    size_t       M, N, batch;
    int          steps;
    const float* coefficients;
    float        epsilon;
    hipStream_t  stream;
};

// The scratch memory of an update's matrices, `batch` of them: where each part starts, and its end.
struct steps_scratch
{
    size_t l, h, lp, hp, each, square; // smaller and larger side, padded to multiples of 8; elements of X and S
    size_t diagonal, x32, x16, x16_bytes, s, q, bytes; // (the partial sums of squares come first)
    steps_scratch(size_t M, size_t N, size_t batch)
        : l(std::min(M, N)), h(std::max(M, N)), lp(round_up8(l)), hp(round_up8(h)), each(lp * hp), square(lp * lp)
    {
        diagonal  = whole_lines(batch * device::square_parts * sizeof(double));
        x32       = diagonal + whole_lines(batch * lp * sizeof(float));
        x16       = x32 + whole_lines(batch * each * 4);
        x16_bytes = whole_lines(batch * each * 2);
        s         = x16 + 2 * x16_bytes;
        q         = s + whole_lines(batch * square * 2);
        bytes     = q + whole_lines(batch * square * 2);
    }
};

// The products of a step, without their pointers and factors: S = X X^T, Q = b S + c S^2, X = (a + diagonal) X + Q X.
enum class step_part
{
    square,
    poly,
    next,
    last
};

struct step_product
{
    product_args args;
    int          types, layout, finish;
};

step_product product_of_step(step_part part, int out_type, const steps_scratch& at, size_t batch)
{
    product_args p{};
    p.kind            = product_kind::batch;
    p.groups          = static_cast<int>(batch);
    p.stride_diagonal = static_cast<long long>(at.lp);
    p.M               = static_cast<int>(at.lp);
    if(part == step_part::square || part == step_part::poly)
    {
        const bool of_x = part == step_part::square;
        p.N             = p.M;
        p.K             = static_cast<int>(of_x ? at.hp : at.lp);
        p.lda = p.ldb = p.K, p.ldc = at.lp;
        p.stride_a = p.stride_b = static_cast<long long>(of_x ? at.each : at.square);
        p.stride_c              = static_cast<long long>(at.square);
        p.diagonal_is           = of_x ? device::diagonal_use::none : device::diagonal_use::split;
        return {p, types_steps_square, layout_kk, of_x ? finish_square : finish_poly};
    }
    p.N = static_cast<int>(at.hp), p.K = static_cast<int>(at.lp);
    p.lda = at.lp, p.ldb = p.ldc = at.hp;
    p.stride_a = static_cast<long long>(at.square);
    p.stride_b = p.stride_c = static_cast<long long>(at.each);
    p.diagonal_is           = device::diagonal_use::rows;
    if(part == step_part::next)
    {
        return {p, types_steps_next, layout_kn, finish_next};
    }
    return {p, out_type == ROCM_WMMA_GEMM_ELEMENT_F16 ? types_steps_f16 : types_steps_bf16, layout_kn, finish_last};
}

constexpr size_t most_update = size_t{1} << 20, most_updates = most_groups_y; // sides of a matrix, matrices

// How many of a batch's matrices work at the same time: those whose state the scratch buffer may hold, in parts of
// equal size.
size_t updates_at_once(size_t M, size_t N, size_t batch)
{
    const size_t fit = std::max<size_t>(1, workspace_limit_bytes / steps_scratch(M, N, 1).bytes);
    return ceil_div(batch, ceil_div(batch, fit));
}

bool fits_one_workgroup(size_t M, size_t N)
{
    return std::min(M, N) <= device::small_side && std::max(M, N) <= device::small_length;
}

// Newton-Schulz steps X <- a X + (b S + c S^2) X with S = X X^T on X = G / (|G| + epsilon), or on its
// transpose where G is tall.
//
// What is rounded, and why: products of matrices past small_side x small_length take f16 operands.  With the
// coefficients that are the Python default every singular value of X stays below 1.3, so f16 holds X (scaled by
// about the root of its smaller side, a power of two, which keeps its elements near 1), S and Q = b S + c S^2
// with 11 bits; bf16 would leave 8.  Coefficients whose iterates grow are right as long as f16 holds those three:
// |b| s^2 + |c| s^4 and s times twice the root of the smaller side below 65504 for the largest singular value s of an
// iterate.  Past it Q or X turns infinite, and the update is no number.  Two terms are kept from the rounding,
// because it is the largest part of the error there:
//   - a X: small singular directions grow 3.4 times a step, and a rounding of the large ones
//     (white noise in all directions) with them, so X is also kept in fp32 and only the products
//     see the f16 copy;
//   - Q's diagonal: near the end Q is about -2.7 I, and rounding that moves whole rows of X by
//     four times as much.  The diagonal stays in fp32 beside Q, whose own is zero, and meets the
//     fp32 X in the epilogue: X = (a + diagonal) X + Q X.
// Against 64 bits, an f16 update of 512 x 1024 is 7.8e-4 off for noise and 3.2e-4 for a momentum of 16 strong
// directions, where the rounding of the result leaves 2.1e-4 (simulated for the latter: 2.1e-2 with all of it from
// f16, 1.6e-1 from bf16); 1 x 300: 3.7e-4.
int steps_in(char* ws, const update& u)
{
    const size_t        M = u.M, N = u.N, batch = u.batch;
    const steps_scratch at(M, N, batch);
    const size_t        l = at.l, h = at.h, lp = at.lp, hp = at.hp, each = at.each, square = at.square;
    const int           given_type = u.given_type, out_type = u.out_type, steps = u.steps;
    const void*         G = u.G;
    void*               O = u.O;
    const float*        coefficients = u.coefficients;
    const float         epsilon = u.epsilon;
    const hipStream_t   stream = u.stream;
    const bool          tall   = M > N;
    const bool          direct = !tall && lp == l && hp == h && aligned16(O);
    double*   parts    = reinterpret_cast<double*>(ws);
    float*    diagonal = reinterpret_cast<float*>(ws + at.diagonal);
    float*    x32      = reinterpret_cast<float*>(ws + at.x32);
    _Float16* x16[2]   = {reinterpret_cast<_Float16*>(ws + at.x16), reinterpret_cast<_Float16*>(ws + at.x16 + at.x16_bytes)};
    char*     s        = ws + at.s;
    char*     q        = ws + at.q;
    const float scale = std::exp2(std::round(std::log2(std::sqrt(static_cast<float>(l)))));
    const unsigned nb = static_cast<unsigned>(batch);

    auto start = [&](auto* typed) {
        using given_t = std::remove_pointer_t<decltype(typed)>;
        const given_t* given = static_cast<const given_t*>(G);
        constexpr int  wide   = 16 / sizeof(given_t);
        const bool     vector = M * N % wide == 0 && aligned16(given);
        // (a workgroup for every 4096 pieces, but at most eight to a compute unit over the batch)
        const size_t used = std::max<size_t>(
            1, std::min({ceil_div(M * N / (vector ? wide : 1), 4096), size_t{device::square_parts}, ceil_div(2048, batch)}));
        follow(vector ? &device::sum_squares<given_t, wide> : &device::sum_squares<given_t, 1>,
               dim3(static_cast<unsigned>(used), nb), dim3(256), stream, given, static_cast<long long>(M * N), parts);
        const device::start_args args{given, parts, x32, x16[0], static_cast<int>(M), static_cast<int>(N),
                                      static_cast<int>(lp), static_cast<int>(hp), scale, epsilon, static_cast<int>(used)};
        if(tall)
        {
            follow(&device::orthogonal_start_tall<given_t>,
                   dim3(static_cast<unsigned>(ceil_div(lp, 64) * ceil_div(hp, 64)), nb), dim3(256), stream, args);
            return;
        }
        follow(lp == l && hp == h && aligned16(given) ? &device::orthogonal_start<given_t, true>
                                                      : &device::orthogonal_start<given_t, false>,
               dim3(static_cast<unsigned>(std::min<size_t>(lp, std::max<size_t>(1, 2048 / batch))), nb), dim3(256), stream,
               args);
    };
    by_element(given_type, start);
    const float a = coefficients[0], b = coefficients[1], c = coefficients[2];
    const size_t cus = compute_units();
    auto         run = [&](const step_product& f) {
        return launch_product(f.types, f.finish, choose(f.types, f.layout, f.finish, f.args, cus), f.args, nullptr, stream);
    };
    auto part = [&](step_part which, void* to, const void* left, const void* right, const void* added, float alpha, float beta) {
        step_product f = product_of_step(which, out_type, at, batch);
        f.args.diagonal = diagonal;
        f.args.C = to, f.args.A = left, f.args.B = right, f.args.residual = added;
        f.args.alpha = alpha, f.args.beta = beta;
        return f;
    };
    int rc = ROCM_WMMA_GEMM_OK;
    for(int step = 0; step < steps && rc == ROCM_WMMA_GEMM_OK; ++step)
    {
        _Float16 * x = x16[step & 1], *next_x = x16[(step + 1) & 1];
        const bool last = step + 1 == steps;
        rc = run(part(step_part::square, s, x, x, nullptr, 1.0f / (scale * scale), 0.0f));
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            break;
        }
        // (S is its own transpose; Q's diagonal apart)
        rc = run(part(step_part::poly, q, s, s, s, c, b));
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            break;
        }
        if(last)
        {
            rc = run(part(step_part::last, direct ? O : static_cast<void*>(next_x), q, x, x32, 1.0f / scale, a / scale));
            break;
        }
        step_product f  = part(step_part::next, x32, q, x, x32, 1.0f, a);
        f.args.kept     = next_x;
        f.args.keep_sum = 1;
        rc              = run(f);
    }
    if(rc == ROCM_WMMA_GEMM_OK && !direct)
    {
        // (a 16-bit element is a 16-bit element)
        const unsigned short* padded = reinterpret_cast<const unsigned short*>(x16[steps & 1]);
        follow(tall ? &device::orthogonal_end_tall<unsigned short> : &device::orthogonal_end<unsigned short>,
               dim3(static_cast<unsigned>(tall ? ceil_div(M, 64) * ceil_div(N, 64) : std::min<size_t>(M, 4096)), nb), dim3(256),
               stream, padded, static_cast<unsigned short*>(O), static_cast<int>(M), static_cast<int>(N),
               static_cast<int>(lp), static_cast<int>(hp));
    }
    return rc;
}

int orthogonalize(const update& u)
{
    if(fits_one_workgroup(u.M, u.N))
    {
        const device::steps_args small{u.G, u.O, static_cast<int>(u.M), static_cast<int>(u.N), u.steps, u.coefficients[0],
                                       u.coefficients[1], u.coefficients[2], u.epsilon};
        const bool               f16 = u.out_type == ROCM_WMMA_GEMM_ELEMENT_F16;
        auto run = [&](auto* typed) {
            using given_t = std::remove_pointer_t<decltype(typed)>;
            follow(f16 ? &device::orthogonal_small<given_t, _Float16> : &device::orthogonal_small<given_t, __bf16>,
                   dim3(static_cast<unsigned>(u.batch)), dim3(1024), u.stream, small);
        };
        by_element(u.given_type, run);
        return ROCM_WMMA_GEMM_OK;
    }
    const size_t    some = updates_at_once(u.M, u.N, u.batch);
    workspace_lease lease;
    char*           ws = lease.acquire(steps_scratch(u.M, u.N, some).bytes, u.stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    const size_t given_bytes = u.given_type == ROCM_WMMA_GEMM_ELEMENT_F32 ? 4 : 2;
    int          rc          = ROCM_WMMA_GEMM_OK;
    for(size_t first = 0; first < u.batch && rc == ROCM_WMMA_GEMM_OK; first += some)
    {
        update part = u;
        part.batch  = std::min(some, u.batch - first);
        part.G      = static_cast<const char*>(u.G) + first * u.M * u.N * given_bytes;
        part.O      = static_cast<char*>(u.O) + first * u.M * u.N * 2;
        rc          = steps_in(ws, part);
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

int rocm_wmma_gemm_product_select(int product, int type_idx, size_t M, size_t N, size_t K, size_t groups, int layout_b,
                                  int activation, rocm_wmma_gemm_product_plan* plan)
{
    return with_status([&] {
        if(plan == nullptr || product < 0 || product > ROCM_WMMA_GEMM_PRODUCT_STEPS_LAST)
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        const auto answer = [&](const launch_choice& c) {
            plan->form     = c.form;
            plan->block_m  = c.kernel.block_m;
            plan->block_n  = c.kernel.block_n;
            plan->cut_tail = c.kernel.finish != nullptr && c.partial_bytes != 0;
            plan->k_slices = c.k_slices;
            plan->once     = c.once;
            plan->copies   = (c.copy_a ? 1 : 0) | (c.copy_b ? 2 : 0);
            return ROCM_WMMA_GEMM_OK;
        };
        if(product >= ROCM_WMMA_GEMM_PRODUCT_STEPS_S)
        {
            if(type_idx < 0 || type_idx > ROCM_WMMA_GEMM_TYPE_F32_BF16 || M == 0 || N == 0 || groups == 0)
            {
                return ROCM_WMMA_GEMM_ERR_ARGUMENT;
            }
            if(M > most_update || N > most_update || groups > most_updates)
            {
                return ROCM_WMMA_GEMM_ERR_LIMIT;
            }
            if(fits_one_workgroup(M, N))
            {
                *plan = {num_product_forms, rocm_wmma_gemm::device::small_side, rocm_wmma_gemm::device::small_length, 0, 1, 0, 0};
                return ROCM_WMMA_GEMM_OK;
            }
            const size_t       some = updates_at_once(M, N, groups);
            const step_product f = product_of_step(static_cast<step_part>(product - ROCM_WMMA_GEMM_PRODUCT_STEPS_S),
                                                   is_bf16(type_idx) ? ROCM_WMMA_GEMM_ELEMENT_BF16 : ROCM_WMMA_GEMM_ELEMENT_F16,
                                                   steps_scratch(M, N, some), some);
            return answer(choose(f.types, f.layout, f.finish, f.args, compute_units()));
        }
        // (offsets that nobody reads: groups of rows are told by their presence)
        static const int somewhere = 0;
        layer            p{type_idx, M, N, K, layout_b, groups != 0 ? &somewhere : nullptr, groups != 0 ? groups : 1, {}};
        const int        rc = check_layer(p);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(!activation_of(activation, &p.act) || M == 0 || N == 0)
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        // dZ is written to rows that start on 16 bytes where dC's do not
        const size_t        pitch = round_up8(p.N);
        const layer_product f     = product == ROCM_WMMA_GEMM_PRODUCT_FORWARD      ? forward_product(p, true)
                                    : product == ROCM_WMMA_GEMM_PRODUCT_GRADIENT_A ? gradient_a(p, pitch)
                                                                                   : gradient_b(p, pitch, false);
        if(f.args.M == 0 || f.args.N == 0)
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        return answer(choose(p.type_idx, f.layout, f.finish, f.args, compute_units()));
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
        if(M > most_update || N > most_update || batch_count > most_updates)
        {
            return ROCM_WMMA_GEMM_ERR_LIMIT;
        }
        return orthogonalize({given_type, out_type, O, G, M, N, batch_count, steps, coefficients, epsilon, stream_of(stream)});
    });
}

} // extern "C"
