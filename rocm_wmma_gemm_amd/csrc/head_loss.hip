// Host side of a projection onto a vocabulary with its loss: cross entropy against a target, distillation from a
// teacher's listed logits, and their gradients, in pieces of the vocabulary, so that the logits of all of it are never
// kept.  They are additions with no counterpart in the reference.
#include <cmath>

#include "kernel/head_loss.hpp"
#include "product_host.hpp"

namespace rocm_wmma_gemm
{
namespace host
{
namespace
{
using device::product_args;
using device::product_kind;
using device::wanted_args;

constexpr size_t most_rows = size_t{1} << 20; // (a piece of 1024 columns of them fits the scratch buffer)

// A piece of the logits in fp32 is read back from the memory-side cache where it is not larger than this.
constexpr size_t piece_bytes = size_t{128} << 20;
constexpr size_t least_piece = 1024, piece_grain = 256; // columns

// An operand's rows in memory.
struct operand
{
    const void* at;
    size_t      ld;
};

// The problem: states A (M x K), weights B (K x N), what the rows are compared with.
struct head
{
    int         in; // element of A and B
    size_t      M, N, K;
    int         layout_b;
    const void* A;
    const void* B;
    wanted_args want;
    bool        bf16() const
    {
        return in == ROCM_WMMA_GEMM_ELEMENT_BF16;
    }
    // the product's types for C of fp32, and of 16 bits
    int to_f32() const
    {
        return bf16() ? types_f32_bf16 : types_f32_f16;
    }
    int to_16() const
    {
        return bf16() ? types_bf16_bf16 : types_f16_f16;
    }
    size_t b_rows() const
    {
        return layout_b == 1 ? N : K;
    }
    size_t b_length() const
    {
        return layout_b == 1 ? K : N;
    }
};

// Places in the scratch buffer, handed out one after the other.
struct room
{
    size_t bytes = 0;
    size_t take(size_t n)
    {
        const size_t at = bytes;
        bytes += whole_lines(n);
        return at;
    }
};

// Copies of the operands whose rows do not start on 16 bytes, where all of a call's products read them: A always (it is
// small next to the products), B where there are enough rows to pay for reading and writing it, and where pieces of its
// columns would have to be copied out of longer rows.
struct copies
{
    bool   a, b;
    size_t a_at = 0, b_at = 0;
    copies(const head& h, size_t pieces, room& r)
        : a(h.M != 0 && h.K != 0 && (h.K % 8 != 0 || !aligned16(h.A))),
          b(h.N != 0 && h.K != 0 && (h.b_length() % 8 != 0 || !aligned16(h.B)) && (h.M >= 256 || (h.layout_b == 0 && pieces > 1)))
    {
        a_at = a ? r.take(h.M * round_up8(h.K) * 2) : 0;
        b_at = b ? r.take(h.b_rows() * round_up8(h.b_length()) * 2) : 0;
    }
    operand run(bool copied, const void* given, size_t rows, size_t length, char* to, hipStream_t stream) const
    {
        if(!copied)
        {
            return {given, length};
        }
        const size_t           padded = round_up8(length);
        const device::pack_job job{given, to, static_cast<int>(rows), static_cast<int>(length), static_cast<int>(rows),
                                   static_cast<int>(padded), 0, 0};
        follow(&device::pack_padded<unsigned short>,
               dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(rows * padded / 8, 256), 8192))), dim3(256), stream, job, job);
        return {to, padded};
    }
    operand run_a(const head& h, char* ws, hipStream_t stream) const
    {
        return run(a, h.A, h.M, h.K, ws + a_at, stream);
    }
    operand run_b(const head& h, char* ws, hipStream_t stream) const
    {
        return run(b, h.B, h.b_rows(), h.b_length(), ws + b_at, stream);
    }
    // the same as run() leaves, before anything is launched (an aligned address stands for the copies)
    operand plan_a(const head& h) const
    {
        return a ? operand{nullptr, round_up8(h.K)} : operand{h.A, h.K};
    }
    operand plan_b(const head& h) const
    {
        return b ? operand{nullptr, round_up8(h.b_length())} : operand{h.B, h.b_length()};
    }
};

// One product, and the kernel that it runs on.
struct step
{
    int          types, layout, finish;
    product_args args;
    launch_choice plan(size_t cus) const
    {
        // (a product without elements is none)
        return args.M == 0 || args.N == 0 ? launch_choice{} : choose(types, layout, finish, args, cus);
    }
    int run(char* scratch, hipStream_t stream) const
    {
        const launch_choice c = plan(compute_units());
        return launch_product(types, finish, c, args, c.scratch() != 0 ? scratch : nullptr, stream);
    }
};

product_args one_problem(product_kind kind, size_t M, size_t N, size_t K)
{
    product_args a{};
    a.kind   = kind;
    a.groups = 1;
    a.alpha = a.beta = 1.0f;
    a.M              = static_cast<int>(M);
    a.N              = static_cast<int>(N);
    a.K              = static_cast<int>(K);
    return a;
}

// The columns v0 .. v0 + cols - 1 of B.
const void* block_of_b(const head& h, const operand& b, size_t v0)
{
    return b.at == nullptr ? nullptr : static_cast<const char*>(b.at) + v0 * (h.layout_b == 1 ? b.ld : 1) * 2;
}

// z = A B for a piece of the vocabulary, in fp32, rows `pitch` apart
step logits_of(const head& h, const operand& a, const operand& b, size_t v0, size_t cols, float* z, size_t pitch)
{
    step s{h.to_f32(), h.layout_b == 1 ? layout_kk : layout_kn, finish_plain, one_problem(product_kind::rows, h.M, cols, h.K)};
    s.args.A      = a.at;
    s.args.B      = block_of_b(h, b, v0);
    s.args.C      = z;
    s.args.lda    = a.ld;
    s.args.ldb    = b.ld;
    s.args.ldc    = pitch;
    s.args.b_skip = h.layout_b == 1 ? 0 : v0;
    s.args.padded_c = 1;
    return s;
}

// dA += dz B^T for a piece: to fp32 rows `pitch` apart, or (whole) to where they belong
step states_of(const head& h, const void* dz, size_t dz_pitch, const operand& b, size_t v0, size_t cols, int types, void* to, size_t pitch,
               bool add)
{
    step s{types, h.layout_b == 1 ? layout_kn : layout_kk, add ? finish_layer : finish_plain,
           one_problem(product_kind::rows, h.M, h.K, cols)};
    s.args.A        = dz;
    s.args.B        = block_of_b(h, b, v0);
    s.args.C        = to;
    s.args.residual = add ? to : nullptr;
    s.args.lda      = dz_pitch;
    s.args.ldb      = b.ld;
    s.args.ldc      = pitch;
    s.args.b_skip   = h.layout_b == 1 ? 0 : v0;
    s.args.padded_c = pitch % 8 == 0 && pitch != h.K;
    return s;
}

// the piece's part of dB, in B's layout: dz^T A, or A^T dz
step weights_of(const head& h, const operand& a, const void* dz, size_t dz_pitch, size_t cols, int types, void* to, size_t pitch, bool add,
                bool padded)
{
    const bool nk = h.layout_b == 1;
    step       s{types, layout_mn, add ? finish_add : finish_plain, one_problem(product_kind::sum, nk ? cols : h.K, nk ? h.K : cols, h.M)};
    s.args.A        = nk ? dz : a.at;
    s.args.B        = nk ? a.at : dz;
    s.args.lda      = nk ? dz_pitch : a.ld;
    s.args.ldb      = nk ? a.ld : dz_pitch;
    s.args.C        = to;
    s.args.residual = add ? to : nullptr;
    s.args.ldc      = pitch;
    s.args.padded_c = padded;
    return s;
}

struct pieces
{
    size_t cols, count;
    pieces(size_t N, size_t wanted)
    {
        cols  = std::max(least_piece, wanted / piece_grain * piece_grain);
        count = std::max<size_t>(1, ceil_div(N, cols));
        // (of one size, as near as the grain lets them)
        cols  = std::min(round_up8(std::max<size_t>(N, 1)), ceil_div(ceil_div(std::max<size_t>(N, 1), count), piece_grain) * piece_grain);
        count = std::max<size_t>(1, ceil_div(N, cols));
    }
    size_t pitch() const
    {
        return round_up8(cols);
    }
};

int check_head(const head& h, bool listed)
{
    if((h.in != ROCM_WMMA_GEMM_ELEMENT_F16 && h.in != ROCM_WMMA_GEMM_ELEMENT_BF16) || (h.layout_b & ~1) || (h.want.wide & ~1)
       || !(h.want.scale > 0.0f) || !std::isfinite(h.want.scale) || !std::isfinite(1.0f / h.want.scale)
       || (listed && h.want.k < 1))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    if(h.M > most_rows || h.N > most_extent || h.K > most_extent || h.want.k > device::most_entries)
    {
        return ROCM_WMMA_GEMM_ERR_LIMIT;
    }
    if((h.M != 0 && h.want.entries == nullptr) || (h.M != 0 && listed && h.want.teacher == nullptr)
       || (h.M != 0 && h.N != 0 && h.K != 0 && (h.A == nullptr || h.B == nullptr)))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    return ROCM_WMMA_GEMM_OK;
}

unsigned row_groups(size_t rows)
{
    return static_cast<unsigned>(std::min<size_t>(ceil_div(rows, 4), 8192));
}

// loss, lse and (a list) the listed logits
int loss_of(const head& h, float* loss, float* lse, float* picked, hipStream_t stream)
{
    if(h.M == 0)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if(loss == nullptr || lse == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    const pieces  p(h.N, piece_bytes / (4 * h.M));
    const size_t  each = ceil_div(p.cols, device::part_cols), all = h.N != 0 ? each * p.count : 0;
    room          r;
    const copies  c(h, p.count, r);
    const operand plan_a = c.plan_a(h), plan_b = c.plan_b(h);
    const size_t  z_at = r.take(h.M * p.pitch() * 4), parts_at = r.take(h.M * all * sizeof(float2)),
                 picked_at = picked == nullptr ? r.take(h.M * sizeof(float)) : 0, product_at = r.bytes;
    size_t product = 0;
    for(size_t v0 = 0; v0 < h.N; v0 += p.cols)
    {
        product = std::max(product, logits_of(h, plan_a, plan_b, v0, std::min(p.cols, h.N - v0), nullptr, p.pitch()).plan(compute_units()).scratch());
        v0 = v0 == 0 && p.count > 2 ? (p.count - 2) * p.cols : v0; // (the first and the last are all there are)
    }
    workspace_lease lease;
    char*           ws = lease.acquire(product_at + product, stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    const operand a = c.run_a(h, ws, stream), b = c.run_b(h, ws, stream);
    float* const  z    = reinterpret_cast<float*>(ws + z_at);
    float* const  of_targets = picked == nullptr ? reinterpret_cast<float*>(ws + picked_at) : picked;
    float2* const parts = reinterpret_cast<float2*>(ws + parts_at);
    const unsigned pick_groups = static_cast<unsigned>(std::min<size_t>(ceil_div(h.M * h.want.k, 256), 4096));
    for(size_t v0 = 0; v0 < std::max<size_t>(h.N, 1); v0 += p.cols)
    {
        const size_t cols = std::min(p.cols, h.N - v0);
        const int    rc   = logits_of(h, a, b, v0, cols, z, p.pitch()).run(ws + product_at, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        follow(&device::pick_entries, dim3(pick_groups), dim3(256), stream, h.want, static_cast<const float*>(z),
               static_cast<long long>(p.pitch()), static_cast<long long>(v0), static_cast<int>(cols), of_targets);
        if(cols != 0)
        {
            // (the last piece may have fewer parts than the others: its rest has none)
            const device::part_args args{z, parts, static_cast<long long>(p.pitch()), static_cast<int>(cols),
                                         static_cast<int>(v0 / p.cols * each), static_cast<int>(all), h.want.scale};
            follow(&device::softmax_parts, dim3(static_cast<unsigned>(h.M), static_cast<unsigned>(each)), dim3(256), stream, args);
        }
    }
    follow(&device::join_rows, dim3(row_groups(h.M)), dim3(256), stream,
           device::join_args{h.want, parts, of_targets, loss, lse, static_cast<int>(all)});
    return ROCM_WMMA_GEMM_OK;
}

template<class InT>
void launch_slope(const device::softmax_slope_args& s, hipStream_t stream)
{
    follow(&device::softmax_slope<InT>, dim3(static_cast<unsigned>(s.want.rows), static_cast<unsigned>(ceil_div(s.pitch, 2048))), dim3(256),
           stream, s);
    if(s.want.teacher != nullptr)
    {
        follow(&device::listed_slope<InT>, dim3(row_groups(s.want.rows)), dim3(256), stream, s);
    }
}

void launch_scaled(int out_type, const float* from, size_t pitch, void* to, size_t to_pitch, size_t rows, size_t cols, const float* unit,
                   bool add, hipStream_t stream)
{
    if(rows == 0 || cols == 0)
    {
        return;
    }
    by_element(out_type, [&](auto* typed) {
        using out_t = std::remove_pointer_t<decltype(typed)>;
        follow(&device::scaled_rows<out_t>, dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(rows * ceil_div(cols, 4), 256), 8192))),
               dim3(256), stream, from, static_cast<long long>(pitch), static_cast<out_t*>(to), static_cast<long long>(to_pitch),
               static_cast<long long>(rows), static_cast<long long>(cols), unit, add ? 1 : 0);
    });
}

// dA and dB (either may be missing) from the loss's gradient by row.
//
// What is rounded, and why: dz = dloss T (p - q) to A's type, as both products need it.  In bf16 it costs 2.4e-3 of a
// gradient's norm where the result's own rounding leaves 1.7e-3.  f16 would lose what lies below 6e-8: there dz is held
// times a power of two that depends on the largest dloss, and the products come out in fp32 and are brought
// back as they are rounded.
int gradients_of(const head& h, int out, void* dA, void* dB, const float* dloss, const float* lse, const float* picked, bool accumulate,
                 hipStream_t stream)
{
    const bool wants_a = dA != nullptr && h.M != 0 && h.K != 0, wants_b = dB != nullptr && h.N != 0 && h.K != 0;
    if(!wants_a && !wants_b)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    if(h.M != 0 && (dloss == nullptr || lse == nullptr))
    {
        return ROCM_WMMA_GEMM_ERR_ARGUMENT;
    }
    const bool   scaled = !h.bf16(), f32 = out == ROCM_WMMA_GEMM_ELEMENT_F32;
    const size_t size = f32 ? 4 : 2, cus = compute_units();
    const int    direct_types = f32 ? h.to_f32() : h.to_16();
    const pieces p(h.N, piece_bytes / (4 * std::max<size_t>(h.M, 1)));
    const size_t pitch = p.pitch(), k_pitch = round_up8(h.K);
    // dA is added up in fp32 over the pieces, in its own place if that is fp32
    const bool own_place = !scaled && h.K % 8 == 0 && aligned16(dA) && (f32 || p.count == 1);
    // where the weights' part of a piece goes in fp32 first: as dB's rows
    const size_t part_rows = h.layout_b == 1 ? p.cols : h.K, part_pitch = h.layout_b == 1 ? k_pitch : pitch;
    room         r;
    const copies c(h, p.count, r);
    const operand plan_a = c.plan_a(h), plan_b = c.plan_b(h);
    const size_t z_at = r.take(h.M * pitch * 4), dz_at = r.take(h.M * pitch * 2), factor_at = r.take(h.M * 4), unit_at = r.take(8),
                 sum_at = wants_a && !own_place ? r.take(h.M * k_pitch * 4) : 0,
                 part_at = wants_b && scaled ? r.take(part_rows * part_pitch * 4) : 0, product_at = r.bytes;
    auto logits = [&](const operand& a, const operand& b, size_t v0, size_t cols, float* z) {
        return logits_of(h, a, b, v0, cols, z, pitch);
    };
    auto states = [&](const operand& b, size_t v0, size_t cols, const void* dz, void* sum) {
        return states_of(h, dz, pitch, b, v0, cols, own_place ? direct_types : h.to_f32(), own_place ? dA : sum, own_place ? h.K : k_pitch,
                         v0 != 0);
    };
    auto weights = [&](const operand& a, size_t v0, size_t cols, const void* dz, void* part) {
        if(scaled)
        {
            return weights_of(h, a, dz, pitch, cols, h.to_f32(), part, part_pitch, false, true);
        }
        void* to = static_cast<char*>(dB) + v0 * (h.layout_b == 1 ? h.K : 1) * size;
        return weights_of(h, a, dz, pitch, cols, direct_types, to, h.b_length(), accumulate, false);
    };
    size_t product = 0;
    for(size_t v0 = 0; v0 < std::max<size_t>(h.N, 1); v0 += p.cols)
    {
        const size_t cols = std::min(p.cols, h.N - v0);
        product = std::max(product, logits(plan_a, plan_b, v0, cols, nullptr).plan(cus).scratch());
        product = std::max(product, wants_a ? states(plan_b, v0, cols, nullptr, nullptr).plan(cus).scratch() : 0);
        product = std::max(product, wants_b ? weights(plan_a, v0, cols, nullptr, nullptr).plan(cus).scratch() : 0);
        v0 = v0 == p.cols && p.count > 3 ? (p.count - 2) * p.cols : v0; // (the first, one behind it, the last)
    }
    workspace_lease lease;
    char*           ws = lease.acquire(product_at + product, stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    const operand a = c.run_a(h, ws, stream), b = c.run_b(h, ws, stream);
    char* const   scratch = ws + product_at;
    float* const  factor  = reinterpret_cast<float*>(ws + factor_at);
    float* const  unit    = reinterpret_cast<float*>(ws + unit_at);
    const device::factor_args f{h.want, dloss, factor, unit, scaled ? 1 : 0};
    if(h.M != 0)
    {
        if(scaled)
        {
            follow(&device::gradient_unit, dim3(1), dim3(1024), stream, f);
        }
        follow(&device::gradient_factors, dim3(row_groups(h.M)), dim3(256), stream, f);
    }
    const float* back = scaled && h.M != 0 ? unit + 1 : nullptr;
    int          rc   = ROCM_WMMA_GEMM_OK;
    for(size_t v0 = 0; v0 < std::max<size_t>(h.N, 1) && rc == ROCM_WMMA_GEMM_OK; v0 += p.cols)
    {
        const size_t cols = std::min(p.cols, h.N - v0);
        if(h.M != 0 && cols != 0)
        {
            float* const z = reinterpret_cast<float*>(ws + z_at);
            rc             = logits(a, b, v0, cols, z).run(scratch, stream);
            if(rc != ROCM_WMMA_GEMM_OK)
            {
                return rc;
            }
            const device::softmax_slope_args s{h.want, z, ws + dz_at, static_cast<long long>(pitch), static_cast<long long>(v0),
                                               static_cast<int>(cols), lse, factor, picked};
            h.bf16() ? launch_slope<__bf16>(s, stream) : launch_slope<_Float16>(s, stream);
        }
        if(wants_a)
        {
            rc = states(b, v0, cols, ws + dz_at, ws + sum_at).run(scratch, stream);
        }
        if(wants_b && rc == ROCM_WMMA_GEMM_OK)
        {
            rc = weights(a, v0, cols, ws + dz_at, ws + part_at).run(scratch, stream);
            if(scaled)
            {
                const bool nk = h.layout_b == 1;
                launch_scaled(out, reinterpret_cast<const float*>(ws + part_at), part_pitch,
                              static_cast<char*>(dB) + v0 * (nk ? h.K : 1) * size, h.b_length(), nk ? cols : h.K, nk ? h.K : cols, back,
                              accumulate, stream);
            }
        }
    }
    if(rc == ROCM_WMMA_GEMM_OK && wants_a && !own_place)
    {
        launch_scaled(out, reinterpret_cast<const float*>(ws + sum_at), k_pitch, dA, h.K, h.M, h.K, back, false, stream);
    }
    return rc;
}

// The operands' and the gradients' elements of a type pair; false for no pair.
bool elements_of(int type_idx, int* in, int* out)
{
    if(type_idx < 0 || type_idx > ROCM_WMMA_GEMM_TYPE_F32_BF16)
    {
        return false;
    }
    *in  = is_bf16(type_idx) ? ROCM_WMMA_GEMM_ELEMENT_BF16 : ROCM_WMMA_GEMM_ELEMENT_F16;
    *out = out_size(type_idx) == 4 ? ROCM_WMMA_GEMM_ELEMENT_F32 : *in;
    return true;
}

// (a list that is none has one entry, the target)
head head_of(int in, size_t M, size_t N, size_t K, int layout_b, const void* A, const void* B, const void* entries, int wide,
             const float* teacher, size_t k, float temperature)
{
    return {in, M, N, K, layout_b, A, B,
            {entries, wide, teacher, static_cast<long long>(N), static_cast<int>(std::min(M, most_rows + 1)),
             static_cast<int>(std::min<size_t>(k, device::most_entries + 1)), 1.0f / temperature}};
}

} // namespace
} // namespace host
} // namespace rocm_wmma_gemm

extern "C" {

using namespace rocm_wmma_gemm::host;

int rocm_wmma_gemm_linear_cross_entropy(int element, float* loss, float* lse, const void* A, const void* B, const void* targets,
                                        int wide_targets, size_t M, size_t N, size_t K, int layout_b, void* stream)
{
    return with_status([&] {
        const head h  = head_of(element, M, N, K, layout_b, A, B, targets, wide_targets, nullptr, 1, 1.0f);
        const int  rc = check_head(h, false);
        return rc != ROCM_WMMA_GEMM_OK ? rc : loss_of(h, loss, lse, nullptr, stream_of(stream));
    });
}

int rocm_wmma_gemm_linear_cross_entropy_backward(int type_idx, void* dA, void* dB, const float* dloss, const float* lse, const void* A,
                                                 const void* B, const void* targets, int wide_targets, size_t M, size_t N, size_t K,
                                                 int layout_b, int accumulate, void* stream)
{
    return with_status([&] {
        int in, out;
        if(!elements_of(type_idx, &in, &out) || (accumulate & ~1))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        const head h  = head_of(in, M, N, K, layout_b, A, B, targets, wide_targets, nullptr, 1, 1.0f);
        const int  rc = check_head(h, false);
        return rc != ROCM_WMMA_GEMM_OK ? rc : gradients_of(h, out, dA, dB, dloss, lse, nullptr, accumulate != 0, stream_of(stream));
    });
}

int rocm_wmma_gemm_linear_distillation(int element, float* loss, float* lse, float* picked, const void* A, const void* B,
                                       const void* entries, int wide_entries, const float* teacher, size_t M, size_t N, size_t K, size_t k,
                                       float temperature, int layout_b, void* stream)
{
    return with_status([&] {
        const head h  = head_of(element, M, N, K, layout_b, A, B, entries, wide_entries, teacher, k, temperature);
        const int  rc = check_head(h, true);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        return M != 0 && picked == nullptr ? ROCM_WMMA_GEMM_ERR_ARGUMENT : loss_of(h, loss, lse, picked, stream_of(stream));
    });
}

int rocm_wmma_gemm_linear_distillation_backward(int type_idx, void* dA, void* dB, const float* dloss, const float* lse,
                                                const float* picked, const void* A, const void* B, const void* entries, int wide_entries,
                                                const float* teacher, size_t M, size_t N, size_t K, size_t k, float temperature,
                                                int layout_b, int accumulate, void* stream)
{
    return with_status([&] {
        int in, out;
        if(!elements_of(type_idx, &in, &out) || (accumulate & ~1))
        {
            return ROCM_WMMA_GEMM_ERR_ARGUMENT;
        }
        const head h  = head_of(in, M, N, K, layout_b, A, B, entries, wide_entries, teacher, k, temperature);
        const int  rc = check_head(h, true);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        return M != 0 && picked == nullptr ? ROCM_WMMA_GEMM_ERR_ARGUMENT
                                           : gradients_of(h, out, dA, dB, dloss, lse, picked, accumulate != 0, stream_of(stream));
    });
}

} // extern "C"
