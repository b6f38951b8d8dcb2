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

constexpr size_t most_rows = size_t{1} << 20; // (a piece of 1024 columns of them fits the scratch buffer; their dA in fp32 may not: see gradients_of)

// A piece of the logits in fp32 is read back from the memory-side cache where it is not larger than this.
constexpr size_t piece_bytes = size_t{128} << 20;
// A piece of their gradient in 16 bits.
constexpr size_t slope_bytes = size_t{512} << 20;
// The statistics of rows that go together.
constexpr size_t parts_bytes = size_t{256} << 20, most_parts_bytes = size_t{4} << 30;
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

// Copies of the operands whose rows do not start on 16 bytes, which all of a call's products read, in one launch.  (Few rows
// too: 35 of 5787 elements against 55790 take 1040 us on the kernel that reads any address, a copy and the product 350.)
struct copies
{
    bool   a, b;
    size_t a_at = 0, b_at = 0;
    copies(const head& h, room& r)
        : a(h.M != 0 && h.K != 0 && (h.K % 8 != 0 || !aligned16(h.A))),
          b(h.N != 0 && h.M != 0 && h.K != 0 && (h.b_length() % 8 != 0 || !aligned16(h.B)))
    {
        a_at = a ? r.take(h.M * round_up8(h.K) * 2) : 0;
        b_at = b ? r.take(h.b_rows() * round_up8(h.b_length()) * 2) : 0;
    }
    // the operands, and (ws) their copies made; before anything is launched an aligned address stands for a copy
    void make(const head& h, operand* to_a, operand* to_b, char* ws, hipStream_t stream) const
    {
        auto job = [&](const void* given, size_t rows, size_t length, size_t at) {
            return device::pack_job{given, ws + at, static_cast<int>(rows), static_cast<int>(length), static_cast<int>(rows),
                                    static_cast<int>(round_up8(length)), 0, 0};
        };
        const device::pack_job ja = job(h.A, h.M, h.K, a_at), jb = job(h.B, h.b_rows(), h.b_length(), b_at);
        if(ws != nullptr && (a || b))
        {
            const size_t pieces = std::max(a ? h.M * round_up8(h.K) / 8 : 0, b ? h.b_rows() * round_up8(h.b_length()) / 8 : 0);
            follow(&device::pack_padded<unsigned short>,
                   dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(pieces, 256), 8192)), a && b ? 2 : 1), dim3(256), stream, a ? ja : jb,
                   b ? jb : ja);
        }
        *to_a = a ? operand{ws != nullptr ? ws + a_at : nullptr, round_up8(h.K)} : operand{h.A, h.K};
        *to_b = b ? operand{ws != nullptr ? ws + b_at : nullptr, round_up8(h.b_length())} : operand{h.B, h.b_length()};
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

// z = A B for a piece of the vocabulary: in fp32, rows `pitch` apart (finish_plain), or their gradient in 16 bits
// (finish_slope), or their statistics alone (finish_parts)
step logits_of(const head& h, int finish, const operand& a, const operand& b, size_t v0, size_t cols, void* z, size_t pitch)
{
    step s{finish == finish_plain ? h.to_f32() : h.to_16(), h.layout_b == 1 ? layout_kk : layout_kn, finish,
           one_problem(product_kind::rows, h.M, cols, h.K)};
    s.args.A      = a.at;
    s.args.B      = block_of_b(h, b, v0);
    s.args.C      = z;
    s.args.lda    = a.ld;
    s.args.ldb    = b.ld;
    s.args.ldc    = pitch;
    s.args.b_skip = h.layout_b == 1 ? 0 : v0;
    s.args.padded_c = 1;
    s.args.alpha    = finish == finish_plain ? 1.0f : h.want.scale2;
    s.args.col_base = static_cast<int>(v0);
    return s;
}

// How the logits' products run where they end in a tile's statistics (finish_parts) or gradients (finish_slope); no kernel
// where they write the logits for a pass of their own: rows too long for the tiles' offsets.
launch_choice fused_plan(const head& h, int finish, const operand& a, const operand& b, size_t cols)
{
    const launch_choice c = logits_of(h, finish, a, b, 0, cols, nullptr, round_up8(cols)).plan(compute_units());
    return c.copy_a || c.copy_b ? launch_choice{} : c;
}

// dA += dz B^T for a piece, rows `pitch` apart
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

// the piece's part of dB, in B's layout: unit dz^T A, or unit A^T dz
step weights_of(const head& h, const operand& a, const void* dz, size_t dz_pitch, size_t cols, int types, void* to, size_t pitch, bool add,
                const float* unit)
{
    const bool nk = h.layout_b == 1;
    step       s{types, layout_mn, finish_back, one_problem(product_kind::sum, nk ? cols : h.K, nk ? h.K : cols, h.M)};
    s.args.A        = nk ? dz : a.at;
    s.args.B        = nk ? a.at : dz;
    s.args.lda      = nk ? dz_pitch : a.ld;
    s.args.ldb      = nk ? a.ld : dz_pitch;
    s.args.C        = to;
    s.args.residual = add ? to : nullptr;
    s.args.ldc      = pitch;
    s.args.alpha_at = unit;
    return s;
}

// The weights' gradient of few rows is an outer product, bound by its stores; past these a tile's sums are long enough.
constexpr size_t most_outer = 64;

void launch_outer(const head& h, int out, const operand& a, const void* dz, size_t dz_pitch, size_t cols, void* to, const float* unit,
                  bool add, hipStream_t stream)
{
    const bool nk = h.layout_b == 1;
    device::outer_args o{nk ? dz : a.at, nk ? a.at : dz, to, unit, static_cast<long long>(nk ? dz_pitch : a.ld),
                         static_cast<long long>(nk ? a.ld : dz_pitch), static_cast<long long>(nk ? h.K : h.N),
                         static_cast<long long>(nk ? cols : h.K), static_cast<long long>(nk ? h.K : cols), static_cast<int>(h.M), add ? 1 : 0, device::outer_rows};
    // (fewer rows a workgroup where there would be less than two for every compute unit: 1788 x 740 are 21 workgroups of 256
    // rows, which took 16.8 us, nearly all of it one workgroup's way down its rows)
    while(o.each > 16 && ceil_div(o.rows, o.each) * ceil_div(o.cols, device::outer_cols) < 2 * compute_units())
    {
        o.each /= 2;
    }
    auto run = [&](auto* in_typed, auto* out_typed) {
        using in_t  = std::remove_pointer_t<decltype(in_typed)>;
        using out_t = std::remove_pointer_t<decltype(out_typed)>;
        // (a launch has 2^32 threads along x, so 2^24 blocks of rows are enough for any extent; 65535 blocks of columns are not)
        in_parts(ceil_div(o.cols, device::outer_cols), most_groups_y, [&](int block0, unsigned blocks) {
            device::outer_args part = o;
            const long long    skip = static_cast<long long>(block0) * device::outer_cols;
            part.Q                  = static_cast<const in_t*>(o.Q) + skip;
            part.C                  = static_cast<out_t*>(o.C) + skip;
            part.cols               = o.cols - skip;
            follow(h.M <= 32 ? &device::outer_product<in_t, out_t, 1> : &device::outer_product<in_t, out_t, 2>,
                   dim3(static_cast<unsigned>(ceil_div(o.rows, o.each)), blocks), dim3(256), stream, part);
        });
    };
    const bool f32 = out == ROCM_WMMA_GEMM_ELEMENT_F32;
    if(h.bf16())
    {
        __bf16* in = nullptr;
        f32 ? run(in, static_cast<float*>(nullptr)) : run(in, in);
    }
    else
    {
        _Float16* in = nullptr;
        f32 ? run(in, static_cast<float*>(nullptr)) : run(in, in);
    }
}

// Few rows of dA are sums over the whole vocabulary on few tiles: the vocabulary goes in `count` segments of `cols` columns, as
// a batch of products whose sums are added up as they are brought back, and a rest.
struct segments
{
    size_t count = 0, cols = 0;
    segments(const head& h, size_t all, size_t cus)
    {
        // (tiles of 32 columns, two workgroups a compute unit)
        const size_t wanted = std::min<size_t>(16, 2 * cus / std::max<size_t>(1, ceil_div(h.K, 32)));
        if(h.M <= most_outer && wanted >= 4 && all >= wanted * 1024)
        {
            cols  = all / wanted / piece_grain * piece_grain;
            count = wanted;
        }
    }
    size_t parts() const
    {
        return count + 1;
    }
};

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
       || !(h.want.scale > 0.0f) || !std::isfinite(h.want.scale2) || !std::isfinite(1.0f / h.want.scale)
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

// The rows row0 .. row0 + rows - 1 of a problem.
head rows_of(const head& h, size_t row0, size_t rows)
{
    head   p    = h;
    const size_t first = row0 * h.want.k;
    p.M         = rows;
    p.A         = static_cast<const char*>(h.A) + row0 * h.K * 2;
    p.want.rows = static_cast<int>(rows);
    p.want.entries = static_cast<const char*>(h.want.entries) + first * (h.want.wide ? 8 : 4);
    p.want.teacher = h.want.teacher != nullptr ? h.want.teacher + first : nullptr;
    return p;
}

// The listed logits where no logits are written and the tiles do not look for them.
void pick(const head& h, const operand& a, const operand& b, float* picked, hipStream_t stream)
{
    const bool     nk = h.layout_b == 1;
    const bool     eight = nk && h.K % 8 == 0 && a.ld % 8 == 0 && b.ld % 8 == 0 && aligned16(a.at) && aligned16(b.at);
    const unsigned groups = static_cast<unsigned>(std::min<size_t>(ceil_div(h.M * h.want.k, 4), size_t{1} << 16));
    const device::pick_args args{h.want, a.at, b.at, static_cast<long long>(a.ld), nk ? static_cast<long long>(b.ld) : 1,
                                 nk ? 1 : static_cast<long long>(b.ld), static_cast<int>(h.K), picked};
    if(h.bf16())
    {
        follow(eight ? &device::pick_products<__bf16, 8> : &device::pick_products<__bf16, 1>, dim3(groups), dim3(256), stream, args);
    }
    else
    {
        follow(eight ? &device::pick_products<_Float16, 8> : &device::pick_products<_Float16, 1>, dim3(groups), dim3(256), stream, args);
    }
}

// loss, lse and (a list) the listed logits of some rows, from operands whose copies are made
struct loss_plan
{
    bool   fused, gathers; // its tiles end in statistics; the listed logits are worked out on their own
    pieces p;
    size_t each, all; // parts of a piece, of a row
    size_t z_at, parts_at, picked_at, product_at, product;
    launch_choice tiles; // fused
    loss_plan(const head& h, const operand& a, const operand& b, bool own_picked, room r)
        : fused(false), p(0, 0)
    {
        product = 0;
        tiles   = fused_plan(h, finish_parts, a, b, h.N);
        // (the few-row kernels look for the listed entries themselves; a column of weights that are stored K x N is gathered
        // element by element, so a list of them is picked from the logits)
        gathers = tiles.kernel.per_cu != 0;
        fused   = tiles.kernel.fn != nullptr && (!gathers || h.layout_b == 1 || h.want.teacher == nullptr);
        p       = pieces(h.N, fused ? h.N : piece_bytes / (4 * h.M));
        if(fused)
        {
            // (a wave's columns of a tile, or a tile of the few-row kernels)
            each  = ceil_div(h.N, tiles.kernel.per_cu != 0 ? tiles.kernel.block_n / 2 : tiles.kernel.block_n);
            all   = each;
            fused = h.M * all * sizeof(device::softmax_part) <= most_parts_bytes;
            p     = fused ? p : pieces(h.N, piece_bytes / (4 * h.M));
        }
        if(!fused)
        {
            each = ceil_div(p.cols, device::part_cols);
            all  = h.N != 0 ? each * p.count : 0;
            for(size_t v0 = 0; v0 < h.N; v0 += p.cols)
            {
                product = std::max(product, logits_of(h, finish_plain, a, b, v0, std::min(p.cols, h.N - v0), nullptr, p.pitch())
                                                .plan(compute_units())
                                                .scratch());
                v0 = v0 == 0 && p.count > 2 ? (p.count - 2) * p.cols : v0; // (the first and the last are all there are)
            }
        }
        z_at       = fused ? 0 : r.take(h.M * p.pitch() * 4);
        parts_at   = r.take(h.M * all * sizeof(device::softmax_part));
        picked_at  = own_picked ? r.take(h.M * sizeof(float)) : 0;
        product_at = r.bytes;
    }
    size_t bytes() const
    {
        return product_at + product;
    }
};

int loss_of_rows(const head& h, const loss_plan& plan, const operand& a, const operand& b, float* loss, float* lse, float* picked, char* ws,
                 hipStream_t stream)
{
    using device::softmax_part;
    float* const        of_targets = picked == nullptr ? reinterpret_cast<float*>(ws + plan.picked_at) : picked;
    softmax_part* const parts      = reinterpret_cast<softmax_part*>(ws + plan.parts_at);
    char* const         scratch    = ws + plan.product_at;
    if(plan.fused)
    {
        step s              = logits_of(h, finish_parts, a, b, 0, h.N, nullptr, round_up8(h.N));
        s.args.parts        = parts;
        s.args.parts_of_row = static_cast<int>(plan.all);
        s.args.entries      = h.want.entries;
        s.args.wide_entries = h.want.wide;
        s.args.listed       = h.want.k;
        s.args.picked       = of_targets;
        const int rc        = launch_product(s.types, s.finish, plan.tiles, s.args, nullptr, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        if(plan.gathers)
        {
            pick(h, a, b, of_targets, stream);
        }
    }
    const unsigned pick_groups = static_cast<unsigned>(std::min<size_t>(ceil_div(h.M * h.want.k, 256), 4096));
    for(size_t v0 = 0; !plan.fused && v0 < std::max<size_t>(h.N, 1); v0 += plan.p.cols)
    {
        const size_t cols  = std::min(plan.p.cols, h.N - v0), pitch = plan.p.pitch();
        float* const z     = reinterpret_cast<float*>(ws + plan.z_at);
        const int    rc    = logits_of(h, finish_plain, a, b, v0, cols, z, pitch).run(scratch, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
        follow(&device::pick_entries, dim3(pick_groups), dim3(256), stream, h.want, static_cast<const float*>(z),
               static_cast<long long>(pitch), static_cast<long long>(v0), static_cast<int>(cols), of_targets);
        if(cols != 0)
        {
            // (the last piece may have fewer parts than the others: its rest has none)
            const device::part_args args{z, parts, static_cast<long long>(pitch), static_cast<int>(cols),
                                         static_cast<int>(v0 / plan.p.cols * plan.each), static_cast<int>(plan.all), h.want.scale2};
            follow(&device::softmax_parts, dim3(static_cast<unsigned>(h.M), static_cast<unsigned>(plan.each)), dim3(256), stream, args);
        }
    }
    const bool few = h.M < 1024;
    follow(few ? &device::join_rows<4> : &device::join_rows<1>, dim3(few ? static_cast<unsigned>(h.M) : row_groups(h.M)), dim3(256), stream,
           device::join_args{h.want, parts, of_targets, loss, lse, static_cast<int>(plan.all)});
    return ROCM_WMMA_GEMM_OK;
}

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
    // rows have nothing to do with each other: as many go together as leave the statistics their room (64 columns a part)
    const size_t some = std::min(h.M, std::max<size_t>(256, parts_bytes / sizeof(device::softmax_part) / (h.N / 64 + 1)));
    room         r;
    const copies c(h, r);
    operand      a, b;
    c.make(h, &a, &b, nullptr, stream);
    const loss_plan first(rows_of(h, 0, some), a, b, picked == nullptr, r);
    const size_t    rest = h.M % some;
    const loss_plan last  = rest != 0 ? loss_plan(rows_of(h, 0, rest), a, b, picked == nullptr, r) : first;
    workspace_lease lease;
    char*           ws = lease.acquire(std::max(first.bytes(), last.bytes()), stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    c.make(h, &a, &b, ws, stream);
    for(size_t row = 0; row < h.M; row += some)
    {
        const size_t  rows = std::min(some, h.M - row);
        const operand from{static_cast<const char*>(a.at) + row * a.ld * 2, a.ld};
        const int     rc = loss_of_rows(rows_of(h, row, rows), rows == some ? first : last, from, b, loss + row, lse + row,
                                        picked != nullptr ? picked + row * h.want.k : nullptr, ws, stream);
        if(rc != ROCM_WMMA_GEMM_OK)
        {
            return rc;
        }
    }
    return ROCM_WMMA_GEMM_OK;
}

template<class InT>
void launch_slope(const device::softmax_slope_args& s, bool fused, hipStream_t stream)
{
    if(!fused)
    {
        follow(&device::softmax_slope<InT>, dim3(static_cast<unsigned>(s.want.rows), static_cast<unsigned>(ceil_div(s.pitch, 2048))),
               dim3(256), stream, s);
    }
    if(s.want.teacher != nullptr)
    {
        follow(&device::listed_slope<InT>, dim3(row_groups(s.want.rows)), dim3(256), stream, s);
    }
}

// dA and dB (either may be missing) from the loss's gradient by row.
//
// What is rounded, and why: dz to A's type, as both products need it, in the units of record_args.  dA's parts are added up in
// fp32 over the pieces.
//
// A million rows of thousands of elements in fp32 are more than the scratch buffer may hold: then dB is worked out for itself, from all
// rows, so that its sums are rounded once, and dA behind it in blocks of rows, which have nothing to do with each other, at the
// price of the logits a third time.  asked: only whether there is room, nothing is launched.
int gradients_of(const head& h, int out, void* dA, void* dB, const float* dloss, const float* lse, const float* picked, bool accumulate,
                 hipStream_t stream, bool asked = false)
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
    const bool   f32 = out == ROCM_WMMA_GEMM_ELEMENT_F32;
    const size_t size = f32 ? 4 : 2, cus = compute_units(), rows = std::max<size_t>(h.M, 1);
    const int    types = f32 ? h.to_f32() : h.to_16();
    room         r;
    const copies c(h, r);
    operand      plan_a, plan_b;
    c.make(h, &plan_a, &plan_b, nullptr, stream);
    const bool   fused = h.N != 0 && fused_plan(h, finish_slope, plan_a, plan_b, h.N).kernel.fn != nullptr;
    const pieces p(h.N, fused ? slope_bytes / (2 * rows) : piece_bytes / (4 * rows));
    const size_t pitch = p.pitch(), k_pitch = round_up8(h.K);
    const bool   outer = h.M <= most_outer && h.M != 0;
    // (segments of a single piece: few rows have no more)
    const segments seg = p.count == 1 ? segments(h, h.N, cus) : segments(h, 0, cus);
    const size_t z_at = fused ? 0 : r.take(h.M * pitch * 4), dz_at = r.take(h.M * pitch * 2 + (seg.count != 0 ? h.N * 2 : 0)), // (a segment's loads may reach so far past the last row)
                 records_at = r.take(h.M * sizeof(device::loss_record)), unit_at = r.take(8),
                 counted_at = h.want.teacher != nullptr ? r.take(h.M * sizeof(float)) : 0,
                 sum_at = wants_a ? r.take(seg.parts() * h.M * k_pitch * 4) : 0, product_at = r.bytes;
    auto logits = [&](const operand& a, const operand& b, size_t v0, size_t cols, char* ws) {
        step s = logits_of(h, fused ? finish_slope : finish_plain, a, b, v0, cols, ws != nullptr ? ws + (fused ? dz_at : z_at) : nullptr, pitch);
        s.args.records = ws != nullptr ? reinterpret_cast<const device::loss_record*>(ws + records_at) : nullptr;
        return s;
    };
    auto states = [&](const operand& b, size_t v0, size_t cols, char* ws) {
        return states_of(h, ws != nullptr ? ws + dz_at : nullptr, pitch, b, v0, cols, h.to_f32(), ws != nullptr ? ws + sum_at : nullptr,
                         k_pitch, v0 != 0);
    };
    auto weights = [&](const operand& a, size_t v0, size_t cols, char* ws) {
        return weights_of(h, a, ws != nullptr ? ws + dz_at : nullptr, pitch, cols, types,
                          static_cast<char*>(dB) + v0 * (h.layout_b == 1 ? h.K : 1) * size, h.b_length(), accumulate,
                          ws != nullptr ? reinterpret_cast<const float*>(ws + unit_at) : nullptr);
    };
    // part 0: all segments in one launch (seg.count of them), part 1: the rest behind them; without segments part 0 is all
    auto states_part = [&](const operand& b, size_t v0, size_t cols, size_t part, char* ws) {
        if(seg.count == 0)
        {
            return states(b, v0, cols, ws);
        }
        if(part == 0)
        {
            step s          = states(b, 0, seg.cols, ws);
            s.args.kind     = product_kind::batch;
            s.args.groups   = static_cast<int>(seg.count);
            s.args.stride_a = static_cast<long long>(seg.cols);
            s.args.stride_b = static_cast<long long>(seg.cols * (h.layout_b == 1 ? b.ld : 1));
            s.args.stride_c = static_cast<long long>(h.M * k_pitch);
            // (a block of columns ends with the last row of the matrix, not of the block's rows)
            s.args.b_skip = h.layout_b == 1 ? 0 : static_cast<long long>((seg.count - 1) * seg.cols);
            return s;
        }
        const size_t first = seg.count * seg.cols;
        step         s     = states(b, first, cols - first, ws);
        if(ws != nullptr)
        {
            s.args.A = static_cast<const char*>(s.args.A) + first * 2;
            s.args.C = static_cast<char*>(s.args.C) + seg.count * h.M * k_pitch * 4;
        }
        s.finish        = finish_plain;
        s.args.residual = nullptr;
        return s;
    };
    const size_t launches = seg.count == 0 || seg.count * seg.cols == h.N ? 1 : 2;
    size_t product = 0;
    for(size_t v0 = 0; v0 < std::max<size_t>(h.N, 1); v0 += p.cols)
    {
        const size_t cols = std::min(p.cols, h.N - v0);
        product = std::max(product, logits(plan_a, plan_b, v0, cols, nullptr).plan(cus).scratch());
        for(size_t part = 0; wants_a && part < launches; ++part)
        {
            product = std::max(product, states_part(plan_b, v0, cols, part, nullptr).plan(cus).scratch());
        }
        product = std::max(product, wants_b && !outer ? weights(plan_a, v0, cols, nullptr).plan(cus).scratch() : 0);
        v0 = v0 == p.cols && p.count > 3 ? (p.count - 2) * p.cols : v0; // (the first, one behind it, the last)
    }
    if(product_at + product > workspace_limit_bytes)
    {
        if(!wants_a || (!wants_b && h.M == 1))
        {
            return ROCM_WMMA_GEMM_ERR_SCRATCH;
        }
        auto parts = [&](bool only_asked) {
            if(wants_b)
            {
                const int rc = gradients_of(h, out, nullptr, dB, dloss, lse, picked, accumulate, stream, only_asked);
                return rc != ROCM_WMMA_GEMM_OK ? rc
                                               : gradients_of(h, out, dA, nullptr, dloss, lse, picked, false, stream, only_asked);
            }
            const size_t half = ceil_div(h.M, 2);
            for(size_t row = 0; row < h.M; row += half)
            {
                const int rc = gradients_of(rows_of(h, row, std::min(half, h.M - row)), out, static_cast<char*>(dA) + row * h.K * size, nullptr,
                                            dloss + row, lse + row, picked != nullptr ? picked + row * h.want.k : nullptr, false, stream,
                                            only_asked);
                if(rc != ROCM_WMMA_GEMM_OK || only_asked) // (the second half is no larger)
                {
                    return rc;
                }
            }
            return ROCM_WMMA_GEMM_OK;
        };
        const int rc = parts(true);
        return rc != ROCM_WMMA_GEMM_OK || asked ? rc : parts(false);
    }
    if(asked)
    {
        return ROCM_WMMA_GEMM_OK;
    }
    workspace_lease lease;
    char*           ws = lease.acquire(product_at + product, stream);
    if(ws == nullptr)
    {
        return ROCM_WMMA_GEMM_ERR_SCRATCH;
    }
    operand       a, b;
    c.make(h, &a, &b, ws, stream);
    char* const   scratch = ws + product_at;
    device::record_args f{h.want, dloss, lse, reinterpret_cast<device::loss_record*>(ws + records_at),
                          reinterpret_cast<float*>(ws + unit_at)};
    if(h.want.teacher != nullptr && h.M != 0)
    {
        float* const counted = reinterpret_cast<float*>(ws + counted_at);
        follow(&device::counted_gradients, dim3(row_groups(h.M)), dim3(256), stream, h.want, dloss, counted);
        f.dloss = counted;
    }
    const unsigned groups = static_cast<unsigned>(ceil_div(rows, 256));
    if(h.M > device::most_alone)
    {
        follow(&device::gradient_unit, dim3(1), dim3(1024), stream, f);
        follow(&device::gradient_records<false>, dim3(groups), dim3(256), stream, f);
    }
    else
    {
        follow(&device::gradient_records<true>, dim3(groups), dim3(256), stream, f);
    }
    int rc = ROCM_WMMA_GEMM_OK;
    for(size_t v0 = 0; v0 < std::max<size_t>(h.N, 1) && rc == ROCM_WMMA_GEMM_OK; v0 += p.cols)
    {
        const size_t cols = std::min(p.cols, h.N - v0);
        if(h.M != 0 && cols != 0)
        {
            rc = logits(a, b, v0, cols, ws).run(scratch, stream);
            if(rc != ROCM_WMMA_GEMM_OK)
            {
                return rc;
            }
            const device::softmax_slope_args s{h.want, reinterpret_cast<const float*>(ws + z_at), ws + dz_at, static_cast<long long>(pitch),
                                               static_cast<long long>(v0), static_cast<int>(cols), f.records, picked};
            h.bf16() ? launch_slope<__bf16>(s, fused, stream) : launch_slope<_Float16>(s, fused, stream);
        }
        for(size_t part = 0; wants_a && rc == ROCM_WMMA_GEMM_OK && part < launches; ++part)
        {
            rc = states_part(b, v0, cols, part, ws).run(scratch, stream);
        }
        if(wants_b && rc == ROCM_WMMA_GEMM_OK)
        {
            if(outer && cols != 0)
            {
                launch_outer(h, out, a, ws + dz_at, pitch, cols, static_cast<char*>(dB) + v0 * (h.layout_b == 1 ? h.K : 1) * size, f.unit,
                             accumulate, stream);
            }
            else
            {
                rc = weights(a, v0, cols, ws).run(scratch, stream);
            }
        }
    }
    if(rc == ROCM_WMMA_GEMM_OK && wants_a)
    {
        const size_t sums = seg.count == 0 ? 1 : seg.count + launches - 1;
        by_element(out, [&](auto* typed) {
            using out_t = std::remove_pointer_t<decltype(typed)>;
            follow(&device::scaled_rows<out_t>, dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(h.M * k_pitch, 1024), 8192))), dim3(256),
                   stream, reinterpret_cast<const float*>(ws + sum_at), static_cast<int>(sums), static_cast<long long>(h.M * k_pitch),
                   static_cast<long long>(k_pitch), static_cast<out_t*>(dA),
                   static_cast<long long>(h.M), static_cast<long long>(h.K), f.unit);
        });
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
             static_cast<int>(std::min<size_t>(k, device::most_entries + 1)), 1.0f / temperature, device::log2_of_e / temperature}};
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
