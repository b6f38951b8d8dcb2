// What the kernels of the layer products share (C = act(alpha A B + bias) + beta R for one
// weight, for a batch, or for groups of rows with a weight each): their arguments, the table of
// the groups, where an item of work lies, and the mathematics of the epilogue.
//
// A product works on `groups` problems of one of three kinds:
//   batch   problem e is A + e stride_a times B + e stride_b, all of one shape;
//   rows    A's rows are sorted by group: problem e has rows [o_e, o_e+1) of A and of C and a
//           weight of its own (a forward product of experts, or the gradient of its input);
//   sum     the sum runs over the rows of a group: problem e is the product of rows
//           [o_e, o_e+1) of A (transposed) with the same rows of B (the gradient of the weights).
// The offsets o live on the device, so a router's answer never travels to the host: every
// workgroup scans them into its LDS (E + 1 integers, one wave, two scans of 64 lanes) and finds
// its tile there.
#ifndef ROCM_WMMA_GEMM_PRODUCT_COMMON_HPP
#define ROCM_WMMA_GEMM_PRODUCT_COMMON_HPP

#include "gemm_kernel.hpp"
#include "product_cut.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

// y = x s(u) with s the logistic function covers silu (u = x) and the tanh form of gelu
// (0.5 (1 + tanh t) = s(2 t), so u = 2 sqrt(2/pi) (x + 0.044715 x^3)): u = k1 x + k3 x^3.
enum class act_kind
{
    none     = 0,
    relu     = 1,
    logistic = 2
};

// What a product does with a diagonal that is held beside its matrix in fp32 (diagonal).
enum class diagonal_use
{
    none  = 0,
    split = 1, // C is square: its diagonal goes there, and C gets zeros in its place
    rows  = 2 // row i of R is multiplied by beta + alpha diagonal[i]
};

struct act_args
{
    act_kind kind;
    float    k1, k3;
};

constexpr int max_groups = 512; // two tables of this many integers fit beside every ring in LDS

struct product_args
{
    void*        C;
    void*        kept; // nullptr, or where a second output goes (see finish)
    const void*  A;
    const void*  B;
    const void*  bias; // nullptr, or N values of A's type per group
    const void*  residual; // nullptr, or a matrix laid out as C; may be C itself
    const int*   offsets; // groups + 1 row offsets on the device (rows, sum), not decreasing;
                          // nullptr: one group of all rows
    product_kind kind;
    int          groups;
    int          M, N, K; // of every problem; rows: M counts the rows of all groups, sum: K does
    long long    lda, ldb, ldc; // of the contiguous rows in memory
    long long    stride_a, stride_b, stride_c, stride_bias; // elements from group to group (batch)
    float        alpha, beta;
    act_args     act;
    int          keep_sum; // kept holds 0: alpha A B + bias, before the activation (A's type);
                           // 1: the finished value, C's, in A's type
    diagonal_use diagonal_is;
    float*       diagonal; // stride_diagonal values from group to group
    long long    stride_diagonal;
    int          grid_m, grid_n; // tiles of a problem (rows: grid_m is not used)
    int          wide; // few-row kernel: rows of C and of what is added start on 16 bytes
    float*       partials; // tiled kernels: nullptr, or room for a tile of fp32 per workgroup of the
                           // grid; the tiles of the last round may then be cut along K (cut_tail)
    int          workgroups; // of the grid that writes them
    int           k_slices; // few-row kernel: workgroups that share a tile, each with a run of K; 1: none do
    unsigned int* arrivals; // with k_slices > 1: a counter per tile, and this launch's tag in them
    unsigned int  arrival_epoch;
};

__device__ __forceinline__ int clamped_offset(int v, int rows)
{
    return v < 0 ? 0 : v > rows ? rows : v;
}

// The groups' row offsets and, for tiles of BM rows, how many row tiles lie before each group:
// off[0 .. groups], first[0 .. groups].  Offsets that decrease or leave [0, rows] are clamped, so that
// no value of theirs makes a kernel touch memory outside its operands.  Called by all threads of
// a workgroup; the tables are ready behind its barrier.
template<class IntPtr>
__device__ __forceinline__ void build_group_table(const int* offsets, int groups, int rows, int BM, IntPtr off,
                                                  IntPtr first)
{
    if(threadIdx.x < 64)
    {
        const int lane       = threadIdx.x;
        int       carry_off  = offsets != nullptr ? clamped_offset(offsets[0], rows) : 0;
        int       carry_tile = 0;
        if(lane == 0)
        {
            off[0]   = carry_off;
            first[0] = 0;
        }
        for(int base = 0; base < groups; base += 64)
        {
            const int e = base + lane;
            int       v = e < groups ? (offsets != nullptr ? clamped_offset(offsets[e + 1], rows) : rows) : 0;
            v           = v > carry_off ? v : carry_off;
#pragma unroll
            for(int d = 1; d < 64; d *= 2)
            {
                const int u = __shfl_up(v, d);
                v           = lane >= d && u > v ? u : v;
            }
            const int before = __shfl_up(v, 1);
            const int own    = v - (lane == 0 ? carry_off : before);
            int       t      = (own + BM - 1) / BM;
#pragma unroll
            for(int d = 1; d < 64; d *= 2)
            {
                const int u = __shfl_up(t, d);
                t += lane >= d ? u : 0;
            }
            t += carry_tile;
            if(e < groups)
            {
                off[e + 1]   = v;
                first[e + 1] = t;
            }
            carry_off  = __shfl(v, 63);
            carry_tile = __shfl(t, 63);
        }
    }
    __syncthreads();
}

// order[0 .. groups]: the groups by falling size (ties by number), for launches whose groups cost as
// much as they have rows: dealt in this order, round by round, the persistent workgroups end nearly
// together.  Ready behind its barrier.
template<class IntPtr>
__device__ __forceinline__ void order_groups(int groups, IntPtr off, IntPtr order)
{
    for(int e = threadIdx.x; e < groups; e += blockDim.x)
    {
        const int own  = off[e + 1] - off[e];
        int       rank = 0;
#pragma unroll 8
        for(int j = 0; j < groups; ++j)
        {
            const int other = off[j + 1] - off[j];
            rank += other > own || (other == own && j < e);
        }
        order[rank] = e;
    }
    __syncthreads();
}

// Where a group's tiles fit the grid several times, the workgroups form that many teams of `tiles`, and a
// team takes whole groups: each group, in order_groups' order, goes to the team with the least to do
// so far.  A group costs its K tiles and what a tile's start and end take, about 5 more.
constexpr int most_teamed_groups = 64, most_teams = 64, tile_overhead = 5;

RWG_HD inline int teams_of(int groups, int tiles, int workgroups)
{
    const int teams = workgroups / tiles;
    // (left-over workgroups stay idle: not more than one in eight)
    return groups <= most_teamed_groups && groups > teams && teams >= 2 && teams <= most_teams && teams * tiles * 8 >= workgroups * 7 ? teams
                                                                                                                  : 0;
}

// The least of a wave's 64 values, in every lane: four shifts within rows of 16 lanes, two broadcasts
// across them (a few cycles each, where a shuffle through LDS takes sixty).
__device__ __forceinline__ unsigned int least_of_wave(unsigned int v)
{
    constexpr int most = -1; // (all ones: no lane's value is more)
    auto least = [&](int other) { v = v < (unsigned int)other ? v : (unsigned int)other; };
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x111, 0xf, 0xf, false)); // row_shr:1
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x112, 0xf, 0xf, false));
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x114, 0xf, 0xf, false));
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x118, 0xf, 0xf, false));
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x142, 0xa, 0xf, false)); // row_bcast:15
    least(__builtin_amdgcn_update_dpp(most, (int)v, 0x143, 0xc, 0xf, false)); // row_bcast:31
    return (unsigned int)__builtin_amdgcn_readlane((int)v, 63);
}

// The groups of team `team`, into mine[0 ..]; returns how many.  Called by all threads of a workgroup;
// ready behind its barrier.
template<class IntPtr>
__device__ __forceinline__ int deal_groups(int groups, int teams, int team, int BK, IntPtr off, IntPtr order, IntPtr mine,
                                           IntPtr count)
{
    if(threadIdx.x < 64)
    {
        const int lane  = threadIdx.x;
        const int group = order[lane < groups ? lane : 0]; // the lane-th in order, and its cost
        const int cost  = (off[group + 1] - off[group] + BK - 1) / BK + tile_overhead;
        int       load = 0, taken = 0;
        for(int i = 0; i < groups; ++i)
        {
            // the least load, of those the first team (all K tiles of 2^31 rows, times 64, fit 32 bits unsigned)
            const int to = (int)(least_of_wave(lane < teams ? (unsigned int)load * 64 + lane : ~0u) & 63u);
            load += lane == to ? __builtin_amdgcn_readlane(cost, i) : 0;
            if(to == team)
            {
                const int e = __builtin_amdgcn_readlane(group, i);
                if(lane == 0)
                {
                    mine[taken] = e;
                }
                ++taken;
            }
        }
        if(lane == 0)
        {
            *count = taken;
        }
    }
    __syncthreads();
    return *count;
}

// The group that row tile number `tile` belongs to: the last e with first[e] <= tile (groups
// without rows share their successor's number and are passed over).  Asked by whole waves, 64
// groups at a time.
template<class IntPtr>
__device__ __forceinline__ int group_of_tile(IntPtr first, int groups, int tile)
{
    const int lane = threadIdx.x & 63;
    int       e    = 0;
    for(int base = 0; base < groups; base += 64)
    {
        const int  i    = base + lane + 1;
        const bool pass = i < groups && first[i < groups ? i : 0] <= tile;
        e += __popcll(__ballot(pass));
    }
    return __builtin_amdgcn_readfirstlane(e);
}

// One tile of work: its group, where its corner lies in that group's C, the group's extents and
// where its operands start.
struct product_item
{
    int       group;
    int       row0, col0;
    int       m, k; // the group's rows of C and length of the sums
    long long a_at, b_at, c_at; // elements from the operands' bases to the group's
};

template<class IntPtr>
__device__ __forceinline__ void place_group(const product_args& args, IntPtr off, product_item& x)
{
    if(args.kind == product_kind::batch)
    {
        x.m    = args.M;
        x.k    = args.K;
        x.a_at = x.group * args.stride_a;
        x.b_at = x.group * args.stride_b;
        x.c_at = x.group * args.stride_c;
        return;
    }
    const int begin = __builtin_amdgcn_readfirstlane(off[x.group]);
    const int count = __builtin_amdgcn_readfirstlane(off[x.group + 1]) - begin;
    x.a_at          = begin * args.lda;
    if(args.kind == product_kind::rows)
    {
        x.m    = count;
        x.k    = args.K;
        x.b_at = x.group * args.stride_b;
        x.c_at = begin * args.ldc;
    }
    else
    {
        x.m    = args.M;
        x.k    = count;
        x.b_at = begin * args.ldb;
        x.c_at = x.group * args.stride_c;
    }
}

// How many tiles a launch has.
template<class IntPtr>
__device__ __forceinline__ int count_items(const product_args& args, IntPtr first)
{
    return args.kind == product_kind::rows ? first[args.groups] * args.grid_n
                                           : args.groups * args.grid_m * args.grid_n;
}

__device__ __forceinline__ float logistic(float u)
{
    // exp2 and the reciprocal are the hardware's (1 ulp each): e^-u overflows to infinity below
    // u = -88 and its reciprocal is the 0 that belongs there
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u));
}

__device__ __forceinline__ float activate(const act_args& act, float x)
{
    if(act.kind == act_kind::relu)
    {
        return x < 0.0f ? 0.0f : x; // (NaN stays)
    }
    if(act.kind == act_kind::logistic)
    {
        // (s(u) is 0 or 1 long before |x| = 1e4; the clamp keeps x^2 from overflowing, where the
        // product with k3 = 0 would be no number.  A NaN comes back through the factor x.)
        const float c = __builtin_amdgcn_fmed3f(x, -1.0e4f, 1.0e4f);
        return x * logistic(c * (act.k1 + act.k3 * c * c));
    }
    return x;
}

// d activate / dx.  Past |x| = 64 the slope of both logistic forms is 0 or 1 to the last bit of
// fp32; the clamp keeps x^3 from turning into infinity times zero.
__device__ __forceinline__ float activate_slope(const act_args& act, float x)
{
    if(act.kind == act_kind::relu)
    {
        return x <= 0.0f ? 0.0f : 1.0f;
    }
    if(act.kind == act_kind::logistic)
    {
        const float c = x > 64.0f ? 64.0f : x < -64.0f ? -64.0f : x;
        const float s = logistic(c * (act.k1 + act.k3 * c * c));
        return s + c * s * (1.0f - s) * (act.k1 + 3.0f * act.k3 * c * c);
    }
    return 1.0f;
}

// One element of C from its accumulated product: z = alpha sum + bias, y = act(z) + beta R,
// everything in fp32 and each output rounded once.
template<class InT, class OutT, class ResT>
__device__ __forceinline__ void finish_element(const product_args& args, const product_item& x, int row, int col,
                                               float sum)
{
    float z = args.alpha * sum;
    if(args.bias != nullptr)
    {
        z += (float)static_cast<const InT*>(args.bias)[x.group * args.stride_bias + col];
    }
    const long long at = x.c_at + row * args.ldc + col;
    float           y  = activate(args.act, z);
    if(args.residual != nullptr)
    {
        float beta = args.beta;
        if(args.diagonal_is == diagonal_use::rows)
        {
            beta += args.alpha * args.diagonal[x.group * args.stride_diagonal + row];
        }
        y += beta * (float)static_cast<const ResT*>(args.residual)[at];
    }
    if(args.diagonal_is == diagonal_use::split && row == col)
    {
        args.diagonal[x.group * args.stride_diagonal + row] = y;
        y                                                   = 0.0f;
    }
    if(args.kept != nullptr)
    {
        static_cast<InT*>(args.kept)[at] = to_out<InT>(args.keep_sum ? y : z);
    }
    static_cast<OutT*>(args.C)[at] = to_out<OutT>(y);
}

// Eight consecutive elements of a row, as 16-byte pieces: for operands whose rows start on 16 bytes.
template<class InT, class OutT, class ResT>
__device__ __forceinline__ void finish_piece(const product_args& args, const product_item& x, int row, int col,
                                             const float (&sum)[8])
{
    typedef InT     in8 __attribute__((ext_vector_type(8)));
    typedef OutT    out8 __attribute__((ext_vector_type(8)));
    typedef ResT    res8 __attribute__((ext_vector_type(8)));
    const long long at = x.c_at + row * args.ldc + col;
    float           z[8], y[8];
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        z[e] = args.alpha * sum[e];
    }
    if(args.bias != nullptr)
    {
        const in8 b = *reinterpret_cast<const in8*>(static_cast<const InT*>(args.bias) + x.group * args.stride_bias + col);
#pragma unroll
        for(int e = 0; e < 8; ++e)
        {
            z[e] += (float)b[e];
        }
    }
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        y[e] = activate(args.act, z[e]);
    }
    if(args.residual != nullptr)
    {
        const res8 r = *reinterpret_cast<const res8*>(static_cast<const ResT*>(args.residual) + at);
        const float beta = args.diagonal_is == diagonal_use::rows
                               ? args.beta + args.alpha * args.diagonal[x.group * args.stride_diagonal + row]
                               : args.beta;
#pragma unroll
        for(int e = 0; e < 8; ++e)
        {
            y[e] += beta * (float)r[e];
        }
    }
    if(args.diagonal_is == diagonal_use::split && row >= col && row < col + 8)
    {
#pragma unroll
        for(int e = 0; e < 8; ++e)
        {
            if(row == col + e)
            {
                args.diagonal[x.group * args.stride_diagonal + row] = y[e];
                y[e]                                                = 0.0f;
            }
        }
    }
    if(args.kept != nullptr)
    {
        in8 k;
#pragma unroll
        for(int e = 0; e < 8; ++e)
        {
            k[e] = to_out<InT>(args.keep_sum ? y[e] : z[e]);
        }
        *reinterpret_cast<in8*>(static_cast<InT*>(args.kept) + at) = k;
    }
    out8 o;
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        o[e] = to_out<OutT>(y[e]);
    }
    *reinterpret_cast<out8*>(static_cast<OutT*>(args.C) + at) = o;
}

template<class Impl>
__global__ void __launch_bounds__(Impl::THREADS) product_entry(const product_args args)
{
    Impl::run(args);
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_COMMON_HPP
