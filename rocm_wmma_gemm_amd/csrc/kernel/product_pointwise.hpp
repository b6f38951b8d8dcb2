// The element-wise passes around the layer products: the gradient through an activation with
// the column sums that a bias needs, and the start and end of the Newton-Schulz steps.  Each is
// bound by memory.
#ifndef ROCM_WMMA_GEMM_PRODUCT_POINTWISE_HPP
#define ROCM_WMMA_GEMM_PRODUCT_POINTWISE_HPP

#include "product_common.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

// dZ = dC * act'(Z), and the sums of its columns over runs of slope_rows rows of a group.
constexpr int slope_rows = 32; // rows of a run (a workgroup's); a group's last run is shorter

struct slope_args
{
    const void* dc; // rows x cols of 16-bit elements
    const void* z; // the same, or nullptr: dZ = dC
    void*       dz; // nullptr: not wanted (dZ = dC)
    int         dz_pitch; // its row length, a multiple of 8: columns past cols are written as zeros
    float*      sums; // nullptr, or [run][cols]
    const int*  offsets; // groups + 1, or nullptr: one group
    int         groups, rows, cols;
    act_args    act;
};

// A wave takes 64 * WIDTH columns, the four waves of a workgroup every fourth row of a run
// (blockIdx.x); WIDTH = 8 where rows start on 16 bytes, else 1.  The sums of a run are added in
// the order of its rows within a wave, then in wave order: the same in every call.
template<class InT, int WIDTH>
__global__ void __launch_bounds__(256) activation_slope(const slope_args args)
{
    __shared__ int   off[max_groups + 1], first[max_groups + 1];
    __shared__ float part[4][64 * WIDTH];
    build_group_table(args.offsets, args.groups, args.rows, slope_rows, &off[0], &first[0]);
    const int run = blockIdx.x;
    if(run >= first[args.groups])
    {
        return;
    }
    const int group = group_of_tile(&first[0], args.groups, run);
    const int row0  = off[group] + (run - first[group]) * slope_rows;
    const int row1  = row0 + slope_rows < off[group + 1] ? row0 + slope_rows : off[group + 1];
    const int lane  = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col   = (blockIdx.y * 64 + lane) * WIDTH;
    typedef InT in_t __attribute__((ext_vector_type(WIDTH)));
    float       sum[WIDTH];
#pragma unroll
    for(int v = 0; v < WIDTH; ++v)
    {
        sum[v] = 0.0f;
    }
    if(args.dz != nullptr && col >= args.cols && col < args.dz_pitch)
    {
        for(int row = row0 + wave; row < row1; row += 4)
        {
            static_cast<InT*>(args.dz)[(long long)row * args.dz_pitch + col] = to_out<InT>(0.0f);
        }
    }
    if(col < args.cols)
    {
#pragma unroll 8
        for(int row = row0 + wave; row < row1; row += 4)
        {
            const long long at = (long long)row * args.cols + col;
            in_t            d  = *reinterpret_cast<const in_t*>(static_cast<const InT*>(args.dc) + at);
            in_t            o;
            if(args.z != nullptr)
            {
                const in_t z = *reinterpret_cast<const in_t*>(static_cast<const InT*>(args.z) + at);
#pragma unroll
                for(int v = 0; v < WIDTH; ++v)
                {
                    const float g = (float)d[v] * activate_slope(args.act, (float)z[v]);
                    sum[v] += g; // (before it is rounded)
                    o[v] = to_out<InT>(g);
                }
            }
            else
            {
#pragma unroll
                for(int v = 0; v < WIDTH; ++v)
                {
                    sum[v] += (float)d[v];
                }
                o = d;
            }
            if(args.dz != nullptr)
            {
                *reinterpret_cast<in_t*>(static_cast<InT*>(args.dz) + (long long)row * args.dz_pitch + col) = o;
            }
        }
    }
    if(args.sums == nullptr)
    {
        return;
    }
#pragma unroll
    for(int v = 0; v < WIDTH; ++v)
    {
        part[wave][v * 64 + lane] = sum[v];
    }
    __syncthreads();
    for(int i = threadIdx.x; i < 64 * WIDTH; i += 256)
    {
        const int c = (blockIdx.y * 64 + i % 64) * WIDTH + i / 64;
        if(c < args.cols)
        {
            args.sums[(long long)run * args.cols + c] = ((part[0][i] + part[1][i]) + part[2][i]) + part[3][i];
        }
    }
}

// The sums of a group's runs: the gradient of its bias (blockIdx.y: the group).  Each of four waves
// adds up a quarter of the runs in their order, then the quarters are added in theirs.
template<class OutT>
__global__ void __launch_bounds__(256) column_sums(const slope_args args, OutT* __restrict__ dbias, int accumulate)
{
    __shared__ int   off[max_groups + 1], first[max_groups + 1];
    __shared__ float part[4][64];
    build_group_table(args.offsets, args.groups, args.rows, slope_rows, &off[0], &first[0]);
    const int group = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    const int run0 = first[group], runs = first[group + 1] - run0, each = (runs + 3) / 4;
    const int begin = run0 + wave * each, end = run0 + ((wave + 1) * each < runs ? (wave + 1) * each : runs);
    float     s = 0.0f;
    if(col < args.cols)
    {
#pragma unroll 8
        for(int run = begin; run < end; ++run)
        {
            s += args.sums[(long long)run * args.cols + col];
        }
    }
    part[wave][lane] = s;
    __syncthreads();
    if(wave == 0 && col < args.cols)
    {
        s        = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
        OutT& to = dbias[(long long)group * args.cols + col];
        to       = to_out<OutT>(accumulate ? s + (float)to : s);
    }
}

// ---------------------------------------------------------------------------
// Newton-Schulz steps: X is held twice, scaled by a power of two, padded with zeros to rows of multiples
// of 8 (and, where it is not tall, to a multiple of 8 of them): in fp32 (its linear term, see operators.hip) and in f16 (what is multiplied).
// ---------------------------------------------------------------------------
constexpr int square_parts = 1024; // the most workgroups that add up the squares of one matrix

// blockIdx.y: the matrix, blockIdx.x: one of `parts` runs of it.  One partial sum per workgroup, in a
// fixed order.  WIDTH elements at a time (16 bytes where the matrices are aligned, else one).
template<class GivenT, int WIDTH>
__global__ void __launch_bounds__(256) sum_squares(const GivenT* __restrict__ given, long long count,
                                                   float* __restrict__ parts)
{
    typedef GivenT given_t __attribute__((ext_vector_type(WIDTH)));
    const given_t* g    = reinterpret_cast<const given_t*>(given + blockIdx.y * count);
    const long long n   = count / WIDTH, hop = 256ll * gridDim.x;
    float           s[WIDTH];
#pragma unroll
    for(int v = 0; v < WIDTH; ++v)
    {
        s[v] = 0.0f;
    }
#pragma unroll 4
    for(long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += hop)
    {
        const given_t x = g[i];
#pragma unroll
        for(int v = 0; v < WIDTH; ++v)
        {
            s[v] += (float)x[v] * (float)x[v];
        }
    }
    float t = 0.0f;
#pragma unroll
    for(int v = 0; v < WIDTH; ++v)
    {
        t += s[v];
    }
#pragma unroll
    for(int d = 32; d > 0; d /= 2)
    {
        t += __shfl_xor(t, d);
    }
    __shared__ float wave_sum[4];
    if((threadIdx.x & 63) == 0)
    {
        wave_sum[threadIdx.x >> 6] = t;
    }
    __syncthreads();
    if(threadIdx.x == 0)
    {
        parts[blockIdx.y * square_parts + blockIdx.x] = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    }
}

// X = G scale / (|G| + epsilon), padded.  A thread writes 8 elements of a row at a time; WIDE: G's
// rows are whole pieces of 8 that start on 16 bytes.
template<class GivenT, bool WIDE>
__global__ void __launch_bounds__(256) orthogonal_start(const GivenT* __restrict__ given,
                                                        const float* __restrict__ parts,
                                                        float*    x32,
                                                        _Float16* x16,
                                                        int       rows,
                                                        int       cols,
                                                        int       rows_pad,
                                                        int       cols_pad,
                                                        float     scale,
                                                        float     epsilon,
                                                        int       used_parts)
{
    const long long matrix = blockIdx.y;
    float           t      = 0.0f;
    for(int i = threadIdx.x & 63; i < used_parts; i += 64)
    {
        t += parts[matrix * square_parts + i];
    }
#pragma unroll
    for(int d = 32; d > 0; d /= 2)
    {
        t += __shfl_xor(t, d);
    }
    const float   f      = scale / (sqrtf(t) + epsilon);
    const int     pieces = cols_pad / 8;
    const GivenT* g      = given + matrix * rows * cols;
    for(int row = blockIdx.x; row < rows_pad; row += gridDim.x)
    {
        for(int piece = threadIdx.x; piece < pieces; piece += 256)
        {
            typedef GivenT given8 __attribute__((ext_vector_type(8)));
            const int      col = piece * 8;
            float          y[8];
            if constexpr(WIDE)
            {
                const given8 v = *reinterpret_cast<const given8*>(g + (long long)row * cols + col);
#pragma unroll
                for(int e = 0; e < 8; ++e)
                {
                    y[e] = (float)v[e] * f;
                }
            }
            else
            {
#pragma unroll
                for(int e = 0; e < 8; ++e)
                {
                    y[e] = row < rows && col + e < cols ? (float)g[(long long)row * cols + col + e] * f : 0.0f;
                }
            }
            f16x8 h;
#pragma unroll
            for(int e = 0; e < 8; ++e)
            {
                h[e] = (_Float16)y[e];
            }
            const long long at = (matrix * rows_pad + row) * cols_pad + col;
            *reinterpret_cast<f32x4*>(x32 + at)     = f32x4{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<f32x4*>(x32 + at + 4) = f32x4{y[4], y[5], y[6], y[7]};
            *reinterpret_cast<f16x8*>(x16 + at)     = h;
        }
    }
}

// All steps of one small matrix (smaller side up to 64, larger up to 256) in one workgroup, in
// fp32 from LDS: X with the smaller side as its rows, S and Q.  One launch instead of seventeen, and
// nothing is rounded to f16: in a small matrix few roundings average out (8 x 8 with one strong
// direction: 4.8e-3 off by the f16 products, 1e-6 here).  A thread of the S and Q products owns 4 x 4
// elements, of the update whole columns of X, which depend on nothing but themselves and Q.
constexpr int small_side = 64, small_length = 256;

struct steps_args
{
    const void* given;
    void*       out;
    int         rows, cols; // of every matrix
    int         steps;
    float       a, b, c, epsilon;
};

template<class GivenT, class OutT>
__global__ void __launch_bounds__(256) orthogonal_small(const steps_args args)
{
    constexpr int XP = small_length + 1, SP = small_side + 4;
    __shared__ float x[small_side * XP];
    __shared__ float s[small_side * SP], q[small_side * SP];
    __shared__ float wave_sum[4];
    const int       tid  = threadIdx.x;
    const bool      tall = args.rows > args.cols;
    const int       l = tall ? args.cols : args.rows, h = tall ? args.rows : args.cols;
    const long long at = (long long)blockIdx.x * l * h;
    const GivenT*   g  = static_cast<const GivenT*>(args.given) + at;
    OutT*           o  = static_cast<OutT*>(args.out) + at;
    auto place = [&](int i) { return tall ? (i % l) * XP + i / l : (i / h) * XP + i % h; };

    float t = 0.0f;
    for(int i = tid; i < l * h; i += 256)
    {
        const float v = (float)g[i];
        x[place(i)]   = v;
        t += v * v;
    }
#pragma unroll
    for(int d = 32; d > 0; d /= 2)
    {
        t += __shfl_xor(t, d);
    }
    if((tid & 63) == 0)
    {
        wave_sum[tid >> 6] = t;
    }
    __syncthreads();
    const float f = 1.0f / (sqrtf((wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3])) + args.epsilon);
    for(int i = tid; i < l * h; i += 256)
    {
        x[place(i)] *= f;
    }
    const int ti = tid / 16 * 4, tj = tid % 16 * 4; // this thread's 4 x 4 elements of S and Q
    for(int step = 0; step < args.steps; ++step)
    {
        __syncthreads();
        if(ti < l && tj < l)
        {
            float acc[4][4] = {};
            for(int k = 0; k < h; ++k)
            {
                float u[4], v[4];
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    // (rows past l: read as row 0, their sums are not stored)
                    u[e] = x[(ti + e < l ? ti + e : 0) * XP + k];
                    v[e] = x[(tj + e < l ? tj + e : 0) * XP + k];
                }
#pragma unroll
                for(int e = 0; e < 16; ++e)
                {
                    acc[e / 4][e % 4] += u[e / 4] * v[e % 4];
                }
            }
#pragma unroll
            for(int e = 0; e < 16; ++e)
            {
                s[(ti + e / 4) * SP + tj + e % 4] = ti + e / 4 < l && tj + e % 4 < l ? acc[e / 4][e % 4] : 0.0f;
            }
        }
        __syncthreads();
        if(ti < l && tj < l)
        {
            float acc[4][4] = {};
            for(int k = 0; k < l; ++k)
            {
                // (S is its own transpose: row k holds what column k does)
                const f32x4 u = *reinterpret_cast<const f32x4*>(&s[k * SP + ti]);
                const f32x4 v = *reinterpret_cast<const f32x4*>(&s[k * SP + tj]);
#pragma unroll
                for(int e = 0; e < 16; ++e)
                {
                    acc[e / 4][e % 4] += u[e / 4] * v[e % 4];
                }
            }
#pragma unroll
            for(int e = 0; e < 16; ++e)
            {
                const int to = (ti + e / 4) * SP + tj + e % 4;
                q[to]        = args.b * s[to] + args.c * acc[e / 4][e % 4];
            }
        }
        __syncthreads();
        for(int col = tid; col < h; col += 256)
        {
            float acc[small_side];
#pragma unroll
            for(int i = 0; i < small_side; ++i)
            {
                acc[i] = 0.0f;
            }
            for(int k = 0; k < l; ++k)
            {
                const float v = x[k * XP + col];
#pragma unroll
                for(int i = 0; i < small_side; i += 4)
                {
                    if(i < l)
                    {
                        const f32x4 u = *reinterpret_cast<const f32x4*>(&q[k * SP + i]);
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            acc[i + e] += u[e] * v;
                        }
                    }
                }
            }
#pragma unroll
            for(int i = 0; i < small_side; ++i)
            {
                if(i < l)
                {
                    x[i * XP + col] = args.a * x[i * XP + col] + acc[i];
                }
            }
        }
    }
    __syncthreads();
    for(int i = tid; i < l * h; i += 256)
    {
        o[i] = to_out<OutT>(x[place(i)]);
    }
}

// The finished update from its padded form (where rows and columns are no multiples of 8).
template<class OutT>
__global__ void __launch_bounds__(256) orthogonal_end(const OutT* __restrict__ padded, OutT* __restrict__ out, int rows,
                                                      int cols, int rows_pad, int cols_pad)
{
    const long long matrix = blockIdx.y;
    for(int row = blockIdx.x; row < rows; row += gridDim.x)
    {
        for(int col = threadIdx.x; col < cols; col += 256)
        {
            out[(matrix * rows + row) * cols + col] = padded[(matrix * rows_pad + row) * cols_pad + col];
        }
    }
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_POINTWISE_HPP
