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

// dZ = dC * act'(Z), and the sums of its columns over runs of slope_rows rows of a group.  dZ is rounded to A's
// type, as both products need it: the matrix cores' 16-bit rate takes 16-bit operands, and one for its upper
// and one for its lower half would double the products.  It costs 2.3e-3 of a bf16 gradient's norm against 1.7e-3
// for the rounding of the result alone.  The sums are of the values before that rounding.  4096 x 5120 bf16: 29 us,
// 4.35 TB/s; 8192 x 4096 in 16 groups 52 us, 3.9 TB/s.  Runs of 16 or 64 rows and non-temporal loads change
// a backward pass by less than 2 %, up for some sizes and down for others.
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
    int         run0, block0; // the launch's first run and block of columns: a grid holds fewer than there can be
};

// A wave takes 64 * WIDTH columns (blockIdx.y), the four waves of a workgroup every fourth row of a run
// (blockIdx.x); WIDTH = 8 where rows start on 16 bytes, else 1.  The sums of a run are added in
// the order of its rows within a wave, then in wave order: the same in every call.
template<class InT, int WIDTH>
__global__ void __launch_bounds__(256) activation_slope(const slope_args args)
{
    __shared__ int   off[max_groups + 1], first[max_groups + 1];
    __shared__ float part[4][64 * WIDTH];
    build_group_table(args.offsets, args.groups, args.rows, slope_rows, &off[0], &first[0]);
    const int run = args.run0 + blockIdx.x;
    if(run >= first[args.groups])
    {
        return;
    }
    const int group = group_of_tile(&first[0], args.groups, run);
    const int row0  = off[group] + (run - first[group]) * slope_rows;
    const int row1  = row0 + slope_rows < off[group + 1] ? row0 + slope_rows : off[group + 1];
    const int lane  = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int block = args.block0 + blockIdx.y, col = (block * 64 + lane) * WIDTH;
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
        const int c = (block * 64 + i % 64) * WIDTH + i / 64;
        if(c < args.cols)
        {
            args.sums[(long long)run * args.cols + c] = ((part[0][i] + part[1][i]) + part[2][i]) + part[3][i];
        }
    }
}

// The sums of a group's runs: the gradient of its bias (blockIdx.y: the group, blockIdx.x: 64 columns).  Each of four waves
// adds up a quarter of the runs in their order, then the quarters are added in theirs.
template<class OutT>
__global__ void __launch_bounds__(256) column_sums(const slope_args args, OutT* __restrict__ dbias, int accumulate)
{
    __shared__ int   off[max_groups + 1], first[max_groups + 1];
    __shared__ float part[4][64];
    build_group_table(args.offsets, args.groups, args.rows, slope_rows, &off[0], &first[0]);
    const int group = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = (args.block0 + blockIdx.x) * 64 + lane;
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
// Newton-Schulz steps: X has the smaller side as its rows (a tall G is transposed on the way in and
// out) and is held twice, scaled by a power of two, padded with zeros to multiples of 8: in fp32
// (its linear term, see operators.hip) and in f16 (what is multiplied).
// ---------------------------------------------------------------------------
constexpr int square_parts = 1024; // the most workgroups that add up the squares of one matrix

// blockIdx.y: the matrix, blockIdx.x: one of `parts` runs of it.  One partial sum per workgroup, in a
// fixed order.  WIDTH elements at a time (16 bytes where the matrices are aligned, else one).  In fp64, as the
// norm and the factor made of it: the square of an fp32 or bf16 element may lie outside fp32's range.
template<class GivenT, int WIDTH>
__global__ void __launch_bounds__(256) sum_squares(const GivenT* __restrict__ given, long long count,
                                                   double* __restrict__ parts)
{
    typedef GivenT given_t __attribute__((ext_vector_type(WIDTH)));
    const given_t* g    = reinterpret_cast<const given_t*>(given + blockIdx.y * count);
    const long long n   = count / WIDTH, hop = 256ll * gridDim.x;
    double          s[WIDTH];
#pragma unroll
    for(int v = 0; v < WIDTH; ++v)
    {
        s[v] = 0.0;
    }
#pragma unroll 4
    for(long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += hop)
    {
        const given_t x = g[i];
#pragma unroll
        for(int v = 0; v < WIDTH; ++v)
        {
            s[v] += (double)x[v] * (double)x[v];
        }
    }
    double t = 0.0;
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
    __shared__ double wave_sum[4];
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

// The norm of a matrix from its partial sums, by every wave.
__device__ __forceinline__ double norm_of(const double* parts, long long matrix, int used_parts)
{
    double t = 0.0;
    for(int i = threadIdx.x & 63; i < used_parts; i += 64)
    {
        t += parts[matrix * square_parts + i];
    }
#pragma unroll
    for(int d = 32; d > 0; d /= 2)
    {
        t += __shfl_xor(t, d);
    }
    return sqrt(t);
}

struct start_args
{
    const void*   given;
    const double* parts;
    float*       x32;
    _Float16*    x16;
    int          rows, cols; // of G
    int          rows_pad, cols_pad; // of X
    float        scale, epsilon;
    int          used_parts;
};

__device__ __forceinline__ void store_start(const start_args& args, long long at, const float (&y)[8])
{
    f16x8 h;
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        h[e] = (_Float16)y[e];
    }
    *reinterpret_cast<f32x4*>(args.x32 + at)     = f32x4{y[0], y[1], y[2], y[3]};
    *reinterpret_cast<f32x4*>(args.x32 + at + 4) = f32x4{y[4], y[5], y[6], y[7]};
    *reinterpret_cast<f16x8*>(args.x16 + at)     = h;
}

// X = G scale / (|G| + epsilon), padded (blockIdx.y: the matrix).  A thread writes 8 elements of a row at a time;
// WIDE: G needs no padding and its rows are whole pieces of 8 that start on 16 bytes.
template<class GivenT, bool WIDE>
__global__ void __launch_bounds__(256) orthogonal_start(const start_args args)
{
    const long long matrix = blockIdx.y;
    const double    f      = args.scale / (norm_of(args.parts, matrix, args.used_parts) + args.epsilon);
    const int       pieces = args.cols_pad / 8;
    const GivenT*   g      = static_cast<const GivenT*>(args.given) + matrix * args.rows * args.cols;
    for(int row = blockIdx.x; row < args.rows_pad; row += gridDim.x)
    {
        for(int piece = threadIdx.x; piece < pieces; piece += 256)
        {
            typedef GivenT given8 __attribute__((ext_vector_type(8)));
            const int      col = piece * 8;
            float          y[8];
            if constexpr(WIDE)
            {
                const given8 v = *reinterpret_cast<const given8*>(g + (long long)row * args.cols + col);
#pragma unroll
                for(int e = 0; e < 8; ++e)
                {
                    y[e] = (float)((double)v[e] * f);
                }
            }
            else
            {
#pragma unroll
                for(int e = 0; e < 8; ++e)
                {
                    y[e] = row < args.rows && col + e < args.cols ? (float)((double)g[(long long)row * args.cols + col + e] * f)
                                                                        : 0.0f;
                }
            }
            store_start(args, (matrix * args.rows_pad + row) * args.cols_pad + col, y);
        }
    }
}

// The same for a tall G: X is its transpose.  A workgroup turns 64 x 64 elements round in LDS
// (blockIdx.x: tiles of X, row by row of tiles).
template<class GivenT>
__global__ void __launch_bounds__(256) orthogonal_start_tall(const start_args args)
{
    __shared__ float tile[64][65];
    const long long  matrix = blockIdx.y;
    const double     f      = args.scale / (norm_of(args.parts, matrix, args.used_parts) + args.epsilon);
    const GivenT*    g      = static_cast<const GivenT*>(args.given) + matrix * args.rows * args.cols;
    const int        across = (args.cols_pad + 63) / 64;
    const int        x_row0 = blockIdx.x / across * 64, x_col0 = blockIdx.x % across * 64;
    for(int i = threadIdx.x; i < 64 * 64; i += 256)
    {
        const int row = x_col0 + i / 64, col = x_row0 + i % 64; // of G
        tile[i % 64][i / 64] = row < args.rows && col < args.cols ? (float)((double)g[(long long)row * args.cols + col] * f) : 0.0f;
    }
    __syncthreads();
    for(int i = threadIdx.x; i < 64 * 8; i += 256)
    {
        const int row = i / 8, col = i % 8 * 8;
        if(x_row0 + row < args.rows_pad && x_col0 + col < args.cols_pad)
        {
            float y[8];
#pragma unroll
            for(int e = 0; e < 8; ++e)
            {
                y[e] = tile[row][col + e];
            }
            store_start(args, (matrix * args.rows_pad + x_row0 + row) * args.cols_pad + x_col0 + col, y);
        }
    }
}

// The finished update (rows x cols) from its padded form.
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

// The same where the update is tall: out = X^T, X of cols rows padded to rows_pad x cols_pad.
template<class OutT>
__global__ void __launch_bounds__(256) orthogonal_end_tall(const OutT* __restrict__ padded, OutT* __restrict__ out,
                                                           int rows, int cols, int rows_pad, int cols_pad)
{
    __shared__ OutT tile[64][66];
    const long long matrix = blockIdx.y;
    const int       across = (cols + 63) / 64, row0 = blockIdx.x / across * 64, col0 = blockIdx.x % across * 64; // of out
    for(int i = threadIdx.x; i < 64 * 64; i += 256)
    {
        const int xr = col0 + i / 64, xc = row0 + i % 64;
        if(xr < rows_pad && xc < cols_pad)
        {
            tile[i % 64][i / 64] = padded[(matrix * rows_pad + xr) * cols_pad + xc];
        }
    }
    __syncthreads();
    for(int i = threadIdx.x; i < 64 * 64; i += 256)
    {
        const int row = row0 + i / 64, col = col0 + i % 64;
        if(row < rows && col < cols)
        {
            out[(matrix * rows + row) * cols + col] = tile[i / 64][i % 64];
        }
    }
}

// All steps of one small matrix (smaller side up to 64, larger up to 256) in one workgroup, in
// fp32 on the matrix cores (v_mfma_f32_16x16x4_f32), from LDS: X with the smaller side as its rows, and S,
// then Q, in one buffer; rows and columns past the matrix are zeros throughout.  One launch instead of
// seventeen, and nothing is rounded to f16: in a small matrix few roundings average out (8 x 8 with
// one strong direction: 4.8e-3 off by the f16 products, 1e-6 here).  Five steps of 64 x 64 take 29 us,
// of 64 x 256 63 us (16 of them; 512 136).  Wave w of sixteen owns tile
// (w / 4, w mod 4) of S and Q, and of X the tiles (w mod 4, w / 4 + 4 i).  Pitches of 4 mod 64 floats spread the
// 16 rows x 4 columns that a fragment read touches over all 64 banks.  Bound by the latency of LDS
// and the matrix cores' fp32 rate; past 256 columns the seventeen launches are as fast.
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
__global__ void __launch_bounds__(1024) orthogonal_small(const steps_args args)
{
    constexpr int XP = small_length + 4, SP = small_side + 4, THREADS = 1024, COLS = small_length / 16 / 4;
    __shared__ float x[small_side * XP];
    __shared__ float s[small_side * SP];
    __shared__ double wave_sum[16];
    const int       tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, k4 = lane >> 4;
    const int       wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool      tall = args.rows > args.cols;
    const int       l = tall ? args.cols : args.rows, h = tall ? args.rows : args.cols;
    const int       l16 = (l + 15) / 16 * 16, h16 = (h + 15) / 16 * 16;
    const long long at = (long long)blockIdx.x * l * h;
    const GivenT*   g  = static_cast<const GivenT*>(args.given) + at;
    OutT*           o  = static_cast<OutT*>(args.out) + at;
    auto place = [&](int i) { return tall ? (i % l) * XP + i / l : (i / h) * XP + i % h; };

    for(int i = tid; i < small_side * XP; i += THREADS)
    {
        x[i] = 0.0f;
    }
    __syncthreads();
    double t = 0.0;
    for(int i = tid; i < l * h; i += THREADS)
    {
        const float v = (float)g[i];
        x[place(i)]   = v;
        t += (double)v * (double)v;
    }
#pragma unroll
    for(int d = 32; d > 0; d /= 2)
    {
        t += __shfl_xor(t, d);
    }
    if(lane == 0)
    {
        wave_sum[wave] = t;
    }
    __syncthreads();
    t = 0.0;
#pragma unroll
    for(int w = 0; w < 16; ++w)
    {
        t += wave_sum[w];
    }
    const double f = 1.0 / (sqrt(t) + args.epsilon);
    for(int i = tid; i < l * h; i += THREADS)
    {
        float& to = x[place(i)];
        to        = (float)((double)to * f);
    }
    const int ti = wave >> 2, tj = wave & 3;
    float*    own = &s[(ti * 16 + 4 * k4) * SP + tj * 16 + r16]; // this lane's 4 rows of its tile of S
    const bool used = ti * 16 < l16 && tj * 16 < l16; // (the others' tiles are zeros)
    for(int step = 0; step < args.steps; ++step)
    {
        __syncthreads();
        // S = X X^T
        f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
        if(used)
        {
            for(int k0 = 0; k0 < h16; k0 += 16)
            {
#pragma unroll
                for(int k = k0; k < k0 + 16; k += 4)
                {
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[(ti * 16 + r16) * XP + k + k4],
                                                               x[(tj * 16 + r16) * XP + k + k4], acc, 0, 0, 0);
                }
            }
        }
#pragma unroll
        for(int v = 0; v < 4; ++v)
        {
            own[v * SP] = acc[v];
        }
        __syncthreads();
        // Q = b S + c S^2 (S is its own transpose: column j of it is row j)
        f32x4 q{0.0f, 0.0f, 0.0f, 0.0f};
        if(used)
        {
            for(int k0 = 0; k0 < l16; k0 += 16)
            {
#pragma unroll
                for(int k = k0; k < k0 + 16; k += 4)
                {
                    q = __builtin_amdgcn_mfma_f32_16x16x4f32(s[(ti * 16 + r16) * SP + k + k4],
                                                             s[(tj * 16 + r16) * SP + k + k4], q, 0, 0, 0);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for(int v = 0; v < 4; ++v)
        {
            own[v * SP] = args.b * acc[v] + args.c * q[v];
        }
        __syncthreads();
        // X = a X + Q X: every tile is read before any is written
        f32x4 y[COLS];
#pragma unroll
        for(int i = 0; i < COLS; ++i)
        {
            y[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const int rows = tj * 16;
        if(rows < l16)
        {
            for(int k0 = 0; k0 < l16; k0 += 16)
            {
                float u[4];
#pragma unroll
                for(int k = 0; k < 4; ++k)
                {
                    u[k] = s[(rows + r16) * SP + k0 + 4 * k + k4];
                }
#pragma unroll
                for(int i = 0; i < COLS; ++i)
                {
                    const int cols = (ti + 4 * i) * 16;
                    if(cols < h16)
                    {
#pragma unroll
                        for(int k = 0; k < 4; ++k)
                        {
                            y[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[k], x[(k0 + 4 * k + k4) * XP + cols + r16], y[i], 0,
                                                                        0, 0);
                        }
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for(int i = 0; i < COLS; ++i)
        {
#pragma unroll
            for(int v = 0; v < 4; ++v)
            {
                float& to = x[(rows + 4 * k4 + v) * XP + (ti + 4 * i) * 16 + r16];
                to        = args.a * to + y[i][v];
            }
        }
    }
    __syncthreads();
    for(int i = tid; i < l * h; i += THREADS)
    {
        o[i] = to_out<OutT>(x[place(i)]);
    }
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_POINTWISE_HPP
