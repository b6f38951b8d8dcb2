// The kernels between the products of a projection onto a vocabulary and its loss: softmax statistics of pieces of
// the logits, the loss by row, the gradient of the logits.
//
// Mathematics, for a row with logits x = z / T (T: the temperature, 1 for cross entropy), lse = log sum_v e^x_v and a
// wanted distribution q (of the target alone, or the softmax of a teacher's listed logits over T):
//   loss = T^2 sum_v q_v (log q_v - x_v + lse), d loss / d z_v = T (e^(x_v - lse) - q_v).
// A part of a row leaves its largest x and its sum of e^(x - largest); the parts of a row are joined by one wave in
// a fixed order, in fp32.
#ifndef ROCM_WMMA_GEMM_HEAD_LOSS_HPP
#define ROCM_WMMA_GEMM_HEAD_LOSS_HPP

#include "product_common.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

constexpr int most_entries = 256; // that a row's list may have
constexpr int part_cols = 4096; // of a row that a workgroup reads for its statistics

// What a row is compared with: its target, or a list of entries with a teacher's logits.
struct wanted_args
{
    const void*  entries; // rows x k indices
    int          wide; // 1: of 64 bits
    const float* teacher; // rows x k, nullptr: a target (k = 1)
    long long    vocabulary;
    int          rows, k;
    float        scale; // 1 / T
};

// Entry j of a row, -1 where it lies outside the vocabulary.
__device__ __forceinline__ long long entry_of(const wanted_args& w, long long at)
{
    const long long v = w.wide ? static_cast<const long long*>(w.entries)[at] : (long long)static_cast<const int*>(w.entries)[at];
    return v >= 0 && v < w.vocabulary ? v : -1;
}

// Joins two parts' (largest, sum).
__device__ __forceinline__ void join_part(float& top, float& sum, float other_top, float other_sum)
{
    const float most = __builtin_fmaxf(top, other_top);
    // (a part without a finite value: e^(-inf - -inf) would be no number)
    sum = (top == most ? sum : sum * expf(top - most)) + (other_top == most ? other_sum : other_sum * expf(other_top - most));
    top = most;
}

template<int LANES>
__device__ __forceinline__ float sum_of_lanes(float v)
{
#pragma unroll
    for(int d = 1; d < LANES; d *= 2)
    {
        v += __shfl_xor(v, d);
    }
    return v;
}

// The statistics of part blockIdx.y of row blockIdx.x: 256 threads, four columns at a time.
struct part_args
{
    const float* z; // rows x pitch
    float2*      parts; // rows x all
    long long    pitch;
    int          cols, part0, all;
    float        scale;
};

__global__ void __launch_bounds__(256) softmax_parts(const part_args args)
{
    __shared__ float2  of_wave[4];
    const long long    row   = blockIdx.x;
    const int          begin = blockIdx.y * part_cols, end = args.cols - begin < part_cols ? args.cols : begin + part_cols;
    const float* const z     = args.z + row * args.pitch;
    float              x[part_cols / 256];
    float              top = -__builtin_inff();
#pragma unroll
    for(int i = 0; i < part_cols / 1024; ++i)
    {
        const int col = begin + i * 1024 + threadIdx.x * 4;
        f32x4     v   = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        if(col < end)
        {
            v = *reinterpret_cast<const f32x4*>(z + col); // (rows are padded to whole pieces)
        }
#pragma unroll
        for(int e = 0; e < 4; ++e)
        {
            x[4 * i + e] = col + e < end ? v[e] * args.scale : -__builtin_inff();
            top          = __builtin_fmaxf(top, x[4 * i + e]);
        }
    }
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
    {
        top = __builtin_fmaxf(top, __shfl_xor(top, d));
    }
    const float from = top > -__builtin_inff() ? top : 0.0f;
    float       sum  = 0.0f;
#pragma unroll
    for(int i = 0; i < part_cols / 256; ++i)
    {
        sum += expf(x[i] - from);
    }
    sum = sum_of_lanes<64>(sum);
    if((threadIdx.x & 63) == 0)
    {
        of_wave[threadIdx.x >> 6] = {top, sum};
    }
    __syncthreads();
    if(threadIdx.x == 0)
    {
#pragma unroll
        for(int w = 1; w < 4; ++w)
        {
            join_part(top, sum, of_wave[w].x, of_wave[w].y);
        }
        args.parts[row * args.all + args.part0 + blockIdx.y] = {top, sum};
    }
}

// The listed logits that lie in a piece; on the first piece, 0 for entries outside the vocabulary.
__global__ void __launch_bounds__(256)
    pick_entries(const wanted_args w, const float* __restrict__ z, long long pitch, long long col0, int cols, float* __restrict__ picked)
{
    const long long total = (long long)w.rows * w.k;
    for(long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long long)gridDim.x * 256)
    {
        const long long v = entry_of(w, at);
        if(v >= col0 && v < col0 + cols)
        {
            picked[at] = z[at / w.k * pitch + (v - col0)];
        }
        else if(v < 0 && col0 == 0)
        {
            picked[at] = 0.0f;
        }
    }
}

// A teacher's distribution over a row's list, a wave a row: q of entries lane, lane + 64, ...; the largest logit and the
// sum, 0 where the list is empty.
constexpr int list_rounds = most_entries / 64;
struct listed_row
{
    long long entry[list_rounds];
    float     x[list_rounds]; // the teacher's logit over T, less the row's largest
    float     e[list_rounds]; // its exponential
    float     sum;
};

__device__ __forceinline__ listed_row read_list(const wanted_args& w, long long row)
{
    const int  lane = threadIdx.x & 63;
    listed_row l;
    float      top = -__builtin_inff();
#pragma unroll
    for(int r = 0; r < list_rounds; ++r)
    {
        const int j = r * 64 + lane;
        l.entry[r]  = j < w.k ? entry_of(w, row * w.k + j) : -1;
        l.x[r]      = l.entry[r] >= 0 ? w.teacher[row * w.k + j] * w.scale : -__builtin_inff();
        top         = __builtin_fmaxf(top, l.x[r]);
    }
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
    {
        top = __builtin_fmaxf(top, __shfl_xor(top, d));
    }
    top   = top > -__builtin_inff() ? top : 0.0f; // (an empty list, or one of -infinity: the sum is 0)
    l.sum = 0.0f;
#pragma unroll
    for(int r = 0; r < list_rounds; ++r)
    {
        l.x[r] -= top;
        l.e[r] = l.entry[r] >= 0 ? expf(l.x[r]) : 0.0f;
        l.sum += l.e[r];
    }
    l.sum = sum_of_lanes<64>(l.sum);
    return l;
}

struct join_args
{
    wanted_args   want;
    const float2* parts; // rows x all
    const float*  picked; // rows x k
    float*        loss;
    float*        lse;
    int           all;
};

// The loss of a row from its parts: a wave a row.
__global__ void __launch_bounds__(256) join_rows(const join_args args)
{
    const int lane = threadIdx.x & 63;
    for(long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < args.want.rows; row += (long long)gridDim.x * 4)
    {
        float top = -__builtin_inff(), sum = 0.0f;
        for(int p = lane; p < args.all; p += 64)
        {
            const float2 part = args.parts[row * args.all + p];
            join_part(top, sum, part.x, part.y);
        }
#pragma unroll
        for(int d = 1; d < 64; d *= 2)
        {
            const float t = __shfl_xor(top, d), s = __shfl_xor(sum, d);
            join_part(top, sum, t, s);
        }
        const float rest = logf(sum), lse = top + rest;
        float       loss = 0.0f;
        if(args.want.teacher == nullptr)
        {
            // (what lies between the largest logit and the target first: it is exact where the two are near)
            loss = entry_of(args.want, row) >= 0 ? (top - args.picked[row]) + rest : 0.0f;
        }
        else
        {
            const listed_row l = read_list(args.want, row);
            const float      norm = l.sum > 0.0f ? 1.0f / l.sum : 0.0f, log_norm = l.sum > 0.0f ? logf(l.sum) : 0.0f;
#pragma unroll
            for(int r = 0; r < list_rounds; ++r)
            {
                const int   j = r * 64 + lane;
                const float q = l.e[r] * norm;
                if(q > 0.0f || q != q)
                {
                    loss += q * ((l.x[r] - log_norm) + ((top - args.picked[row * args.want.k + j] * args.want.scale) + rest));
                }
            }
            loss = sum_of_lanes<64>(loss) / (args.want.scale * args.want.scale);
        }
        if(lane == 0)
        {
            args.lse[row]  = lse;
            args.loss[row] = loss;
        }
    }
}

// ------------------------------------------------------------------ the gradient

// What every row's gradient is multiplied by: the loss's gradient times T, times a power of two that brings the largest to
// 2^13 .. 2^14 where the logits' gradient is held in f16 (whose range ends at 6e-5 below and at 65504 above; p - q is at most 1),
// 0 for a row that is compared with nothing.  unit[0]: that power of two, unit[1]: 1 over it.
struct factor_args
{
    wanted_args  want;
    const float* dloss;
    float*       factor;
    float*       unit;
    int          scaled; // 0: the power of two is 1
};

// (one workgroup: the largest of all rows)
__global__ void __launch_bounds__(1024) gradient_unit(const factor_args args)
{
    __shared__ float of_wave[16];
    float            most = 0.0f;
#pragma unroll 8
    for(int row = threadIdx.x; row < args.want.rows; row += 1024)
    {
        const float d = __builtin_fabsf(args.dloss[row] / args.want.scale);
        most          = d > most && d < __builtin_inff() ? d : most;
    }
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
    {
        most = __builtin_fmaxf(most, __shfl_xor(most, d));
    }
    if((threadIdx.x & 63) == 0)
    {
        of_wave[threadIdx.x >> 6] = most;
    }
    __syncthreads();
    if(threadIdx.x == 0)
    {
        for(int w = 1; w < 16; ++w)
        {
            most = __builtin_fmaxf(most, of_wave[w]);
        }
        // (both the power and 1 over it are fp32 numbers)
        int up = most > 0.0f ? 13 - ilogbf(most) : 0;
        up     = up > 120 ? 120 : up < -120 ? -120 : up;
        args.unit[0] = args.scaled ? ldexpf(1.0f, up) : 1.0f;
        args.unit[1] = args.scaled ? ldexpf(1.0f, -up) : 1.0f;
    }
}

// A wave a row (a list has to be looked through for an entry).
__global__ void __launch_bounds__(256) gradient_factors(const factor_args args)
{
    const int lane = threadIdx.x & 63;
    for(long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < args.want.rows; row += (long long)gridDim.x * 4)
    {
        bool is;
        if(args.want.teacher == nullptr)
        {
            is = entry_of(args.want, row) >= 0;
        }
        else
        {
            const float sum = read_list(args.want, row).sum;
            is              = sum > 0.0f || sum != sum;
        }
        if(lane == 0)
        {
            args.factor[row] = is ? args.dloss[row] / args.want.scale * (args.scaled ? args.unit[0] : 1.0f) : 0.0f;
        }
    }
}

struct softmax_slope_args
{
    wanted_args  want;
    const float* z; // rows x pitch
    void*        dz; // rows x pitch
    long long    pitch; // a multiple of 8
    long long    col0; // of the piece in the vocabulary
    int          cols; // columns past them are written as zeros
    const float* lse;
    const float* factor;
    const float* picked; // rows x k (a list)
};

// dz = factor (e^(x - lse) - q), 8 columns a thread; q of a target alone (a list's entries are put right by listed_slope).
template<class InT>
__global__ void __launch_bounds__(256) softmax_slope(const softmax_slope_args args)
{
    typedef InT     in8 __attribute__((ext_vector_type(8)));
    const long long row = blockIdx.x;
    const int       col = (blockIdx.y * 256 + threadIdx.x) * 8;
    if(col >= args.pitch)
    {
        return;
    }
    const float  factor = args.factor[row], lse = args.lse[row];
    const float* z      = args.z + row * args.pitch + col;
    const f32x4  lo = *reinterpret_cast<const f32x4*>(z), hi = *reinterpret_cast<const f32x4*>(z + 4);
    long long    target = -1;
    if(args.want.teacher == nullptr)
    {
        target = entry_of(args.want, row) - args.col0;
    }
    in8 o;
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        const float p = expf((e < 4 ? lo[e & 3] : hi[e & 3]) * args.want.scale - lse);
        const float d = factor * (p - (target == col + e ? 1.0f : 0.0f));
        o[e]          = to_out<InT>(factor == 0.0f || col + e >= args.cols ? 0.0f : d);
    }
    *reinterpret_cast<in8*>(static_cast<InT*>(args.dz) + row * args.pitch + col) = o;
}

// The listed entries of a piece: factor (e^(x - lse) - q), from the logits that the loss picked; q of an entry that is
// listed more than once is the sum of its q, in the order of the list, and each of them writes the same.  A wave a row.
template<class InT>
__global__ void __launch_bounds__(256) listed_slope(const softmax_slope_args args)
{
    __shared__ long long entries[4][most_entries];
    __shared__ float     shares[4][most_entries];
    const int            lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int            k    = args.want.k;
    const long long      step = (long long)gridDim.x * 4;
    // (every wave makes the same number of rounds, for the barriers)
    for(long long first = (long long)blockIdx.x * 4; first < args.want.rows; first += step)
    {
        const long long row    = first + wave;
        const bool      is     = row < args.want.rows;
        const float     factor = is ? args.factor[row] : 0.0f;
        if(is)
        {
            const listed_row l    = read_list(args.want, row);
            const float      norm = l.sum > 0.0f ? 1.0f / l.sum : l.sum;
#pragma unroll
            for(int r = 0; r < list_rounds; ++r)
            {
                entries[wave][r * 64 + lane] = l.entry[r];
                shares[wave][r * 64 + lane]  = l.e[r] * norm;
            }
        }
        __syncthreads();
        if(factor != 0.0f)
        {
            const float lse = args.lse[row];
            for(int j = lane; j < k; j += 64)
            {
                const long long v = entries[wave][j];
                if(v >= args.col0 && v < args.col0 + args.cols)
                {
                    float q = 0.0f;
                    for(int i = 0; i < k; ++i)
                    {
                        q += entries[wave][i] == v ? shares[wave][i] : 0.0f;
                    }
                    const float p = expf(args.picked[row * k + j] * args.want.scale - lse);
                    static_cast<InT*>(args.dz)[row * args.pitch + (v - args.col0)] = to_out<InT>(factor * (p - q));
                }
            }
        }
        __syncthreads();
    }
}

// out (rows of `cols` elements, `out_pitch` apart) = from (pitch apart) * unit, added to what is there or not.
template<class OutT>
__global__ void __launch_bounds__(256)
    scaled_rows(const float* __restrict__ from, long long pitch, OutT* out, long long out_pitch, long long rows, long long cols,
                const float* __restrict__ unit, int add)
{
    const float     by     = unit != nullptr ? *unit : 1.0f;
    const long long pieces = (cols + 3) / 4, total = rows * pieces; // (from's rows are padded to whole pieces)
    const bool      whole  = cols % 4 == 0 && out_pitch % 4 == 0 && reinterpret_cast<unsigned long long>(out) % (4 * sizeof(OutT)) == 0;
    typedef OutT    out4 __attribute__((ext_vector_type(4)));
    for(long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long long)gridDim.x * 256)
    {
        const long long row = at / pieces, col = (at - row * pieces) * 4;
        const f32x4     v   = *reinterpret_cast<const f32x4*>(from + row * pitch + col);
        OutT* const     to  = out + row * out_pitch + col;
        if(whole)
        {
            out4 o = add ? *reinterpret_cast<const out4*>(to) : out4{};
#pragma unroll
            for(int e = 0; e < 4; ++e)
            {
                o[e] = to_out<OutT>(add ? (float)o[e] + v[e] * by : v[e] * by);
            }
            *reinterpret_cast<out4*>(to) = o;
            continue;
        }
#pragma unroll
        for(int e = 0; e < 4; ++e)
        {
            if(col + e < cols)
            {
                to[e] = to_out<OutT>(add ? (float)to[e] + v[e] * by : v[e] * by);
            }
        }
    }
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_HEAD_LOSS_HPP
