// The kernels between the products of a projection onto a vocabulary and its loss: softmax statistics of pieces of
// the logits, the loss by row, the gradient of the logits.
//
// Mathematics, for a row with logits x = z / T (T: the temperature, 1 for cross entropy), lse = log sum_v e^x_v and a
// wanted distribution q (of the target alone, or the softmax of a teacher's listed logits over T):
//   loss = T^2 sum_v q_v (log q_v - x_v + lse), d loss / d z_v = T (e^(x_v - lse) - q_v).
// Powers are of 2, which the hardware has: x log2(e) = scale2 z.  A part of a row leaves its largest such number and the sum of
// 2^(number - largest) (softmax_part); the parts of a row are joined by one wave in a fixed order, in fp32.
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
    float        scale, scale2; // 1 / T, log2(e) / T
};

constexpr float log2_of_e = 1.4426950408889634f, log_of_2 = 0.6931471805599453f;

// Entry j of a row, -1 where it lies outside the vocabulary.
__device__ __forceinline__ long long entry_of(const wanted_args& w, long long at)
{
    const long long v = w.wide ? static_cast<const long long*>(w.entries)[at] : (long long)static_cast<const int*>(w.entries)[at];
    return v >= 0 && v < w.vocabulary ? v : -1;
}

// Joins two parts.
__device__ __forceinline__ softmax_part joined(softmax_part a, softmax_part b)
{
    const float most = __builtin_fmaxf(a.top, b.top);
    // (a part without a finite value: 2^(-inf - -inf) would be no number)
    return {most, (a.top == most ? a.sum : a.sum * __builtin_amdgcn_exp2f(a.top - most))
                      + (b.top == most ? b.sum : b.sum * __builtin_amdgcn_exp2f(b.top - most))};
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
    const float*  z; // rows x pitch
    softmax_part* parts; // rows x all
    long long     pitch;
    int           cols, part0, all;
    float         scale2;
};

__global__ void __launch_bounds__(256) softmax_parts(const part_args args)
{
    __shared__ softmax_part of_wave[4];
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
            x[4 * i + e] = col + e < end ? v[e] * args.scale2 : -__builtin_inff();
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
        sum += __builtin_amdgcn_exp2f(x[i] - from);
    }
    sum = sum_of_lanes<64>(sum);
    if((threadIdx.x & 63) == 0)
    {
        of_wave[threadIdx.x >> 6] = {top, sum};
    }
    __syncthreads();
    if(threadIdx.x == 0)
    {
        args.parts[row * args.all + args.part0 + blockIdx.y]
            = joined(joined(of_wave[0], of_wave[1]), joined(of_wave[2], of_wave[3]));
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

// The listed logits worked out on their own, where no logits are written: a wave an entry, the product of the row's state with
// the entry's weights.  Bound by the gather of the weights' rows: 2048 rows of 32 entries, a tenth of them none, and a K of
// 2048, 242 MB, take 42 us (5.8 TB/s, part of it from the caches).  STEP: elements of a load; step_b: from one element of
// an entry's weights to the next.
struct pick_args
{
    wanted_args want;
    const void* A; // rows, lda apart
    const void* B;
    long long   lda, entry_b, step_b; // elements from an entry to the next, and within one
    int         K;
    float*      picked;
};

template<class InT, int STEP>
__global__ void __launch_bounds__(256) pick_products(const pick_args args)
{
    typedef InT     in_t __attribute__((ext_vector_type(STEP)));
    const int       lane  = threadIdx.x & 63;
    const long long total = (long long)args.want.rows * args.want.k;
    for(long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); at < total; at += (long long)gridDim.x * 4)
    {
        const long long v   = entry_of(args.want, at);
        float           sum = 0.0f;
        if(v >= 0)
        {
            const InT* const a = static_cast<const InT*>(args.A) + at / args.want.k * args.lda;
            const InT* const b = static_cast<const InT*>(args.B) + v * args.entry_b;
#pragma unroll 4
            for(int i = lane * STEP; i < args.K; i += 64 * STEP)
            {
                const in_t x = *reinterpret_cast<const in_t*>(a + i), y = *reinterpret_cast<const in_t*>(b + i * args.step_b);
#pragma unroll
                for(int e = 0; e < STEP; ++e)
                {
                    sum += (float)x[e] * (float)y[e];
                }
            }
            sum = sum_of_lanes<64>(sum);
        }
        if(lane == 0)
        {
            args.picked[at] = sum;
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
    wanted_args         want;
    const softmax_part* parts; // rows x all
    const float*        picked; // rows x k
    float*              loss;
    float*              lse;
    int                 all;
};

// The loss of a row from its parts: a wave a row, or (WAVES 4) a workgroup a row, where there are few with many parts.
template<int WAVES>
__global__ void __launch_bounds__(256) join_rows(const join_args args)
{
    __shared__ softmax_part of_wave[4];
    const int               lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long         step = (long long)gridDim.x * (4 / WAVES);
    for(long long row = (long long)blockIdx.x * (4 / WAVES) + wave / WAVES; row < args.want.rows; row += step)
    {
        softmax_part all{-__builtin_inff(), 0.0f};
#pragma unroll 4
        for(int p = wave % WAVES * 64 + lane; p < args.all; p += 64 * WAVES)
        {
            all = joined(all, args.parts[row * args.all + p]);
        }
#pragma unroll
        for(int d = 1; d < 64; d *= 2)
        {
            const softmax_part other{__shfl_xor(all.top, d), __shfl_xor(all.sum, d)};
            all = joined(all, other);
        }
        if constexpr(WAVES == 4)
        {
            // (a workgroup's rows are its own: every thread is in the loop as often)
            __syncthreads();
            of_wave[wave] = all;
            __syncthreads();
            all = joined(joined(of_wave[0], of_wave[1]), joined(of_wave[2], of_wave[3]));
            if(wave != 0)
            {
                continue;
            }
        }
        // What lies between the largest logit and a listed one first: it is exact where the two are near, 0 where they are one
        // (z scale2 is rounded as it was for the largest: no multiply-add).  Where tiles leave the statistics the listed logit comes
        // from pick_products, whose sum has another order: it may be a rounding above the largest, but -log p is not below 0.
        const float rest = log2f(all.sum);
        auto        less_log_p = [&](float z) {
#pragma clang fp contract(off)
            const float x = z * args.want.scale2, bits = (all.top - x) + rest;
            return (bits < 0.0f ? 0.0f : bits) * log_of_2;
        };
        float       loss = 0.0f;
        if(args.want.teacher == nullptr)
        {
            loss = entry_of(args.want, row) >= 0 ? less_log_p(args.picked[row]) : 0.0f;
        }
        else
        {
            const listed_row l = read_list(args.want, row);
            const float      norm = l.sum > 0.0f ? 1.0f / l.sum : 0.0f, log_norm = l.sum > 0.0f ? logf(l.sum) : 0.0f;
#pragma unroll
            for(int r = 0; r < list_rounds; ++r)
            {
                const float q = l.e[r] * norm;
                if(q > 0.0f || q != q)
                {
                    loss += q * ((l.x[r] - log_norm) + less_log_p(args.picked[row * args.want.k + r * 64 + lane]));
                }
            }
            loss = sum_of_lanes<64>(loss) / args.want.scale / args.want.scale; // (the square may leave fp32)
        }
        if(lane == 0)
        {
            args.lse[row]  = (all.top + rest) * log_of_2;
            args.loss[row] = loss;
        }
    }
}

// ------------------------------------------------------------------ the gradient

// The gradient of a row's logits is worked out as T dloss / most 2^14 (p - q), with `most` the largest T |dloss| of the
// rows that are compared with something, and 0 for the others, whatever their dloss; the products' sums are brought back by
// unit = most 2^-14 as they are rounded.  It is held in 16 bits, whose smallest number in f16 is 6e-8 (p - q is at most 1, so 2^14
// stays in range), and where all rows have one dloss, as under a mean, its rounding leaves p - q of a target with a small p as it is: against 64 bits a bf16
// gradient is 1.9e-3 off instead of 2.6e-3 with dloss itself in it (1.7e-3 is its own last rounding).  Gradients in fp32 hold no more
// of it: they are 8.4e-4 off from bf16 operands and 1.3e-4 from f16 (4096 x 65536 x 4096, 2048 x 32000 x 2048).  More bits would take
// the products of both dA and dB twice.
struct record_args
{
    wanted_args  want;
    const float* dloss; // (of lists: counted_gradients')
    const float* lse;
    loss_record* records;
    float*       unit; // [0]: unit, [1]: most
};

// dloss of the rows whose list has a share, 0 of the others: a list takes a wave to look through, so it is done once, before
// all rows are looked through for the largest.  A wave a row.
__global__ void __launch_bounds__(256)
    counted_gradients(const wanted_args want, const float* __restrict__ dloss, float* __restrict__ counted)
{
    for(long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < want.rows; row += (long long)gridDim.x * 4)
    {
        const float sum = read_list(want, row).sum;
        if((threadIdx.x & 63) == 0)
        {
            counted[row] = sum > 0.0f || sum != sum ? dloss[row] : 0.0f;
        }
    }
}

// The largest T |dloss| of the rows that count, 1 if there is none; by all threads of a workgroup.
template<int THREADS>
__device__ __forceinline__ float largest_gradient(const record_args& args)
{
    __shared__ float of_wave[THREADS / 64];
    float            most = 0.0f;
    auto look = [&](auto entry) { // (a loop for every width of an index: the loads of eight rows go out together)
        const int last = args.want.rows - 1;
        for(int first = threadIdx.x; first <= last; first += 8 * THREADS)
        {
            float     said[8];
            long long v[8];
#pragma unroll
            for(int u = 0; u < 8; ++u)
            {
                const int row = first + u * THREADS < last ? first + u * THREADS : last; // (the last row again changes nothing)
                said[u]       = args.dloss[row];
                v[u]          = entry(row);
            }
#pragma unroll
            for(int u = 0; u < 8; ++u)
            {
                const float d = __builtin_fabsf(said[u] / args.want.scale);
                most = v[u] >= 0 && v[u] < args.want.vocabulary && d > most && d < __builtin_inff() ? d : most;
            }
        }
    };
    if(args.want.teacher != nullptr)
    {
        look([](int) { return 0ll; }); // (with a list that counts there is a vocabulary)
    }
    else if(args.want.wide)
    {
        look([&](int row) { return static_cast<const long long*>(args.want.entries)[row]; });
    }
    else
    {
        look([&](int row) { return (long long)static_cast<const int*>(args.want.entries)[row]; });
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
    most = of_wave[0];
    for(int w = 1; w < THREADS / 64; ++w)
    {
        most = __builtin_fmaxf(most, of_wave[w]);
    }
    return most > 0.0f ? most : 1.0f;
}

__device__ __forceinline__ void write_unit(const record_args& args, float most)
{
    args.unit[0] = most * 0x1p-14f;
    args.unit[1] = most;
}

// (one workgroup)
__global__ void __launch_bounds__(1024) gradient_unit(const record_args args)
{
    const float most = largest_gradient<1024>(args);
    if(threadIdx.x == 0)
    {
        write_unit(args, most);
    }
}

// A thread a row.  ALONE: every workgroup looks for the largest gradient itself, where that is less than waiting for a launch that
// does (4 us; 64 KB of dloss and the targets are read in less).
constexpr int most_alone = 16384; // rows
template<bool ALONE>
__global__ void __launch_bounds__(256) gradient_records(const record_args args)
{
    float most;
    if constexpr(ALONE)
    {
        most = largest_gradient<256>(args);
        if(blockIdx.x == 0 && threadIdx.x == 0)
        {
            write_unit(args, most);
        }
    }
    else
    {
        most = args.unit[1];
    }
    for(long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < args.want.rows; row += (long long)gridDim.x * 256)
    {
        const bool      listed = args.want.teacher != nullptr;
        const long long target = listed ? -1 : entry_of(args.want, row);
        const float     dloss  = args.dloss[row];
        const bool      is     = listed ? dloss != 0.0f : target >= 0;
        const float     factor = dloss / args.want.scale / most * 0x1p14f;
        args.records[row]      = is ? loss_record{args.lse[row] * log2_of_e, factor, (int)target, 0}
                                    : loss_record{__builtin_inff(), 0.0f, -1, 0};
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
    const loss_record* records;
    const float* picked; // rows x k (a list)
};

// dz = factor (2^(scale2 z - lse) - q), 8 columns a thread; q of a target alone (a list's entries are put right by listed_slope).
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
    const loss_record own    = args.records[row];
    const long long   target = own.target - args.col0;
    const float*      z      = args.z + row * args.pitch + col;
    const f32x4  lo = *reinterpret_cast<const f32x4*>(z), hi = *reinterpret_cast<const f32x4*>(z + 4);
    in8 o;
#pragma unroll
    for(int e = 0; e < 8; ++e)
    {
        const float p = __builtin_amdgcn_exp2f((e < 4 ? lo[e & 3] : hi[e & 3]) * args.want.scale2 - own.lse);
        const float d = own.factor * (p - (target == col + e ? 1.0f : 0.0f));
        o[e]          = to_out<InT>(col + e >= args.cols ? 0.0f : d);
    }
    *reinterpret_cast<in8*>(static_cast<InT*>(args.dz) + row * args.pitch + col) = o;
}

// The listed entries of a piece: factor (2^(scale2 z - lse) - q), from the logits that the loss picked; q of an entry that is
// listed more than once is the sum of its q, in the order of the list, and each of them writes the same.  A wave a row.
template<class InT>
__global__ void __launch_bounds__(256) listed_slope(const softmax_slope_args args)
{
    typedef int      i32x4 __attribute__((ext_vector_type(4)));
    __shared__ int   entries[4][most_entries] __attribute__((aligned(16)));
    __shared__ float shares[4][most_entries] __attribute__((aligned(16)));
    const int            lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int            k    = args.want.k;
    const long long      step = (long long)gridDim.x * 4;
    // (every wave makes the same number of rounds, for the barriers)
    for(long long first = (long long)blockIdx.x * 4; first < args.want.rows; first += step)
    {
        const long long row    = first + wave;
        const bool      is     = row < args.want.rows;
        const loss_record own = is ? args.records[row] : loss_record{};
        const float     factor = own.factor;
        if(is)
        {
            const listed_row l    = read_list(args.want, row);
            const float      norm = l.sum > 0.0f ? 1.0f / l.sum : l.sum;
#pragma unroll
            for(int r = 0; r < list_rounds; ++r)
            {
                entries[wave][r * 64 + lane] = (int)l.entry[r]; // (-1 past the list's end)
                shares[wave][r * 64 + lane]  = l.e[r] * norm;
            }
        }
        __syncthreads();
        if(factor != 0.0f)
        {
            for(int j = lane; j < k; j += 64)
            {
                const int v = entries[wave][j];
                if(v >= args.col0 && v < args.col0 + args.cols)
                {
                    float q = 0.0f;
#pragma unroll 4
                    for(int i = 0; i < k; i += 4)
                    {
                        const i32x4 listed = *reinterpret_cast<const i32x4*>(&entries[wave][i]);
                        const f32x4 share  = *reinterpret_cast<const f32x4*>(&shares[wave][i]);
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            q += listed[e] == v ? share[e] : 0.0f;
                        }
                    }
                    const float p = __builtin_amdgcn_exp2f(args.picked[row * k + j] * args.want.scale2 - own.lse);
                    static_cast<InT*>(args.dz)[row * args.pitch + (v - args.col0)] = to_out<InT>(factor * (p - q));
                }
            }
        }
        __syncthreads();
    }
}

// The weights' gradient from few rows: C_ij = unit sum_t P_ti Q_tj (+ C_ij), P and Q row by row t, at most 32 DEPTH of them.
// Bound by C's stores.  A wave holds 64 columns of Q as four operands of the 16x16x32 MFMA and walks down C's rows, 16 at a
// time; which column an operand's row stands for is chosen so that a lane's four results of four columns are 16 columns in a
// row.  (2 rows of 100848 x 1288, 260 MB: 63 us, 4.1 TB/s; the tiles of
// the layer products spend a round of their ring on so short a sum and took 202.)
struct outer_args
{
    const void*  P; // t x rows, p_pitch apart
    const void*  Q; // t x cols
    void*        C; // rows x cols, c_pitch apart
    const float* unit;
    long long    p_pitch, q_pitch, c_pitch;
    long long    rows, cols;
    int          t, add;
    int          each; // rows of a workgroup, a multiple of 16
};

constexpr int outer_rows = 256, outer_cols = 256; // of a workgroup, at most

__device__ __forceinline__ f32x4 multiply_outer(__bf16 __attribute__((ext_vector_type(8))) a, __bf16 __attribute__((ext_vector_type(8))) b,
                                                f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply_outer(_Float16 __attribute__((ext_vector_type(8))) a,
                                                _Float16 __attribute__((ext_vector_type(8))) b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template<class InT, class OutT, int DEPTH>
__global__ void __launch_bounds__(256) outer_product(const outer_args args)
{
    typedef InT     in8 __attribute__((ext_vector_type(8)));
    constexpr int   PIECE = 16 / (int)sizeof(OutT); // columns of a store
    typedef OutT    piece_t __attribute__((ext_vector_type(PIECE)));
    typedef piece_t piece_anywhere __attribute__((aligned(sizeof(OutT))));
    const int       lane = threadIdx.x & 63, c16 = lane & 15, g = lane >> 4;
    const long long col0 = (long long)blockIdx.y * outer_cols + (threadIdx.x >> 6) * 64;
    if(col0 >= args.cols)
    {
        return;
    }
    // element [t][at] of an operand, 0 outside (the address is always inside)
    auto element = [&](const void* from, long long pitch, int t, long long at, long long end) {
        const bool is = t < args.t && at < end;
        const InT  v  = static_cast<const InT*>(from)[is ? t * pitch + at : 0];
        return is ? v : (InT)0.0f;
    };
    in8 q[4][DEPTH];
#pragma unroll
    for(int f = 0; f < 4; ++f)
    {
#pragma unroll
        for(int d = 0; d < DEPTH; ++d)
        {
#pragma unroll
            for(int u = 0; u < 8; ++u)
            {
                q[f][d][u] = element(args.Q, args.q_pitch, d * 32 + g * 8 + u, col0 + (c16 >> 2) * 16 + f * 4 + (c16 & 3), args.cols);
            }
        }
    }
    const float     unit = *args.unit;
    const long long row1 = (long long)(blockIdx.x + 1) * args.each, end = row1 < args.rows ? row1 : args.rows;
    const long long col  = col0 + g * 16; // this lane's 16
    for(long long row0 = (long long)blockIdx.x * args.each; row0 < end; row0 += 16)
    {
        in8 p[DEPTH];
#pragma unroll
        for(int d = 0; d < DEPTH; ++d)
        {
#pragma unroll
            for(int u = 0; u < 8; ++u)
            {
                p[d][u] = element(args.P, args.p_pitch, d * 32 + g * 8 + u, row0 + c16, end);
            }
        }
        float y[16];
#pragma unroll
        for(int f = 0; f < 4; ++f)
        {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for(int d = 0; d < DEPTH; ++d)
            {
                sum = multiply_outer(q[f][d], p[d], sum);
            }
#pragma unroll
            for(int e = 0; e < 4; ++e)
            {
                y[4 * f + e] = unit * sum[e];
            }
        }
        if(row0 + c16 >= end)
        {
            continue;
        }
        OutT* const to = static_cast<OutT*>(args.C) + (row0 + c16) * args.c_pitch + col;
#pragma unroll
        for(int s = 0; s < 16; s += PIECE)
        {
            if(col + s + PIECE <= args.cols)
            {
                piece_t o{};
                if(args.add)
                {
                    o = *reinterpret_cast<const piece_anywhere*>(to + s);
                }
#pragma unroll
                for(int e = 0; e < PIECE; ++e)
                {
                    o[e] = to_out<OutT>(args.add ? y[s + e] + (float)o[e] : y[s + e]);
                }
                *reinterpret_cast<piece_anywhere*>(to + s) = o;
                continue;
            }
#pragma unroll
            for(int e = 0; e < PIECE; ++e)
            {
                if(col + s + e < args.cols)
                {
                    to[s + e] = to_out<OutT>(args.add ? y[s + e] + (float)to[s + e] : y[s + e]);
                }
            }
        }
    }
}

// out (rows of `cols` elements) = the sum of `parts` (part_size apart, rows pitch apart), in their order, times unit.
template<class OutT>
__global__ void __launch_bounds__(256)
    scaled_rows(const float* __restrict__ from, int parts, long long part_size, long long pitch, OutT* __restrict__ out, long long rows,
                long long cols, const float* __restrict__ unit)
{
    const float     by     = *unit;
    const long long pieces = (cols + 3) / 4, total = rows * pieces; // (from's rows are padded to whole pieces)
    const bool      whole  = cols % 4 == 0 && reinterpret_cast<unsigned long long>(out) % (4 * sizeof(OutT)) == 0;
    typedef OutT    out4 __attribute__((ext_vector_type(4)));
    for(long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long long)gridDim.x * 256)
    {
        const long long row = at / pieces, col = (at - row * pieces) * 4;
        f32x4           v   = *reinterpret_cast<const f32x4*>(from + row * pitch + col);
#pragma unroll 4
        for(int part = 1; part < parts; ++part)
        {
            v += *reinterpret_cast<const f32x4*>(from + part * part_size + row * pitch + col);
        }
        OutT* const to = out + row * cols + col;
        out4        o;
#pragma unroll
        for(int e = 0; e < 4; ++e)
        {
            o[e] = to_out<OutT>(v[e] * by);
        }
        if(whole)
        {
            *reinterpret_cast<out4*>(to) = o;
            continue;
        }
#pragma unroll
        for(int e = 0; e < 4; ++e)
        {
            if(col + e < cols)
            {
                to[e] = o[e];
            }
        }
    }
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_HEAD_LOSS_HPP
