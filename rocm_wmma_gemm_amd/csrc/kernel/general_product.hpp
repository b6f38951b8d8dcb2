// The layer products for operands of any alignment and extent: register-staged, guarded loads
// (the scalar mode of gemm_kernel.hpp's staging) and stores element by element.
//
// C tile of 128 x 128 (64 x 64 for small problems) per workgroup, 4 waves, 32x32x16 MFMA, two
// stages of BK in LDS.  It serves what the direct-to-LDS kernels cannot: rows that do not start
// on 16 bytes.  Bound by the 2-byte gathers of operands that are contiguous along M or N:
// 1999 x 1001 x 999 takes 115 us here and 32 on padded copies, so it is left with what is too
// small for copies to pay and with calls that get no scratch memory.
#ifndef ROCM_WMMA_GEMM_GENERAL_PRODUCT_HPP
#define ROCM_WMMA_GEMM_GENERAL_PRODUCT_HPP

#include "product_common.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

template<in_kind IN, class OutT, class ResT, bool A_KMAJOR, bool B_KMAJOR, int BM, int BN, int BK>
struct general_product
{
    using gemm = staged_gemm<IN, OutT, A_KMAJOR, B_KMAJOR, BM, BN, BK, 2, 2, load_mode::scalar>;
    using InT  = typename gemm::InT;
    static constexpr int THREADS = gemm::THREADS;
    static constexpr int TM = gemm::TM, TN = gemm::TN;

    __device__ __forceinline__ static void run(const product_args& args)
    {
        __shared__ u32x4 lds[2 * gemm::STAGE];
        __shared__ int   off[max_groups + 1], first[max_groups + 1];
        if(args.kind != product_kind::batch)
        {
            build_group_table(args.offsets, args.groups, args.kind == product_kind::rows ? args.M : args.K, BM,
                              &off[0], &first[0]);
        }
        const int items = count_items(args, &first[0]);
        for(int item = blockIdx.x; item < items; item += gridDim.x)
        {
            product_item x;
            const int    row_tile = item / args.grid_n; // of all groups
            x.col0                = (item - row_tile * args.grid_n) * BN;
            if(args.kind == product_kind::rows)
            {
                x.group = group_of_tile(&first[0], args.groups, row_tile);
                x.row0  = (row_tile - first[x.group]) * BM;
            }
            else
            {
                x.group = row_tile / args.grid_m;
                x.row0  = (row_tile - x.group * args.grid_m) * BM;
            }
            place_group(args, &off[0], x);
            tile(args, x, lds);
        }
    }

    __device__ __forceinline__ static void tile(const product_args& args, const product_item& x, u32x4* lds)
    {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int wave_m = wave / 2, wave_n = wave % 2, lane_lo = lane & 31, lane_hi = lane >> 5;
        const long long a_sr = A_KMAJOR ? args.lda : 1, a_sk = A_KMAJOR ? 1 : args.lda;
        const long long b_sr = B_KMAJOR ? args.ldb : 1, b_sk = B_KMAJOR ? 1 : args.ldb;
        const InT*      a    = static_cast<const InT*>(args.A) + x.a_at + x.row0 * a_sr;
        const InT*      b    = static_cast<const InT*>(args.B) + x.b_at + x.col0 * b_sr;
        const int       rows_a = x.m - x.row0, rows_b = args.N - x.col0;

        f32x16 acc[TM][TN];
#pragma unroll
        for(int i = 0; i < TM; ++i)
        {
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
#pragma unroll
                for(int v = 0; v < 16; ++v)
                {
                    acc[i][j][v] = 0.0f;
                }
            }
        }
        typename gemm::stage_a sa;
        typename gemm::stage_b sb;
        const int              steps = (x.k + BK - 1) / BK;
        if(steps > 0)
        {
            sa.fetch(a, a_sr, a_sk, rows_a, x.k, tid);
            sb.fetch(b, b_sr, b_sk, rows_b, x.k, tid);
            sa.commit(lds, tid);
            sb.commit(lds + gemm::A_TILE, tid);
        }
        __syncthreads();
        for(int step = 0; step < steps; ++step)
        {
            const bool more = step + 1 < steps;
            if(more)
            {
                const long long k0 = (long long)(step + 1) * BK;
                sa.fetch(a + k0 * a_sk, a_sr, a_sk, rows_a, x.k - (int)k0, tid);
                sb.fetch(b + k0 * b_sk, b_sr, b_sk, rows_b, x.k - (int)k0, tid);
            }
            const u32x4* here = lds + (step & 1) * gemm::STAGE;
            gemm::compute_stage(here, here + gemm::A_TILE, acc, wave_m * gemm::WTM + lane_lo,
                                wave_n * gemm::WTN + lane_lo, lane_hi);
            if(more)
            {
                u32x4* next = lds + ((step + 1) & 1) * gemm::STAGE;
                sa.commit(next, tid);
                sb.commit(next + gemm::A_TILE, tid);
            }
            __syncthreads();
        }
        // Accumulator register v of a 32x32 tile: row 8*(v/4) + 4*(lane/32) + v%4, column lane%32.
#pragma unroll
        for(int i = 0; i < TM; ++i)
        {
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
                const int col = x.col0 + wave_n * gemm::WTN + j * 32 + lane_lo;
#pragma unroll
                for(int v = 0; v < 16; ++v)
                {
                    const int row = x.row0 + wave_m * gemm::WTM + i * 32 + 8 * (v / 4) + 4 * lane_hi + (v % 4);
                    if(row < x.m && col < args.N)
                    {
                        finish_element<InT, OutT, ResT>(args, x, row, col, acc[i][j][v]);
                    }
                }
            }
        }
    }
};

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_GENERAL_PRODUCT_HPP
