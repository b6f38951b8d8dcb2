// The layer products where few rows meet a weight (decode; experts with a handful of tokens): the
// streaming kernel's data path (stream_kernel.hpp) with a group's tiles and the layer's epilogue.
//
// A workgroup owns BM rows x BN columns of a group's C and the whole sum: it streams its BN rows
// of the weight from memory exactly once, BM rows of A come out of L2.  Bound by the weights'
// bytes: 16 rows on 14 of 64 weights of 2048 x 4096 take 41 us, 5.75 TB/s; 32 x 4096 x 14336 on 32 x 16 tiles
// 29.4 us, 4.0 TB/s (16 x 32 tiles 33.8, two slices of K 39).  Experts without rows have no tiles, so their
// weights are never read.  Ring, swizzles and waits are the streaming kernel's; the four waves split K and their partial tiles meet in LDS,
// where bias, activation and residual join them.  The row tiles that share a slice of a weight are
// neighbours on one XCD.
//
// Where the tiles are too few for the compute units, args.k_slices workgroups share one, as in the
// streaming kernel: each leaves its part in args.partials, counts itself in, and the last to arrive
// adds the parts up in slice order and finishes the tile.
#ifndef ROCM_WMMA_GEMM_SKINNY_PRODUCT_HPP
#define ROCM_WMMA_GEMM_SKINNY_PRODUCT_HPP

#include "product_common.hpp"
#include "stream_kernel.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

// ONCE: the weight's loads carry the non-temporal hint (product_kernel::once).
template<in_kind IN, class OutT, class ResT, int BM, int BN, bool B_KMAJOR, bool ONCE>
struct skinny_product
{
    using S   = stream_gemm<IN, OutT, BM, BN, true, B_KMAJOR>;
    using InT = typename S::InT;
    static constexpr int THREADS = S::THREADS, BK = S::BK, TM = S::TM, TN = S::TN, DEPTH = S::DEPTH;

    __device__ __forceinline__ static void run(const product_args& args)
    {
        __shared__ __attribute__((aligned(1024))) char lds_raw[S::LDS_BYTES];
        lds_char_ptr       lds      = (lds_char_ptr)lds_raw;
        const unsigned int lds_addr = (unsigned int)(size_t)lds;
        const int          lane     = threadIdx.x & 63;
        const int          wave     = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

        // Which tile.  The group table is built in the ring, which is empty yet.
        product_item x;
        int          tm, tn, slice, tile;
        {
            using lds_int  = __attribute__((address_space(3))) int;
            lds_int* off   = reinterpret_cast<lds_int*>(lds);
            lds_int* first = off + max_groups + 1;
            static_assert(2 * (max_groups + 1) * 4 <= S::LDS_BYTES, "the table fits the ring");
            const bool batch = args.kind == product_kind::batch;
            if(!batch)
            {
                build_group_table(args.offsets, args.groups, args.M, BM, off, first);
            }
            const int per_group = args.grid_m * args.grid_n;
            const int total = batch ? args.groups * per_group : __builtin_amdgcn_readfirstlane(first[args.groups]) * args.grid_n;
            // (slices outermost over the grid's tiles, so that a tile's slices have one counter)
            const int most = gridDim.x / args.k_slices;
            slice          = blockIdx.x / most;
            tile           = blockIdx.x - slice * most;
            if(tile >= total)
            {
                return; // (the grid covers the most tiles that this many rows can have)
            }
            const int item = xcd_remap(tile, total);
            int       high = args.grid_m, local;
            if(batch)
            {
                x.group = __builtin_amdgcn_readfirstlane(item / per_group);
                local   = item - x.group * per_group;
            }
            else
            {
                x.group     = group_of_tile(first, args.groups, item / args.grid_n);
                const int f = __builtin_amdgcn_readfirstlane(first[x.group]);
                high        = __builtin_amdgcn_readfirstlane(first[x.group + 1]) - f;
                local       = item - f * args.grid_n;
            }
            tn              = local / high;
            tm              = local - tn * high;
            place_group(args, off, x);
            __syncthreads(); // every wave has read the table: the ring may fill
        }
        x.row0 = __builtin_amdgcn_readfirstlane(tm * BM);
        x.col0 = __builtin_amdgcn_readfirstlane(tn * BN);

        const long long lda = args.lda, ldb = args.ldb;
        const InT*      a0 = static_cast<const InT*>(args.A) + x.a_at + x.row0 * lda;
        const InT*      b0 = static_cast<const InT*>(args.B) + x.b_at + (B_KMAJOR ? x.col0 * ldb : (long long)x.col0);
        const u32x4     rsrc_a = S::descriptor(a0, (x.m - x.row0) * lda * 2);
        const u32x4     rsrc_b = S::descriptor(b0, B_KMAJOR ? (args.N - x.col0) * ldb * 2 : (args.K * ldb - x.col0) * 2);
        const int          sub    = lane >> 4, slot = lane & 15;
        const int          chunk  = slot ^ ((4 * wave + sub) & 15);
        const unsigned int voff_a = (unsigned int)(((4 * wave + sub) * lda + chunk * 8) * 2);
        const unsigned int voff_b = B_KMAJOR ? (unsigned int)(((4 * wave + sub) * ldb + chunk * 8) * 2)
                                             : S::template mn_load_offset<BN>(lane, wave, ldb);
        const unsigned int step_a  = (unsigned int)(16 * lda * 2);
        const unsigned int step_b  = (unsigned int)((B_KMAJOR ? 16 : 4 * (512 / BN)) * ldb * 2);
        const unsigned int stage_b = B_KMAJOR ? (unsigned int)S::ROW_BYTES : (unsigned int)(BK * ldb * 2);
        const int          k_tail  = args.K % BK;
        const unsigned int past    = 0x80000000u;
        const unsigned int voff_a_tail = k_tail != 0 && chunk * 8 >= k_tail ? past : voff_a;
        const unsigned int voff_b_tail = B_KMAJOR && k_tail != 0 && chunk * 8 >= k_tail ? past : voff_b;
        // this workgroup's run of the stages
        const int all = (args.K + BK - 1) / BK, each = (all + args.k_slices - 1) / args.k_slices, from = slice * each;
        const int stages = all - from < each ? all - from : each; // >= 1 (host)
        auto issue = [&](int run_stage, int at) {
            const int          stage = from + run_stage;
            const unsigned int base = lds_addr + at * S::STAGE + wave * 1024;
            const bool         last = stage == all - 1; // the stage that K may cut short
            const unsigned int va = last ? voff_a_tail : voff_a, vb = last ? voff_b_tail : voff_b;
#pragma unroll
            for(int i = 0; i < S::LOADS_A; ++i)
            {
                S::template load_block<false>(
                    base + i * 4096, va, rsrc_a,
                    __builtin_amdgcn_readfirstlane((unsigned int)stage * (unsigned int)S::ROW_BYTES + i * step_a));
            }
#pragma unroll
            for(int i = 0; i < S::LOADS_B; ++i)
            {
                S::template load_block<ONCE>(base + S::A_BYTES + i * 4096, vb, rsrc_b,
                                              __builtin_amdgcn_readfirstlane((unsigned int)stage * stage_b + i * step_b));
            }
        };
        // The column panels of a weight start their walk along K at staggered stages and wrap
        // round, so that they do not all ask the same memory channels at the same time.
        const int turn    = (int)(((long long)tn * stages) / args.grid_n);
        auto      clamped = [&](int stage) {
            const int at = (stage < stages ? stage : stages - 1) + turn;
            return at >= stages ? at - stages : at;
        };

        f32x4 acc[TM][TN];
#pragma unroll
        for(int i = 0; i < TM; ++i)
        {
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        const int frag_off = slot * S::ROW_BYTES + (((4 * wave + sub) ^ slot) & 15) * 16;
        const int tr_off_b = S::template mn_read_offset<BN>(wave, sub, slot);
        using lds_u32x4    = __attribute__((address_space(3))) u32x4;
        for(int t = 0; t < DEPTH - 1; ++t)
        {
            issue(clamped(t), t);
        }
        S::settle(acc);
        int slot_index = 0;
        for(int t = 0; t < stages; ++t)
        {
            // stage t has landed in every wave; the slot of stage t - 1 may be filled again
            __builtin_amdgcn_s_waitcnt(S::vmcnt_imm((DEPTH - 2) * S::PER));
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            issue(clamped(t + DEPTH - 1), slot_index == 0 ? DEPTH - 1 : slot_index - 1);
            lds_char_ptr       sa   = lds + slot_index * S::STAGE + frag_off;
            const unsigned int sb_t = lds_addr + slot_index * S::STAGE + S::A_BYTES + tr_off_b;
            u32x4              fa[TM], fb[TN];
#pragma unroll
            for(int i = 0; i < TM; ++i)
            {
                fa[i] = *reinterpret_cast<lds_u32x4*>(sa + i * 16 * S::ROW_BYTES);
            }
            if constexpr(B_KMAJOR)
            {
#pragma unroll
                for(int j = 0; j < TN; ++j)
                {
                    fb[j] = *reinterpret_cast<lds_u32x4*>(sa + S::A_BYTES + j * 16 * S::ROW_BYTES);
                }
            }
            else
            {
                S::transposed(sb_t, fb);
            }
#pragma unroll
            for(int i = 0; i < TM; ++i)
            {
#pragma unroll
                for(int j = 0; j < TN; ++j)
                {
                    S::multiply_add(acc[i][j], fa[i], fb[j]);
                }
            }
            slot_index = slot_index + 1 == DEPTH ? 0 : slot_index + 1;
        }
        S::settle(acc);
        __builtin_amdgcn_s_waitcnt(S::vmcnt_imm(0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        using lds_float = __attribute__((address_space(3))) float;
        lds_float* part = reinterpret_cast<lds_float*>(lds);
#pragma unroll
        for(int i = 0; i < TM; ++i)
        {
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
#pragma unroll
                for(int v = 0; v < 4; ++v)
                {
                    part[(wave * BM + 16 * i + 4 * sub + v) * BN + 16 * j + slot] = acc[i][j][v];
                }
            }
        }
        __syncthreads();
        // (wave order: the sum of an element is the same in every run)
        auto tile_sum = [&](int e) {
            return ((part[e] + part[BM * BN + e]) + part[2 * BM * BN + e]) + part[3 * BM * BN + e];
        };
        // Finishes the tile from sums that `sum_of` gives by element: 8 columns a thread where rows
        // of C start on 16 bytes, else one.
        auto finish = [&](auto sum_of) {
            if(args.wide)
            {
                for(int piece = threadIdx.x; piece < BM * BN / 8; piece += THREADS)
                {
                    const int row = x.row0 + piece / (BN / 8), col = x.col0 + piece % (BN / 8) * 8;
                    if(row < x.m && col < args.N)
                    {
                        float sum[8];
#pragma unroll
                        for(int e = 0; e < 8; ++e)
                        {
                            sum[e] = sum_of(piece * 8 + e);
                        }
                        finish_piece<InT, OutT, ResT>(args, x, row, col, sum);
                    }
                }
                return;
            }
            for(int e = threadIdx.x; e < BM * BN; e += THREADS)
            {
                const int row = x.row0 + e / BN, col = x.col0 + e % BN;
                if(row < x.m && col < args.N)
                {
                    finish_element<InT, OutT, ResT>(args, x, row, col, sum_of(e));
                }
            }
        };
        if(args.k_slices == 1)
        {
            finish(tile_sum);
            return;
        }
        // Parts travel at device scope, past the XCD's own L2; a workgroup counts itself in when its
        // stores have been acknowledged (see stream_gemm::run, whose exchange this is).
        constexpr int DEVICE_SCOPE = 16, TILE = BM * BN, MAX_SLICES = S::MAX_SLICES;
        const __amdgpu_buffer_rsrc_t shared = __builtin_amdgcn_make_buffer_rsrc(
            args.partials + (long long)tile * args.k_slices * TILE, 0, args.k_slices * TILE * 4, 0x00020000);
        for(int e = threadIdx.x; e < TILE; e += THREADS)
        {
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned int, tile_sum(e)), shared,
                                                  (slice * TILE + e) * 4, 0, DEVICE_SCOPE);
        }
        __builtin_amdgcn_s_waitcnt(S::vmcnt_imm(0));
        __syncthreads();
        __shared__ unsigned int arrived_before;
        if(threadIdx.x == 0)
        {
            // the counter holds (epoch << 8 | arrivals); a count under another epoch starts from zero
            unsigned int seen = __hip_atomic_load(args.arrivals + tile, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            for(;;)
            {
                const unsigned int count = (seen >> 8) == args.arrival_epoch ? (seen & 255u) : 0u;
                if(__hip_atomic_compare_exchange_strong(args.arrivals + tile, &seen,
                                                        (args.arrival_epoch << 8) | (count + 1u), __ATOMIC_RELAXED,
                                                        __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
                {
                    arrived_before = count;
                    break;
                }
            }
        }
        __syncthreads();
        if(arrived_before != (unsigned int)(args.k_slices - 1))
        {
            return; // the last one to arrive finishes the tile
        }
        // (every slice's value of an element is on its way before the first is added)
        finish([&](int e) {
            float v[MAX_SLICES];
#pragma unroll
            for(int q = 0; q < MAX_SLICES; ++q)
            {
                v[q] = q < args.k_slices ? __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                                                         shared, (q * TILE + e) * 4, 0, DEVICE_SCOPE))
                                         : 0.0f;
            }
            float sum = v[0];
#pragma unroll
            for(int q = 1; q < MAX_SLICES; ++q)
            {
                sum = q < args.k_slices ? sum + v[q] : sum;
            }
            return sum;
        });
        if(threadIdx.x == 0)
        {
            // back to zero arrivals, for a replay of this launch (same epoch)
            __hip_atomic_store(args.arrivals + tile, args.arrival_epoch << 8, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
};

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_SKINNY_PRODUCT_HPP
