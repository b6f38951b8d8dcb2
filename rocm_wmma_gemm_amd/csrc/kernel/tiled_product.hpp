// The layer products on the persistent kernel's K loop (solo_kernel.hpp): 256 x 256 or 128 x 128
// tiles, four waves, direct-to-LDS loads, hand-placed MFMAs.  What differs from the GEMM is which
// tiles there are (groups of rows whose sizes only the device knows, sums over a group's rows)
// and what happens to a finished tile (bias, activation, residual, a second output).
//
// Mathematics: C = act(alpha A B + bias) + beta R, in fp32 from the accumulators, rounded once.
// The tile leaves the registers through a strip of LDS per wave in fp32, half of its columns at a time, so
// that a lane holds 8 (16-bit C) or 4 consecutive columns of a row: bias, residual, C and the
// second output are then 16-byte pieces, and a row of a half is whole cache lines.  Pieces past a
// ragged edge get an offset beyond the descriptors' range: their loads give zeros and their stores
// are dropped, without a branch (behind the hand-placed loop the compiler must find none that
// could make it move accumulators).  An output or input that a call does not have is a descriptor
// of range zero.  The residual's pieces are fetched several rows of MFMA tiles ahead: one at a time
// each would wait out the latency of memory.
//
// Bound: the matrix cores for 256 x 256 tiles (the loop is the GEMM's); the epilogue adds what
// the activation costs, which nothing overlaps with one wave per SIMD.  128 x 128 tiles run two
// workgroups per compute unit.  Measured, bf16: dB of 4096 x 5120 x 5120 213 us (1.01 PFLOP/s; 400 tiles on 256
// compute units), 777 x 28672 x 8192 with gelu 373 us (0.98), 4099 rows over 32 weights of 2048 x 4096 157 us
// on 128 x 256 tiles (weights from memory at 3.4 TB/s; 194 on 128 x 128 tiles, 241 on 256 x 256),
// 8192 rows over 8 of 8192 x 4096 561 us on 256 x 256 tiles (625 on 128 x 256).
#ifndef ROCM_WMMA_GEMM_TILED_PRODUCT_HPP
#define ROCM_WMMA_GEMM_TILED_PRODUCT_HPP

#include "product_common.hpp"
#include "solo_kernel.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

// What a kernel does to its tiles, at compile time.
template<bool LAYER, bool LOGISTIC, bool RESIDUAL, bool KEPT, bool SCALED, bool MIRROR, diagonal_use DIAGONAL,
         bool BACK = false, loss_use LOSS = loss_use::none>
struct product_epilogue
{
    static constexpr bool back = BACK; // alpha lies on the device
    static constexpr loss_use loss = LOSS;
    static constexpr bool layer = LAYER; // bias, and relu or nothing; the sum before it is kept
    static constexpr bool logistic = LOGISTIC; // the activation is x s(u)
    static constexpr bool residual = RESIDUAL;
    static constexpr bool kept     = KEPT; // the finished value is kept in A's type
    static constexpr bool scaled   = SCALED; // by alpha and beta
    static constexpr bool mirror = MIRROR; // C is symmetric: tiles on and above the diagonal, written twice
    static constexpr diagonal_use diagonal = DIAGONAL;
};
using epilogue_plain    = product_epilogue<false, false, false, false, false, false, diagonal_use::none>;
using epilogue_add      = product_epilogue<false, false, true, false, false, false, diagonal_use::none>;
using epilogue_layer    = product_epilogue<true, false, true, false, false, false, diagonal_use::none>;
using epilogue_logistic = product_epilogue<true, true, true, false, false, false, diagonal_use::none>;
using epilogue_square   = product_epilogue<false, false, false, false, true, true, diagonal_use::none>;
using epilogue_poly     = product_epilogue<false, false, true, false, true, true, diagonal_use::split>;
using epilogue_next     = product_epilogue<false, false, true, true, true, false, diagonal_use::rows>;
using epilogue_last     = product_epilogue<false, false, true, false, true, false, diagonal_use::rows>;

using epilogue_back     = product_epilogue<false, false, true, false, true, false, diagonal_use::none, true>;
using epilogue_parts    = product_epilogue<false, false, false, false, false, false, diagonal_use::none, false, loss_use::parts>;
using epilogue_slope    = product_epilogue<false, false, false, false, false, false, diagonal_use::none, false, loss_use::slope>;

// NARROW: rows of C, the residual, the second output or the bias do not start on 16 bytes: they go
// element by element, a lane a column, so that a store instruction still writes runs of a row.  ANYWHERE: 16-byte pieces on
// whatever address they start (buffer accesses need no alignment here), element by element in the last column of tiles alone,
// where a piece may reach past its row: dB of 1999 x 32003 x 999, rows of 32003, 189 us, where elements on 128 x 128 tiles took 207.
template<in_kind IN, class OutT, class ResT, bool A_KMAJOR, bool B_KMAJOR, int BM, int BN, class EPI, bool NARROW = false,
         bool ANYWHERE = false>
struct tiled_product
{
    static_assert(!ANYWHERE || (NARROW && !EPI::mirror && EPI::loss == loss_use::none), "whole pieces of rows that start anywhere");
    using loop = solo_gemm<IN, OutT, A_KMAJOR, B_KMAJOR, BM, BN, 64, 2, 2, 2, true>;
    using InT  = typename loop::InT;
    static constexpr int THREADS = loop::THREADS, TM = loop::TM, TN = loop::TN, BK = 64;
    static constexpr int STAGE = loop::STAGE, VM_LOADS = loop::VM_LOADS;
    // The ring: 2 stages, as the GEMM; 3 for 128 x 256 tiles, whose groups have few rows for a weight that
    // comes from memory: the loads of two K tiles are then always on their way.
    static constexpr int RING = BM == 128 && BN == 256 ? 3 : 2, RING_BYTES = RING * STAGE;
    // a wave's strip: 16 rows of a part of the columns of its tile in fp32, 16 bytes of padding a row
    static constexpr int PASSES = RING == 3 ? 4 : 2;
    static constexpr int HALF = TN / PASSES, ROW_BYTES = HALF * 64, PITCH = ROW_BYTES + 16, STRIP = 16 * PITCH;
    static constexpr int TABLE = (3 * (max_groups + 1) + most_teamed_groups + 1) * 4;
    static constexpr int LDS_BYTES = RING_BYTES + 4 * STRIP + TABLE;
    // workgroups per compute unit: what the LDS holds
    static constexpr int PER_CU = LDS_BYTES <= 80 * 1024 ? 2 : 1;
    static_assert(LDS_BYTES <= 160 * 1024 && TN % PASSES == 0 && TM % 2 == 0, "tile");
    static_assert(!EPI::mirror || (TM == TN && BM == BN), "a mirrored tile is square");

    using lds_int   = __attribute__((address_space(3))) int;
    using lds_f32x4 = __attribute__((address_space(3))) f32x4;
    using lds_float = __attribute__((address_space(3))) float;

    // One item of work with what the load stream needs.
    struct work
    {
        product_item x;
        int          nk; // K tiles, at least one
        bool         ends_k; // its last one is the last of K
        float*       partial; // nullptr: a whole tile; else where its [BM][BN] of fp32 goes
        const InT *  a, *b, *a_end, *b_end;
    };

    // The groups' tables and how the launch's tiles are dealt.
    struct plan
    {
        const lds_int *off, *first, *order;
        tail_cut       cut;
        int            teams; // groups go to teams of workgroups (order then lists this team's); 0: tiles are dealt one by one
        int            positions, begin, hop; // of this workgroup: begin, begin + hop, ... < positions
    };

    __device__ __forceinline__ static int tiles_per_group(const product_args& args)
    {
        return EPI::mirror ? args.grid_n * (args.grid_n + 1) / 2 : args.grid_m * args.grid_n;
    }

    __device__ __forceinline__ static plan make_plan(const product_args& args, lds_int* table, int workgroups)
    {
        lds_int *off = table, *first = off + max_groups + 1, *order = first + max_groups + 1;
        int      tiles = args.groups * tiles_per_group(args);
        if(args.kind != product_kind::batch)
        {
            build_group_table(args.offsets, args.groups, args.kind == product_kind::rows ? args.M : args.K, BM, off,
                              first);
            if(args.kind == product_kind::rows)
            {
                tiles = __builtin_amdgcn_readfirstlane(first[args.groups]) * args.grid_n;
            }
            else if(args.groups > 1)
            {
                order_groups(args.groups, off, order);
                const int each = tiles_per_group(args), teams = teams_of(args.groups, each, workgroups);
                if(teams != 0)
                {
                    lds_int*  mine = order + max_groups + 1;
                    const int team = (int)blockIdx.x / each;
                    // (a workgroup beyond the last team has no group)
                    const int n = deal_groups(args.groups, teams, team, BK, off, order, mine, mine + most_teamed_groups);
                    return {off, first, mine, {tiles, 0, 1, 1}, teams,
                            __builtin_amdgcn_readfirstlane(team < teams ? n : 0), 0, 1};
                }
            }
        }
        // (where groups differ in K the slices would too: those launches are not cut; a single group's sum is
        // cut by the rows it has, which its offsets say)
        const bool may_cut = args.partials != nullptr && !EPI::mirror && (args.kind != product_kind::sum || args.groups == 1);
        tail_cut   cut{tiles, 0, 1, 0};
        if(may_cut)
        {
            const int rows = args.kind == product_kind::sum ? off[1] - off[0] : 0;
            cut            = cut_tail(tiles, workgroups, summed_tiles(args.kind, args.K, rows, BK), true);
            cut.whole      = __builtin_amdgcn_readfirstlane(cut.whole);
            cut.cut        = __builtin_amdgcn_readfirstlane(cut.cut);
            cut.slices     = __builtin_amdgcn_readfirstlane(cut.slices);
            cut.each       = __builtin_amdgcn_readfirstlane(cut.each);
        }
        return {off, first, order, cut, 0, cut.positions(), (int)blockIdx.x, workgroups};
    }

    // Tile number `tile` of the launch: its group and place.
    __device__ __forceinline__ static product_item locate(const product_args& args, const plan& pl, int tile)
    {
        product_item x;
        int          local, grid_m = args.grid_m;
        if(args.kind == product_kind::rows)
        {
            x.group     = group_of_tile(pl.first, args.groups, tile / args.grid_n);
            const int f = __builtin_amdgcn_readfirstlane(pl.first[x.group]);
            grid_m      = __builtin_amdgcn_readfirstlane(pl.first[x.group + 1]) - f;
            local       = tile - f * args.grid_n;
        }
        else
        {
            const int tiles = tiles_per_group(args);
            x.group         = tile / tiles;
            local           = tile - x.group * tiles;
            if(pl.teams != 0)
            {
                // position `tile` of the team's list; the workgroup's place in the team is its tile
                x.group = pl.order[tile];
                local   = xcd_remap((int)blockIdx.x % tiles, tiles);
            }
            else if(args.kind == product_kind::sum && args.groups > 1)
            {
                // (one group after the other over the whole GPU, an XCD on neighbouring tiles)
                x.group = pl.order[x.group];
                local   = xcd_remap(local, tiles);
            }
        }
        tile_coord t;
        if constexpr(EPI::mirror)
        {
            t = triangle_tile(local, args.grid_n);
        }
        else
        {
            t = banded_tile(local, grid_m, args.grid_n, 4);
        }
        x.group = __builtin_amdgcn_readfirstlane(x.group);
        x.row0  = __builtin_amdgcn_readfirstlane(t.m * BM);
        x.col0  = __builtin_amdgcn_readfirstlane(t.n * BN);
        place_group(args, pl.off, x);
        return x;
    }

    // Positions congruent mod 8 run on one XCD: it takes a contiguous run of tiles, those of a
    // group in bands of 4 tile rows, so that its L2 serves the panels that its workgroups share (of
    // the cut tiles, a contiguous run of slices over all tiles).
    __device__ __forceinline__ static work decode(const product_args& args, const plan& pl, int pos)
    {
        work w;
        int  tile, slice = 0, k0 = 0;
        w.partial = nullptr;
        if(pos < pl.cut.whole)
        {
            tile = args.kind == product_kind::sum && args.groups > 1 ? pos : xcd_remap(pos, pl.cut.whole);
        }
        else
        {
            const int p = xcd_remap(pos - pl.cut.whole, pl.cut.cut * pl.cut.slices);
            slice       = p / pl.cut.cut;
            const int t = p - slice * pl.cut.cut;
            tile        = pl.cut.whole + t;
            k0          = slice * pl.cut.each;
            w.partial   = args.partials + (long long)(t * pl.cut.slices + slice) * (BM * BN);
        }
        w.x         = locate(args, pl, tile);
        const int k = w.x.k > BK ? (w.x.k + BK - 1) / BK : 1;
        w.nk        = w.partial == nullptr ? k : run_of_slice(pl.cut, slice, k).count;
        w.nk        = __builtin_amdgcn_readfirstlane(w.nk);
        w.ends_k    = k0 + w.nk == k;

        const InT*      A    = static_cast<const InT*>(args.A);
        const InT*      B    = static_cast<const InT*>(args.B);
        const long long from = (long long)k0 * BK;
        w.a = loop::scalar_pointer(A + w.x.a_at + (A_KMAJOR ? w.x.row0 * args.lda + from : w.x.row0 + from * args.lda));
        w.b = loop::scalar_pointer(B + w.x.b_at + (B_KMAJOR ? w.x.col0 * args.ldb + from : w.x.col0 + from * args.ldb));
        // Where the loads' range ends.  K-contiguous: with the operand's last row (rows past the
        // group's only reach rows of C that are not stored).  Else: with the group's K rows, so that
        // the rows of a last K tile past them read zeros, also those of the next group.
        const long long last = args.kind == product_kind::batch ? args.groups - 1 : 0;
        w.a_end = loop::scalar_pointer(A_KMAJOR ? A + last * args.stride_a + args.M * args.lda
                                                : A + w.x.a_at + w.x.k * args.lda);
        w.b_end = loop::scalar_pointer(
            (B_KMAJOR ? B + (args.kind == product_kind::sum ? 0 : (args.groups - 1) * args.stride_b) + args.N * args.ldb
                      : B + w.x.b_at + w.x.k * args.ldb)
            - args.b_skip);
        // (a group without rows to add up: its one K tile is all zeros)
        w.a_end = w.a_end < w.a ? w.a : w.a_end;
        w.b_end = w.b_end < w.b ? w.b : w.b_end;
        return w;
    }

    // A descriptor of the 2 GiB from `base` on, or of nothing.
    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t window(const void* base, bool there)
    {
        const unsigned long long p  = (unsigned long long)base;
        const unsigned int       lo = (unsigned int)__builtin_amdgcn_readfirstlane((unsigned int)p);
        const unsigned int       hi = (unsigned int)__builtin_amdgcn_readfirstlane((unsigned int)(p >> 32));
        const int records = there ? (int)loop::STORE_RANGE : 0;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | (unsigned long long)lo), 0,
                                                 records, 0x00020000);
    }

    // PIECE consecutive elements of T at a byte offset, as fp32.
    template<class T, int PIECE>
    struct piece
    {
        static constexpr int QUADS = PIECE * (int)sizeof(T) / 16;
        static_assert(PIECE == 1 || QUADS > 0, "one element, or 16 bytes at least");
        typename std::conditional<PIECE == 1, unsigned int, u32x4>::type raw[QUADS > 0 ? QUADS : 1];
        __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, unsigned int at, unsigned int wave_at)
        {
            if constexpr(PIECE == 1 && sizeof(T) == 2)
            {
                raw[0] = __builtin_amdgcn_raw_buffer_load_b16(from, at, wave_at, 0);
            }
            else if constexpr(PIECE == 1)
            {
                raw[0] = __builtin_amdgcn_raw_buffer_load_b32(from, at, wave_at, 0);
            }
            else
            {
#pragma unroll
                for(int q = 0; q < QUADS; ++q)
                {
                    raw[q] = __builtin_amdgcn_raw_buffer_load_b128(from, at + 16 * q, wave_at, 0);
                }
            }
        }
        __device__ __forceinline__ float get(int e) const
        {
            if constexpr(PIECE == 1)
            {
                if constexpr(sizeof(T) == 4)
                {
                    return __builtin_bit_cast(float, raw[0]);
                }
                else
                {
                    return (float)__builtin_bit_cast(T, (unsigned short)raw[0]);
                }
            }
            else if constexpr(sizeof(T) == 4)
            {
                // (a bit cast of a vector's element itself gives element 0: it goes through a variable)
                const unsigned int bits = raw[e / 4][e % 4];
                return __builtin_bit_cast(float, bits);
            }
            else
            {
                const unsigned short h = (unsigned short)(raw[0][e / 2] >> (16 * (e % 2)));
                return (float)__builtin_bit_cast(T, h);
            }
        }
    };

    template<class T, int PIECE>
    __device__ __forceinline__ static void store(const float (&y)[PIECE], __amdgpu_buffer_rsrc_t to, unsigned int at,
                                                 unsigned int wave_at)
    {
        // (a layer's C is not read again here, and its stores make the loop's operands no room in the
        // caches: 2 % of a backward pass of experts, 392 us against 400.  What a Newton-Schulz step
        // leaves the next one reads.)
        constexpr int NT = (EPI::scaled && !EPI::back) || EPI::loss == loss_use::slope ? 0 : 2;
        if constexpr(PIECE == 1 && sizeof(T) == 4)
        {
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned int, y[0]), to, at, wave_at, NT);
        }
        else if constexpr(PIECE == 1)
        {
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, to_out<T>(y[0])), to, at, wave_at, NT);
        }
        else if constexpr(sizeof(T) == 4)
        {
            static_assert(PIECE == 4, "one 16-byte piece");
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{y[0], y[1], y[2], y[3]}), to, at,
                                                   wave_at, NT);
        }
        else
        {
            typedef T t8 __attribute__((ext_vector_type(PIECE)));
            t8 v;
#pragma unroll
            for(int e = 0; e < PIECE; ++e)
            {
                v[e] = to_out<T>(y[e]);
            }
            if constexpr(PIECE == 8)
            {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, at, wave_at, NT);
            }
            else
            {
                typedef unsigned int u2 __attribute__((ext_vector_type(2)));
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, v), to, at, wave_at, NT);
            }
        }
    }

    // The wave's part of a finished tile, corner (row_w, col_w) in the workgroup's; MIRRORED: its
    // transpose, to the mirrored place (see has_mirror).
    template<bool MIRRORED, bool BY_ELEMENT = NARROW>
    __device__ __forceinline__ static void write(const product_args& args, const work& w, f32x4 (&acc)[TM][TN],
                                                 int row_w, int col_w, int lane, lds_char_ptr strip)
    {
        constexpr int PIECE = BY_ELEMENT ? 1 : 16 / (int)sizeof(OutT); // columns of a piece
        constexpr int PR    = HALF * 16 / PIECE; // pieces of a strip row
        constexpr int READS = (16 * PR + 63) / 64;
        constexpr bool UNEVEN = 16 * PR % 64 != 0; // the last read has lanes to spare
        constexpr int BLOCKS = MIRRORED ? TN : TM; // 16-row blocks of what is written
        const int       r16 = lane & 15, g = lane >> 4;
        const int       row0 = MIRRORED ? w.x.col0 : w.x.row0, col0 = MIRRORED ? w.x.row0 : w.x.col0;
        const int       rows = (MIRRORED ? args.N : w.x.m) - row0, cols = (MIRRORED ? w.x.m : args.N) - col0;
        const long long at   = w.x.c_at + row0 * args.ldc + col0;
        if constexpr(MIRRORED)
        {
            const int t = row_w;
            row_w       = col_w;
            col_w       = t;
        }
        constexpr bool SLOPE = EPI::loss == loss_use::slope;
        const float    alpha = EPI::back ? *args.alpha_at : args.alpha;
        const bool has_kept = (EPI::layer || EPI::kept) && args.kept != nullptr;
        const bool has_residual = EPI::residual && args.residual != nullptr;
        // (a tile without a mirror has no transposed place: its stores are dropped)
        const __amdgpu_buffer_rsrc_t to
            = window(static_cast<OutT*>(args.C) + at, !MIRRORED || has_mirror(w.x.row0, w.x.col0));
        const __amdgpu_buffer_rsrc_t kept_to
            = window(static_cast<InT*>(args.kept) + at, has_kept);
        const __amdgpu_buffer_rsrc_t from
            = window(static_cast<const ResT*>(args.residual) + at, has_residual);
        const __amdgpu_buffer_rsrc_t bias_from
            = window(static_cast<const InT*>(args.bias) + w.x.group * args.stride_bias + col0,
                     EPI::layer && args.bias != nullptr);
        const __amdgpu_buffer_rsrc_t diagonal_from
            = window(args.diagonal + w.x.group * args.stride_diagonal + row0,
                     EPI::diagonal != diagonal_use::none);

        // this lane's pieces of a strip: row and column, place in the strip, offset in C in elements
        int          piece_row[READS], piece_col[READS], strip_at[READS];
        unsigned int piece_off[READS];
#pragma unroll
        for(int q = 0; q < READS; ++q)
        {
            const int n  = q * 64 + lane;
            piece_row[q] = n / PR;
            piece_col[q] = n % PR * PIECE;
            strip_at[q]  = (UNEVEN && n >= 16 * PR ? 0 : piece_row[q] * PITCH + piece_col[q] * 4);
            piece_off[q] = (unsigned int)(piece_row[q] * args.ldc + piece_col[q]);
        }
        // outside: an element offset that is out of every descriptor's range in bytes
        auto offset = [&](int block, int p, int q, unsigned int size) {
            const int  row = row_w + 16 * block + piece_row[q], col = col_w + p * HALF * 16 + piece_col[q];
            const bool in  = row < rows && col < cols && (!UNEVEN || q * 64 + lane < 16 * PR);
            return in ? piece_off[q] * size : loop::STORE_RANGE;
        };
        auto wave_offset = [&](int block, int p, unsigned int size) {
            return (unsigned int)__builtin_amdgcn_readfirstlane(
                (unsigned int)((row_w + 16 * block) * args.ldc + col_w + p * HALF * 16) * size);
        };

        float bias[PASSES][READS][EPI::layer ? PIECE : 1];
#pragma unroll
        for(int p = 0; p < PASSES; ++p)
        {
#pragma unroll
            for(int q = 0; q < READS; ++q)
            {
                const int col = col_w + p * HALF * 16 + piece_col[q];
                if constexpr(EPI::layer)
                {
                    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
                    constexpr int        PAIRS = PIECE / 4;
                    const unsigned int   from_at = col < cols ? (unsigned int)col * 2 : loop::STORE_RANGE;
                    if constexpr(BY_ELEMENT)
                    {
                        const unsigned short b = __builtin_amdgcn_raw_buffer_load_b16(bias_from, from_at, 0, 0);
                        bias[p][q][0]          = (float)__builtin_bit_cast(InT, b);
                    }
#pragma unroll
                    for(int h = 0; h < PAIRS; ++h)
                    {
                        const u2 v = __builtin_amdgcn_raw_buffer_load_b64(bias_from, from_at + 8 * h, 0, 0);
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            const unsigned short b = (unsigned short)(v[e / 2] >> (16 * (e % 2)));
                            bias[p][q][4 * h + e]  = (float)__builtin_bit_cast(InT, b);
                        }
                    }
                }
            }
        }
        // what a column past the edge adds to its logit (-infinity: its power is 0), and the columns' numbers
        float past_edge[SLOPE ? PASSES : 1][READS][SLOPE ? PIECE : 1];
        const __amdgpu_buffer_rsrc_t records_from = window(args.records + row0, SLOPE);
        const int                    number0      = args.col_base + col0 + col_w;
        if constexpr(SLOPE)
        {
#pragma unroll
            for(int p = 0; p < PASSES; ++p)
            {
#pragma unroll
                for(int q = 0; q < READS; ++q)
                {
#pragma unroll
                    for(int e = 0; e < PIECE; ++e)
                    {
                        past_edge[p][q][e] = col_w + p * HALF * 16 + piece_col[q] + e < cols ? 0.0f : -__builtin_inff();
                    }
                }
            }
        }
        // residual pieces (and, by rows, what they are multiplied by) of AHEAD blocks are on their way
        constexpr int WANT = sizeof(OutT) == 4 || sizeof(ResT) == 4 || PER_CU > 1 || EPI::mirror ? 2 : 4;
        constexpr int AHEAD = BY_ELEMENT ? 1 : BLOCKS < WANT ? BLOCKS : WANT;
        piece<ResT, PIECE> residual[EPI::residual ? AHEAD : 1][PASSES][READS];
        float              by_row[EPI::diagonal == diagonal_use::rows ? AHEAD : 1][READS];
        u32x4              record[SLOPE ? AHEAD : 1][READS];
        auto fetch = [&](int block) {
            if constexpr(SLOPE)
            {
#pragma unroll
                for(int q = 0; q < READS; ++q)
                {
                    const int row = row_w + 16 * block + piece_row[q];
                    record[block % AHEAD][q] = __builtin_amdgcn_raw_buffer_load_b128(
                        records_from, row < rows ? row * (unsigned int)sizeof(loss_record) : loop::STORE_RANGE, 0, 0);
                }
            }
            if constexpr(EPI::residual)
            {
#pragma unroll
                for(int p = 0; p < PASSES; ++p)
                {
#pragma unroll
                    for(int q = 0; q < READS; ++q)
                    {
                        residual[block % AHEAD][p][q].load(from, offset(block, p, q, sizeof(ResT)),
                                                           has_residual ? wave_offset(block, p, sizeof(ResT)) : 0);
                    }
                }
            }
            if constexpr(EPI::diagonal == diagonal_use::rows)
            {
#pragma unroll
                for(int q = 0; q < READS; ++q)
                {
                    const int row = row_w + 16 * block + piece_row[q];
                    by_row[block % AHEAD][q]
                        = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                                        diagonal_from, row < rows ? row * 4u : loop::STORE_RANGE, 0, 0));
                }
            }
        };
#pragma unroll
        for(int block = 0; block < AHEAD; ++block)
        {
            fetch(block);
        }
        const float floor_at = args.act.kind == act_kind::relu ? 0.0f : -__builtin_inff();
#pragma unroll
        for(int block = 0; block < BLOCKS; ++block)
        {
            if constexpr(!MIRRORED)
            {
                loop::pin_row(acc[block]);
            }
#pragma unroll
            for(int p = 0; p < PASSES; ++p)
            {
#pragma unroll
                for(int t = 0; t < HALF; ++t)
                {
                    if constexpr(MIRRORED)
                    {
                        // block = tile column: its 16 columns are the strip's rows
                        const f32x4 v = acc[p * HALF + t][block];
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            *reinterpret_cast<lds_float*>(strip + (4 * g + e) * PITCH + (16 * t + r16) * 4) = v[e];
                        }
                    }
                    else
                    {
                        *reinterpret_cast<lds_f32x4*>(strip + r16 * PITCH + (16 * t + 4 * g) * 4) = acc[block][p * HALF + t];
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                const unsigned int wave_at = wave_offset(block, p, sizeof(OutT));
#pragma unroll
                for(int q = 0; q < READS; ++q)
                {
                    float z[PIECE], y[PIECE];
                    if constexpr(BY_ELEMENT)
                    {
                        const float v = *reinterpret_cast<const lds_float*>(strip + strip_at[q]);
                        z[0]          = EPI::scaled ? alpha * v : v;
                    }
#pragma unroll
                    for(int h = 0; h < PIECE / 4; ++h)
                    {
                        const f32x4 v = *reinterpret_cast<const lds_f32x4*>(strip + strip_at[q] + 16 * h);
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            z[4 * h + e] = EPI::scaled ? alpha * v[e] : v[e];
                        }
                    }
                    const unsigned int off = offset(block, p, q, sizeof(OutT));
#pragma unroll
                    for(int e = 0; e < PIECE; ++e)
                    {
                        if constexpr(EPI::layer)
                        {
                            z[e] += bias[p][q][e];
                        }
                        y[e] = z[e];
                        if constexpr(SLOPE)
                        {
                            // (the power is the hardware's, 1 ulp; below 2^-126 it gives 0, as for a row without a gradient,
                            // whose lse is infinite)
                            const u32x4        r = record[block % AHEAD][q];
                            const unsigned int lse_bits = r[0], factor_bits = r[1];
                            y[e] = __builtin_bit_cast(float, factor_bits)
                                   * __builtin_amdgcn_exp2f(__builtin_fmaf(z[e], args.alpha, past_edge[p][q][e])
                                                            - __builtin_bit_cast(float, lse_bits));
                        }
                        if constexpr(EPI::logistic)
                        {
                            const float c = __builtin_amdgcn_fmed3f(z[e], -1.0e4f, 1.0e4f); // (see activate)
                            y[e]          = z[e] * logistic(c * (args.act.k1 + args.act.k3 * c * c));
                        }
                        else if constexpr(EPI::layer)
                        {
                            y[e] = z[e] < floor_at ? floor_at : z[e];
                        }
                        if constexpr(EPI::residual)
                        {
                            const float r = residual[block % AHEAD][p][q].get(e);
                            if constexpr(EPI::diagonal == diagonal_use::rows)
                            {
                                y[e] += (args.beta + alpha * by_row[block % AHEAD][q]) * r;
                            }
                            else
                            {
                                y[e] += EPI::scaled ? args.beta * r : r;
                            }
                        }
                    }
                    if constexpr(SLOPE)
                    {
                        // (few pieces hold their row's target)
                        const u32x4        r = record[block % AHEAD][q];
                        const unsigned int factor_bits = r[1];
                        const int          hit = (int)r[2] - (number0 + p * HALF * 16 + piece_col[q]);
                        if(__any(hit >= 0 && hit < PIECE))
                        {
#pragma unroll
                            for(int e = 0; e < PIECE; ++e)
                            {
                                y[e] -= hit == e ? __builtin_bit_cast(float, factor_bits) : 0.0f;
                            }
                        }
                    }
                    if constexpr(EPI::diagonal == diagonal_use::split)
                    {
                        // of a piece at most one element is the diagonal's: it goes to the vector
                        // (every lane stores, all but its owner out of range), and a zero to C
                        const int row = row0 + row_w + 16 * block + piece_row[q];
                        const int ahead = row - (col0 + col_w + p * HALF * 16 + piece_col[q]);
                        float     own   = 0.0f;
#pragma unroll
                        for(int e = 0; e < PIECE; ++e)
                        {
                            own  = ahead == e ? y[e] : own;
                            y[e] = ahead == e ? 0.0f : y[e];
                        }
                        if constexpr(!MIRRORED)
                        {
                            const bool mine = ahead >= 0 && ahead < PIECE && row < args.N
                                              && (!UNEVEN || q * 64 + lane < 16 * PR);
                            __builtin_amdgcn_raw_buffer_store_b32(
                                __builtin_bit_cast(unsigned int, own), diagonal_from,
                                mine ? (unsigned int)(row - row0) * 4u : loop::STORE_RANGE, 0, 0);
                        }
                    }
                    if constexpr(EPI::layer || EPI::kept)
                    {
                        const unsigned int kept_at = offset(block, p, q, 2);
                        store<InT, PIECE>(EPI::layer ? z : y, kept_to, kept_at,
                                          has_kept ? wave_offset(block, p, 2) : 0);
                    }
                    store<OutT, PIECE>(y, to, off, wave_at);
                }
                asm volatile("" ::: "memory");
            }
            if(block + AHEAD < BLOCKS)
            {
                fetch(block + AHEAD);
            }
        }
    }

    // The statistics of the wave's rows over its columns, straight from the accumulators: a lane has 4 TN of a row's 16 TN
    // columns, four lanes meet.  What lies past the edge counts as -infinity.  (No load here: it
    // would wait for those of the next tile, which are on their way.  Keeping a target's logit where it comes by did, 557 us
    // against 475 for 2048 x 65536 x 2048.)
    __device__ __forceinline__ static void write_parts(const product_args& args, const work& w, f32x4 (&acc)[TM][TN], int row_w,
                                                       int col_w, int lane)
    {
        const int r16 = lane & 15, g = lane >> 4;
        const int rows = w.x.m - w.x.row0 - row_w, cols = args.N - w.x.col0 - col_w;
        float     past_edge[TN][4], top[TM], sum[TM];
#pragma unroll
        for(int j = 0; j < TN; ++j)
        {
#pragma unroll
            for(int e = 0; e < 4; ++e)
            {
                past_edge[j][e] = 16 * j + 4 * g + e < cols ? 0.0f : -__builtin_inff();
            }
        }
#pragma unroll
        for(int block = 0; block < TM; ++block)
        {
            loop::pin_row(acc[block]);
            float x[TN][4], most = -__builtin_inff();
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    x[j][e] = __builtin_fmaf(acc[block][j][e], args.alpha, past_edge[j][e]);
                    most    = __builtin_fmaxf(most, x[j][e]);
                }
            }
            const float from = most > -__builtin_inff() ? most : 0.0f;
            float       s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for(int j = 0; j < TN; ++j)
            {
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    s[e] += __builtin_amdgcn_exp2f(x[j][e] - from);
                }
            }
            top[block] = most;
            sum[block] = (s[0] + s[1]) + (s[2] + s[3]);
        }
#pragma unroll
        for(int block = 0; block < TM; ++block)
        {
            const float most = top[block];
            float       all  = __builtin_fmaxf(most, __shfl_xor(most, 16));
            all              = __builtin_fmaxf(all, __shfl_xor(all, 32));
            float s          = sum[block] * (most == all ? 1.0f : __builtin_amdgcn_exp2f(most - all));
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            const int row = 16 * block + r16;
            if(g == 0 && row < rows && cols > 0)
            {
                args.parts[(long long)(w.x.row0 + row_w + row) * args.parts_of_row + (w.x.col0 + col_w) / (16 * TN)]
                    = {all, s};
            }
        }
    }

    // A slice's part of a tile, in fp32: [BM][BN].
    __device__ __forceinline__ static void write_partial(const work& w, f32x4 (&acc)[TM][TN], int row_w, int col_w,
                                                         int lane, lds_char_ptr strip)
    {
        constexpr int PR = HALF * 4, READS = 16 * PR / 64; // pieces of 4 columns
        static_assert(16 * PR % 64 == 0, "whole reads");
        const int                    r16 = lane & 15, g = lane >> 4;
        const __amdgpu_buffer_rsrc_t to = window(w.partial, true);
        const int                    row = lane / PR, col = lane % PR * 4;
        const unsigned int           at = (unsigned int)((row * BN + col) * 4);
#pragma unroll
        for(int block = 0; block < TM; ++block)
        {
            loop::pin_row(acc[block]);
#pragma unroll
            for(int p = 0; p < PASSES; ++p)
            {
#pragma unroll
                for(int t = 0; t < HALF; ++t)
                {
                    *reinterpret_cast<lds_f32x4*>(strip + r16 * PITCH + (16 * t + 4 * g) * 4) = acc[block][p * HALF + t];
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                const unsigned int wave_at
                    = (unsigned int)__builtin_amdgcn_readfirstlane(((row_w + 16 * block) * BN + col_w + p * HALF * 16) * 4);
#pragma unroll
                for(int q = 0; q < READS; ++q)
                {
                    const f32x4 v = *reinterpret_cast<const lds_f32x4*>(strip + (q * (64 / PR) + row) * PITCH + col * 4);
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, at + q * (64 / PR) * BN * 4,
                                                           wave_at, 0);
                }
                asm volatile("" ::: "memory");
            }
        }
    }

    // Adds up the slices of the cut tiles, in their order, and finishes them.  A thread takes 8
    // columns of a row; a workgroup FINISH_ROWS rows of a tile.
    static constexpr int FINISH_ROWS = THREADS * 8 / BN, FINISH_PARTS = BM / FINISH_ROWS;
    __device__ __forceinline__ static void finish_cut(const product_args& args)
    {
        __shared__ int table_raw[TABLE / 4];
        lds_int*       table = (lds_int*)table_raw;
        const plan     pl = make_plan(args, table, args.workgroups);
        const int      parts = pl.cut.cut * FINISH_PARTS;
        for(int part = blockIdx.x; part < parts; part += gridDim.x)
        {
            const int          t = part / FINISH_PARTS;
            const product_item x = locate(args, pl, pl.cut.whole + t);
            const int          r = (part - t * FINISH_PARTS) * FINISH_ROWS + (int)threadIdx.x / (BN / 8);
            const int          c = (int)threadIdx.x % (BN / 8) * 8, row = x.row0 + r, col = x.col0 + c;
            if(row >= x.m || col >= args.N)
            {
                continue;
            }
            const float* from = args.partials + (long long)t * pl.cut.slices * (BM * BN) + r * BN + c;
            f32x4        lo{0.0f, 0.0f, 0.0f, 0.0f}, hi{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for(int s = 0; s < pl.cut.slices; ++s)
            {
                lo += *reinterpret_cast<const f32x4*>(from + (long long)s * (BM * BN));
                hi += *reinterpret_cast<const f32x4*>(from + (long long)s * (BM * BN) + 4);
            }
            const float sum[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if constexpr(NARROW)
            {
#pragma unroll
                for(int e = 0; e < 8; ++e)
                {
                    if(col + e < args.N)
                    {
                        finish_element<InT, OutT, ResT>(args, x, row, col + e, sum[e]);
                    }
                }
            }
            else
            {
                finish_piece<InT, OutT, ResT>(args, x, row, col, sum);
            }
        }
    }

    // The K loop and its load stream: see solo_gemm::run; here with a ring of 2 or 3.
    __device__ __forceinline__ static void run(const product_args& args)
    {
        __shared__ __attribute__((aligned(1024))) char lds_raw[LDS_BYTES];
        lds_char_ptr lds   = (lds_char_ptr)lds_raw;

        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wave_m = wave / 2, wave_n = wave % 2;
        const plan pl = make_plan(args, reinterpret_cast<lds_int*>(lds + RING_BYTES + 4 * STRIP), (int)gridDim.x);
        const int  total = pl.positions, hop = pl.hop;
        int        pos = pl.begin;
        if(pos >= total)
        {
            return;
        }

        const long long a_ld = args.lda, b_ld = args.ldb;
        const long long a_step = BK * (A_KMAJOR ? 1 : a_ld), b_step = BK * (B_KMAJOR ? 1 : b_ld);
        typename loop::op_a   oa;
        typename loop::op_b   ob;
        typename loop::addr_a la;
        typename loop::addr_b lb;
        oa.init(wave, lane, a_ld, wave_m * loop::WTM);
        ob.init(wave, lane, b_ld, wave_n * loop::WTN);
        la.init(wave, lane, a_ld);
        lb.init(wave, lane, b_ld);
        // a last K tile that K-contiguous operands hold only in part (all items have the same K)
        const int  k_tail   = A_KMAJOR || B_KMAJOR ? args.K % BK : 0;
        const bool k_ragged = k_tail != 0;
        const typename loop::addr_a la_tail = la.for_tail(lane, wave, k_tail);
        const typename loop::addr_b lb_tail = lb.for_tail(lane, wave, k_tail);

        work       cur  = decode(args, pl, pos);
        const InT* a_src = cur.a;
        const InT* b_src = cur.b;
        const InT* a_end = cur.a_end;
        const InT* b_end = cur.b_end;
        int        stream_left = cur.nk, stream_pos = pos + hop;
        bool       stream_ends = cur.ends_k;
        auto advance = [&]() {
            a_src += a_step;
            b_src += b_step;
            if(--stream_left == 0)
            {
                // (past its last item the stream starts over: the loads go where nobody reads)
                const work nx = decode(args, pl, stream_pos < total ? stream_pos : pl.begin);
                a_src         = nx.a;
                b_src         = nx.b;
                a_end         = nx.a_end;
                b_end         = nx.b_end;
                stream_left   = nx.nk;
                stream_ends   = nx.ends_k;
                stream_pos += hop;
            }
        };
        auto partial_tile = [&]() { return k_ragged && stream_ends && stream_left == 1; };

        const unsigned int lds_addr   = (unsigned int)(size_t)lds;
        const unsigned int wave_block = lds_addr + wave * 1024;
        lds_char_ptr       strip      = lds + RING_BYTES + wave * STRIP;
        u32x4              fa[2][TM], fb[2][TN];
        constexpr int LOADS_A = VM_LOADS / 4, LOADS_B = VM_LOADS - LOADS_A, MFMAS = loop::MFMAS;
        using plan_b = typename loop::template load_plan<2, (MFMAS - 2) / LOADS_B, 0, LOADS_B>;
        using plan_a = typename loop::template load_plan<1, (MFMAS >= 32 ? 4 : 2), LOADS_B, LOADS_A>;
        {
            const bool part = partial_tile();
            loop::issue_loads(std::make_integer_sequence<int, VM_LOADS>{}, la.or_else(part, la_tail),
                              lb.or_else(part, lb_tail), wave_block, loop::descriptor(a_src, a_end),
                              loop::descriptor(b_src, b_end));
        }
        advance();
        if constexpr(RING == 3)
        {
            const bool part = partial_tile();
            loop::issue_loads(std::make_integer_sequence<int, VM_LOADS>{}, la.or_else(part, la_tail),
                              lb.or_else(part, lb_tail), wave_block + STAGE, loop::descriptor(a_src, a_end),
                              loop::descriptor(b_src, b_end));
            advance();
        }
        bool part_prev = partial_tile();
        loop::issue_loads(std::make_integer_sequence<int, LOADS_B>{}, la.or_else(part_prev, la_tail),
                          lb.or_else(part_prev, lb_tail), wave_block + (RING - 1) * STAGE,
                          loop::descriptor(a_src, a_end), loop::descriptor(b_src, b_end));
        const InT* a_prev     = a_src;
        const InT* b_prev     = b_src;
        const InT* a_end_prev = a_end;
        const InT* b_end_prev = b_end;
        advance();
        // (behind tile 0, the first: the loads of the ring's other tiles may still be in flight)
        __builtin_amdgcn_s_waitcnt(loop::waitcnt_imm((RING - 2) * VM_LOADS + LOADS_B));
        __builtin_amdgcn_s_barrier();
        loop::read_first(std::make_integer_sequence<int, TM>{}, std::make_integer_sequence<int, TN>{}, oa, ob, lds_addr,
                         fa[0], fb[0]);

        unsigned int here = 0; // stage (byte offset) of the tile the MFMAs are on
        for(;;)
        {
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
#pragma unroll
            for(int i = 0; i < TM; ++i)
            {
                loop::settle_row(acc[i]);
            }
            for(int it = 0; it < cur.nk; ++it)
            {
                const unsigned int there = here + STAGE == RING_BYTES ? 0 : here + STAGE;
                const unsigned int late  = here == 0 ? RING_BYTES - STAGE : here - STAGE; // of the last tile on its way
                const bool         part  = partial_tile();
                const auto la0 = la.or_else(part_prev, la_tail), la1 = la.or_else(part, la_tail);
                const auto lb0 = lb.or_else(part_prev, lb_tail), lb1 = lb.or_else(part, lb_tail);
                const typename loop::step_ctx c0{oa, ob, la0, lb0, lds_addr + here, wave_block + late,
                                                 loop::descriptor(a_prev, a_end_prev),
                                                 loop::descriptor(b_prev, b_end_prev)};
                const typename loop::step_ctx c1{oa, ob, la1, lb1, lds_addr + there, wave_block + here,
                                                 loop::descriptor(a_src, a_end), loop::descriptor(b_src, b_end)};
                __builtin_amdgcn_s_waitcnt(loop::waitcnt_imm(63));
                loop::template step<1, plan_a>(c0, fa[0], fb[0], fa[1], fb[1], acc);
                // (the next tile has landed; with a ring of 3 the one behind it may be in flight)
                __builtin_amdgcn_s_waitcnt(loop::waitcnt_imm((RING - 2) * VM_LOADS));
                __builtin_amdgcn_s_barrier();
                loop::template step<0, plan_b>(c1, fa[1], fb[1], fa[0], fb[0], acc);
                a_prev     = a_src;
                b_prev     = b_src;
                a_end_prev = a_end;
                b_end_prev = b_end;
                part_prev  = part;
                advance();
                here = there;
            }
            // (the MFMAs are invisible to the compiler: their result latency is covered by hand)
            asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
            if constexpr(EPI::loss == loss_use::parts)
            {
                write_parts(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane);
            }
            else if constexpr(EPI::loss == loss_use::slope)
            {
                write<false>(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
            }
            else if constexpr(!EPI::mirror)
            {
                if(cur.partial != nullptr)
                {
                    // (read next by the kernel that adds the slices up: no streaming hint)
                    write_partial(cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
                }
                else if(ANYWHERE && cur.x.col0 + BN <= args.N)
                {
                    write<false, NARROW && !ANYWHERE>(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
                }
                else
                {
                    write<false>(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
                }
            }
            else
            {
                write<false>(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
                write<true>(args, cur, acc, wave_m * loop::WTM, wave_n * loop::WTN, lane, strip);
            }
            pos += hop;
            if(pos >= total)
            {
                break;
            }
            cur = decode(args, pl, pos);
            loop::read_first(std::make_integer_sequence<int, TM>{}, std::make_integer_sequence<int, TN>{}, oa, ob,
                             lds_addr + here, fa[0], fb[0]);
        }
        // the loads past the last item are still in flight
        __builtin_amdgcn_s_waitcnt(loop::waitcnt_imm(0));
    }
};

template<class Impl>
__global__ void __launch_bounds__(Impl::THREADS) tiled_finish_entry(const product_args args)
{
    Impl::finish_cut(args);
}

template<class Impl>
__global__ void __launch_bounds__(Impl::THREADS, Impl::PER_CU) tiled_product_entry(const product_args args)
{
    Impl::run(args);
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_TILED_PRODUCT_HPP
