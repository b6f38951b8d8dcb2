/*
 * C ABI of librocm_wmma_gemm_gfx950.so -- the drop-in boundary of the GEMM path.
 *
 * The first four functions are exactly the symbols the reference's runtime
 * loader resolves with dlsym (reference rocm_wmma_gemm/include/rocm_wmma_gemm/
 * kernel_loader.hpp:53-54,110-113) and that its arch library defines
 * (reference rocm_wmma_gemm/src/gemm.cpp:219-250).  The rest are additions with
 * no counterpart in the reference: introspection and tuning hooks.
 *
 * Conventions for every gemm entry point:
 *   C (M x N) = A (M x K) * B (K x N); C is overwritten; operands are dense and
 *   packed in the stated layout; layout_* is 0 for row-major, 1 for column-major;
 *   batch b uses A + b*M*K, B + b*K*N, C + b*M*N (elements);
 *   `stream` is the ADDRESS of the caller's hipStream_t (a hipStream_t*), not the
 *   handle itself; the work is enqueued there and the call returns at once;
 *   all pointers are device pointers owned by the caller;
 *   a layout value outside {0,1} makes the call a no-op (reference behaviour,
 *   src/gemm.cpp:243); M, N or batch_count of 0 is a no-op; K of 0 zero-fills C.
 */
#ifndef ROCM_WMMA_GEMM_C_H
#define ROCM_WMMA_GEMM_C_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* fp16 A,B -> fp16 C.  Replaces reference src/gemm.cpp:247 (DEFINE_C_DISPATCH(f16_f16, half, half)). */
void rocm_wmma_gemm_f16_f16(void* C, void* A, void* B, size_t M, size_t N, size_t K,
                            size_t batch_count, int layout_c, int layout_a, int layout_b,
                            void* stream);

/* fp16 A,B -> fp32 C.  Replaces reference src/gemm.cpp:248. */
void rocm_wmma_gemm_f32_f16(void* C, void* A, void* B, size_t M, size_t N, size_t K,
                            size_t batch_count, int layout_c, int layout_a, int layout_b,
                            void* stream);

/* bf16 A,B -> bf16 C.  Replaces reference src/gemm.cpp:249. */
void rocm_wmma_gemm_bf16_bf16(void* C, void* A, void* B, size_t M, size_t N, size_t K,
                              size_t batch_count, int layout_c, int layout_a, int layout_b,
                              void* stream);

/* bf16 A,B -> fp32 C.  Replaces reference src/gemm.cpp:250. */
void rocm_wmma_gemm_f32_bf16(void* C, void* A, void* B, size_t M, size_t N, size_t K,
                             size_t batch_count, int layout_c, int layout_a, int layout_b,
                             void* stream);

/* ---- additions (no counterpart in the reference) ------------------------ */

/* type_idx values, in the reference launcher's order (kernel_launcher.hpp:78-83). */
#define ROCM_WMMA_GEMM_TYPE_F16_F16 0
#define ROCM_WMMA_GEMM_TYPE_F32_F16 1
#define ROCM_WMMA_GEMM_TYPE_BF16_BF16 2
#define ROCM_WMMA_GEMM_TYPE_F32_BF16 3

/* Status codes of the additions that return int (the four reference entry points return
 * void, as in the reference). */
#define ROCM_WMMA_GEMM_OK 0
#define ROCM_WMMA_GEMM_ERR_VARIANT (-1)  /* the forced variant cannot run this problem */
#define ROCM_WMMA_GEMM_ERR_ARGUMENT (-2) /* type index, variant index or layout code out of range */
#define ROCM_WMMA_GEMM_ERR_SCRATCH (-3)  /* the call needs more scratch memory than the fixed buffer holds */
#define ROCM_WMMA_GEMM_ERR_RUNTIME (-4)  /* the HIP runtime reported an error (symbol lookup, launch) */
#define ROCM_WMMA_GEMM_ERR_LIMIT (-5)    /* M, N or K beyond 31 bits, tile grid too large, or no kernel built */

/* Description of one compiled kernel variant. */
typedef struct rocm_wmma_gemm_variant_info
{
    int block_m, block_n, block_k; /* workgroup tile */
    int warps_m, warps_n;          /* wave grid inside the workgroup */
    int warp_tile_m, warp_tile_n;  /* 32x32 MFMA tiles per wave (0: a 16-wide side of the streaming kernel's tile) */
    int pipeline;                  /* 0 = register-staged general path, 1 = direct-to-LDS, 2 = direct-to-LDS ping-pong, 3, 4 = 1, 2 on the 16x16x32 MFMA, 5 = one wave per SIMD, persistent workgroups, 6 = 1 with a ring of 4 tiles at BLOCK_K 64, 7 = whole-K streaming kernel (tiles of 16 to 128 rows by 16 to 64 columns, one workgroup per tile over all of K, for skinny and small problems) */
    int lds_bytes;                 /* static LDS per workgroup */
    int threads;                   /* workgroup size */
} rocm_wmma_gemm_variant_info;

/* "gfx950": the architecture this library was compiled for. */
const char* rocm_wmma_gemm_arch(void);

/* Number of compiled tile variants; fills *info for variant in [0, count). Returns 0 on success. */
int rocm_wmma_gemm_variant_count(void);
int rocm_wmma_gemm_variant_info_get(int variant, rocm_wmma_gemm_variant_info* info);

/* Which variant the dispatcher would pick for this problem (the table built from
 * gemm_config_gfx950_*.json, then shape heuristics).  type_idx as above.
 * Also reports the swizzle (band height of the tile walk: g > 0 bands of g tile rows,
 * g < 0 bands of -g tile columns) and the split field: s > 1 = every
 * tile's K range is cut into s slices (added up by a second kernel; on the whole-K streaming
 * kernel, pipeline 7, s = 2, 4 or 8 workgroups share a tile and the last of them to finish
 * adds the parts up inside the one launch); -s < -1 = only the tiles of the last, partial
 * wave over the compute units are cut into s slices; -1 = the persistent kernel's
 * workgroups each take the same number of K tiles of the sequence of all K tiles of the
 * launch, wherever the tile borders fall, and the cut tiles are added up afterwards (other
 * kernels read -1 as 1); 1 = no split.  Returns the variant index, or -1 for invalid
 * arguments. */
int rocm_wmma_gemm_select(size_t M, size_t N, size_t K, int type_idx, int layout_c, int layout_a,
                          int layout_b, int* swizzle, int* split_k);
/* The same for a strided batch of batch_count problems of this shape: the dispatcher counts
 * the tiles of the whole batch when it weighs tile sizes and splits, so the answer can differ
 * from the single problem's. */
int rocm_wmma_gemm_select_batched(size_t M, size_t N, size_t K, size_t batch_count, int type_idx,
                                  int layout_c, int layout_a, int layout_b, int* swizzle,
                                  int* split_k);

/* rocm_wmma_gemm_select_batched, also reporting the plan's fourth field: touch_ahead d > 0 =
 * the persistent kernel, beside the loads of a K tile, touches the cache lines of the K tile
 * d tiles further on (one dword per line from two waves of each workgroup, the workgroups
 * that share an operand panel touching different quarters), so that those lines are on
 * their way into the XCD's L2 a tile time before the loads that need them; it pays for a
 * long K whose operands outgrow the memory-side cache and costs a few percent elsewhere,
 * so the tuner decides.  0 = off; other kernels ignore it.  The value carries a second small
 * field in bits 4-7: c > 0 = the persistent kernel walks the K tiles of a tile in runs of
 * 2^(c-1) and, within every 8 runs, the workgroups of XCD x start at run x and wrap round,
 * so that the XCDs that share an operand panel are never on the same run (each finds in the
 * memory-side cache what another fetched first, instead of all of them waiting for memory at
 * once); the sums of an element are added in that order, the same in every call.  Worth
 * 7-10 % on operands beyond that cache with a K-contiguous operand, nothing elsewhere.  And a
 * third in bits 8-9: c > 0 = within every aligned group of 2^c K tiles the workgroup of tile
 * (i, j) starts at tile (i + j) mod 2^c of the group and wraps round, so that the workgroups
 * of an XCD that share an operand panel ask for a line at different times and all but the
 * first find it in L2: worth 14-17 % on the same problems; the dispatcher's estimate sets
 * groups of 4 there, the tuner decides per entry.  Both leave the sums of an element in one
 * fixed order, the same in every call.  (JSON keys: "touch_ahead" for bits 0-3, "k_runs" for
 * the run length, "k_group" for the group size.) */
int rocm_wmma_gemm_select_ex(size_t M, size_t N, size_t K, size_t batch_count, int type_idx, int layout_c,
                             int layout_a, int layout_b, int* swizzle, int* split_k, int* touch_ahead);

/* Same computation as the four entry points above, but with the tile variant,
 * swizzle and split field (see above) forced (tuner hook).  Returns ROCM_WMMA_GEMM_OK,
 * ROCM_WMMA_GEMM_ERR_VARIANT if the variant cannot run this problem, or another of the
 * status codes above. */
int rocm_wmma_gemm_run_variant(int type_idx, int variant, int swizzle, int split_k, void* C,
                               void* A, void* B, size_t M, size_t N, size_t K,
                               size_t batch_count, int layout_c, int layout_a, int layout_b,
                               void* stream);

/* rocm_wmma_gemm_run_variant with the plan's touch_ahead field (both parts of it) forced too
 * (see rocm_wmma_gemm_select_ex). */
int rocm_wmma_gemm_run_variant_ex(int type_idx, int variant, int swizzle, int split_k, int touch_ahead,
                                  void* C, void* A, void* B, size_t M, size_t N, size_t K,
                                  size_t batch_count, int layout_c, int layout_a, int layout_b,
                                  void* stream);

/* Adds a tile variant that was compiled outside this library (the tuner builds
 * rocm_wmma_gemm_amd/csrc/kernel_jit.hip for one tuple, type pair and pair of operand layouts
 * and passes that library's rwg_jit_kernels here: nine entry points, for the three load modes,
 * 16-byte unguarded, 16-byte guarded, 2-byte, then the twins of the first two that walk K in
 * runs (see rocm_wmma_gemm_select_ex), then those twins with non-temporal loads of B and of A;
 * null where the pipeline or tile has none).  The
 * variant gets the next index after the compiled ones and runs through
 * rocm_wmma_gemm_run_variant like any other; registering the same tuple again for another
 * type pair or layout pair adds those kernels to the same index.  operand *_kmajor: 1 if K is
 * the operand's contiguous dimension in the kernel's view (C row-major: A row-major, B
 * column-major; a column-major C swaps the operands).  Returns the variant index,
 * ROCM_WMMA_GEMM_ERR_VARIANT if the library already holds a compiled variant of this
 * description, ROCM_WMMA_GEMM_ERR_ARGUMENT for a tuple no kernel can have, or
 * ROCM_WMMA_GEMM_ERR_LIMIT when 64 variants have been registered.  The library that holds
 * the kernels must stay loaded.  The role of the reference tuner's run-time compilation
 * (reference rocm_wmma_gemm/config/tuner.cpp:237-454), split into compile (tuner) and
 * launch (library). */
int rocm_wmma_gemm_register_variant(int block_m, int block_n, int block_k, int warps_m, int warps_n,
                                    int pipeline, int type_idx, int a_kmajor, int b_kmajor,
                                    const void* const* kernels);

/* Gives the current device's library-owned scratch buffer back (split-K partial sums and
 * padded operand copies live there: 256 MiB from the first call that needs it, more when a
 * call needs more).  Waits for the device to finish first.  Returns 0 when the buffer is
 * gone or was never there, 1 when it was kept because a call on a capturing stream has
 * used it (a graph may hold its address), ROCM_WMMA_GEMM_ERR_RUNTIME without a device.
 * The next call that needs scratch memory allocates again.  Also puts the arrival counters
 * of shared tiles back to zero (they return to zero by themselves after every launch that
 * runs to its end; a kernel killed in flight may leave one counting, which later launches
 * ignore anyway because every launch tags its counts).  No counterpart in the reference,
 * which owns no memory. */
int rocm_wmma_gemm_workspace_release(void);

/* Size of the fixed per-GPU scratch buffer behind rocm_wmma_gemm_noalloc. */
#define ROCM_WMMA_GEMM_NOALLOC_SCRATCH_BYTES (64u << 20)

/* The same computation as the four reference entry points (type_idx picks the type pair),
 * for callers that cannot allocate device memory: code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc.  No counterpart in the reference, whose
 * kernels need no scratch memory at all.  Here split-K partial sums and zero-padded copies
 * of ragged operands do; the other entry points keep them in a buffer that the library
 * allocates and grows on demand, this one keeps them in a fixed array of
 * ROCM_WMMA_GEMM_NOALLOC_SCRATCH_BYTES that is part of the library's code object on every
 * GPU (held from the first use of the library on that GPU until the process ends), and
 * calls neither hipMalloc nor hipFree nor anything else that allocates.
 *   - A call whose plan needs more scratch memory than the array holds fails with
 *     ROCM_WMMA_GEMM_ERR_SCRATCH and enqueues nothing (of the shapes the library is
 *     tuned for: K = 65536 at M = N = 1024, which wants 128 MiB of partial tiles, and
 *     (4095, 5121, 3001), which wants 56 MiB of padded copies plus its partial tiles).
 *     Extents whose rows do not start on 16 bytes have a second plan, the nearest tuned
 *     shape's, which needs less or none: it is tried before the call fails, so that such a
 *     call may run on another plan here than through the other entry points, and slower.
 *     Calls that need no scratch memory (whole tiles, no split) have no size limit.
 *   - The first call on a GPU looks the array's address up (hipGetSymbolAddress); make that
 *     call outside graph capture.
 *   - Every call on a GPU uses that GPU's one array, which keeps the previous call's
 *     contents; nothing has to start at zero (each kernel writes what a later one reads).
 *     Calls of THIS entry point that overlap on one GPU (two streams, two threads, replays
 *     of two captured graphs) race on the array and on the arrival counters of shared
 *     tiles that go with it: order them.  Calls of the other entry points may overlap with
 *     them freely: those use the library's allocated buffer and counters of their own.
 * Returns ROCM_WMMA_GEMM_OK or one of the codes above; a layout code outside {0, 1} is
 * ROCM_WMMA_GEMM_ERR_ARGUMENT here rather than a silent no-op. */
int rocm_wmma_gemm_noalloc(int type_idx, void* C, void* A, void* B, size_t M, size_t N, size_t K,
                           size_t batch_count, int layout_c, int layout_a, int layout_b,
                           void* stream);

/* ---------------------------------------------------------------------------------------
 * Layer products: additions with no counterpart in the reference.
 *
 * A linear layer C = act(A B + bias) + residual on rows of activations, the same for groups of
 * rows with a weight each (experts), and their gradients.  A (M x K), C (M x N) and the
 * gradients of both are row-major; B (K x N) is row-major (layout_b 0) or column-major (1: weights
 * stored N x K).  type_idx names the types of C and of A and B as above; bias has A's type,
 * residual and dbias C's, preact (the sum before the activation, M x N) A's, as dC.  Everything is added up
 * and activated in fp32, each output rounded once.  `stream` is the address of a hipStream_t;
 * the calls enqueue and return.  M, N, K up to 2^31 - 256; a size of 0 leaves the sums empty.
 * --------------------------------------------------------------------------------------- */
#define ROCM_WMMA_GEMM_ACT_NONE 0
#define ROCM_WMMA_GEMM_ACT_RELU 1
#define ROCM_WMMA_GEMM_ACT_SILU 2 /* x / (1 + e^-x) */
#define ROCM_WMMA_GEMM_ACT_GELU 3 /* 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) */

/* Most groups of one grouped call. */
#define ROCM_WMMA_GEMM_MAX_GROUPS 512

typedef struct rocm_wmma_gemm_epilogue
{
    const void* bias; /* N values (grouped: N per group), or NULL */
    const void* residual; /* M x N, added behind the activation, or NULL; may be C itself */
    void*       preact; /* M x N, receives A B + bias, or NULL */
    int         activation; /* ROCM_WMMA_GEMM_ACT_* */
} rocm_wmma_gemm_epilogue;

/* C = act(A B + bias) + residual.  epilogue may be NULL: C = A B. */
int rocm_wmma_gemm_linear(int type_idx, void* C, const void* A, const void* B, size_t M, size_t N, size_t K,
                          int layout_b, const rocm_wmma_gemm_epilogue* epilogue, void* stream);

/* With dZ = dC act'(preact) (preact may be NULL for ROCM_WMMA_GEMM_ACT_NONE):
 * dA = dZ B^T (M x K), dB = A^T dZ (in B's layout), dbias = sum of dZ's rows (N); a NULL result is not
 * computed.  accumulate 1: dB and dbias are added to.  dZ is rounded to A's type before it is
 * multiplied (not in dbias), so that behind an activation gradients of type F32 hold dZ's 8 (bf16) or 11 (f16) bits; it and the partial sums of dbias live in the library's scratch buffer, so a call
 * on a capturing stream for which that buffer is too small returns ROCM_WMMA_GEMM_ERR_SCRATCH, and so does
 * any call for which they take more than 16 GiB (2 bytes an element of dZ, where there is an activation or dC's rows
 * do not start on 16 bytes, and N / 8 bytes a row for dbias).
 * (The gradient of the residual is dC.) */
int rocm_wmma_gemm_linear_backward(int type_idx, void* dA, void* dB, void* dbias, const void* dC, const void* A,
                                   const void* B, const void* preact, size_t M, size_t N, size_t K, int layout_b,
                                   int activation, int accumulate, void* stream);

/* The same for `groups` weights (B: groups x K x N, one after the other) and rows sorted by group:
 * group e has rows offsets[e] .. offsets[e+1] - 1 of A and C.  offsets: groups + 1 ints on the
 * device, not decreasing, within 0 .. M (values that break this are clamped).  A group may be empty:
 * its weight is not read, its gradients are zero.  Rows before offsets[0] and from offsets[groups] on are not
 * touched. */
int rocm_wmma_gemm_grouped(int type_idx, void* C, const void* A, const void* B, const int* offsets, size_t groups,
                           size_t M, size_t N, size_t K, int layout_b, const rocm_wmma_gemm_epilogue* epilogue,
                           void* stream);
int rocm_wmma_gemm_grouped_backward(int type_idx, void* dA, void* dB, void* dbias, const void* dC, const void* A,
                                    const void* B, const void* preact, const int* offsets, size_t groups, size_t M,
                                    size_t N, size_t K, int layout_b, int activation, int accumulate, void* stream);

/* How a layer's product would run (operands that start on 16 bytes assumed; groups 0: linear), or one of the
 * products of an update's steps (rocm_wmma_gemm_orthogonalize): of M x N matrices, `groups` of them, type_idx
 * one of those whose A has O's type; K, layout_b and activation are not looked at. */
#define ROCM_WMMA_GEMM_PRODUCT_FORWARD 0
#define ROCM_WMMA_GEMM_PRODUCT_GRADIENT_A 1
#define ROCM_WMMA_GEMM_PRODUCT_GRADIENT_B 2
#define ROCM_WMMA_GEMM_PRODUCT_STEPS_S 3    /* S = X X^T */
#define ROCM_WMMA_GEMM_PRODUCT_STEPS_Q 4    /* Q = b S + c S^2 */
#define ROCM_WMMA_GEMM_PRODUCT_STEPS_X 5    /* X = a X + Q X, but for the last step's */
#define ROCM_WMMA_GEMM_PRODUCT_STEPS_LAST 6 /* the last step's */
typedef struct rocm_wmma_gemm_product_plan
{
    int form; /* kernel: 0, 1 general (any alignment), 2-5 persistent tiles, 6 the same with C of any
                 alignment, 7-13 few rows against a weight, 14 all steps of a matrix in one workgroup */
    int block_m, block_n; /* its tile */
    int cut_tail; /* 1: tiles of the last round are cut along K and added up by a second kernel */
    int k_slices; /* few rows: workgroups that share a tile */
    int once; /* 1: the weight is loaded with the non-temporal hint */
    int copies; /* bit 0: A, bit 1: B is first copied to rows that start on 16 bytes */
} rocm_wmma_gemm_product_plan;
int rocm_wmma_gemm_product_select(int product, int type_idx, size_t M, size_t N, size_t K, size_t groups, int layout_b,
                                  int activation, rocm_wmma_gemm_product_plan* plan);

/* Newton-Schulz steps that bring an update near the closest matrix with orthonormal rows or
 * columns (all singular values near 1): X = G / (|G|_F + epsilon), then `steps` times
 * X = a X + (b S + c S^2) X with S = X X^T, coefficients = {a, b, c}; O = X.  G and O: batch_count
 * row-major M x N matrices; G of type F16, BF16 or F32, O of type F16 or BF16.  M and N up to 2^20.
 * Matrices of up to 64 x 256 (either way up) are worked on in fp32.  The products of larger ones take f16
 * operands (X, S and b S + c S^2 rounded to 11 bits; a X and the diagonal of b S + c S^2 stay in fp32), which leaves
 * up to 8e-4 of an update's norm after five steps with the usual coefficients (3.4445, -4.7750, 2.0315), and
 * needs singular values s of the iterates with |b| s^2 + |c| s^4 and 2 s sqrt(min(M, N)) below 65504: with other
 * coefficients that let them grow past that, O is infinite or no number.
 * Works in the library's scratch buffer (8 bytes an element and 4 min(M, N)^2 per matrix, 16 GiB at most: a
 * batch that needs more goes in parts, a single matrix that does returns ROCM_WMMA_GEMM_ERR_SCRATCH). */
#define ROCM_WMMA_GEMM_ELEMENT_F16 0
#define ROCM_WMMA_GEMM_ELEMENT_BF16 1
#define ROCM_WMMA_GEMM_ELEMENT_F32 2
int rocm_wmma_gemm_orthogonalize(int given_type, int out_type, void* O, const void* G, size_t M, size_t N,
                                 size_t batch_count, int steps, const float* coefficients, float epsilon, void* stream);

/* ---------------------------------------------------------------------------------------
 * From a router to the experts and back: additions with no counterpart in the reference.
 *
 * M tokens choose k of E experts each.  route picks them from the router's logits (M x E), dispatch sorts the
 * tokens' rows by expert and writes the row offsets that rocm_wmma_gemm_grouped reads, combine sums the experts' rows
 * by token.  All matrices are row-major and packed and may start on any element; element types are
 * ROCM_WMMA_GEMM_ELEMENT_* as above.  E up to 512, k up to 32, M k up to 2^31 - 256.  A size of 0 is no error.  The
 * calls enqueue on *stream and return; none but dispatch (past 4096 choices) uses the library's scratch buffer.
 * --------------------------------------------------------------------------------------- */
#define ROCM_WMMA_GEMM_SCORE_SOFTMAX 0 /* e^x over the sum of all e^x */
#define ROCM_WMMA_GEMM_SCORE_SIGMOID 1 /* 1 / (1 + e^-x) */

#define ROCM_WMMA_GEMM_MAX_EXPERTS 512
#define ROCM_WMMA_GEMM_MAX_CHOICES 32
#define ROCM_WMMA_GEMM_MAX_EXPERT_GROUPS 16

typedef struct rocm_wmma_gemm_routing
{
    int                  score; /* ROCM_WMMA_GEMM_SCORE_* */
    const float*         bias; /* E values added to the scores for the choice alone, or NULL */
    const unsigned char* mask; /* M values, 0: the token goes nowhere; or NULL */
    int                  groups; /* the experts form this many groups of neighbours (1: no groups); divides E */
    int                  kept_groups; /* a token chooses from this many of them */
    int                  group_best; /* 1 or 2: the sum of so many of a group's best biased scores decides which are kept */
    int                  renormalize; /* 1: a token's weights are divided by the sum of their scores */
    float                scale; /* and multiplied by this */
} rocm_wmma_gemm_routing;

/* chosen (M x k): the experts of the largest biased score, of the largest logit where there is no bias, the best
 * first; of equal ones the lower expert.  weights (M x k): their scores, without the bias.  What decides is worked out in
 * fp64; biased scores that differ by less than 2^-43 of themselves may count as equal.  A masked token's experts are -1, its
 * weights 0.  A logit of -infinity has the score 0; a token whose chosen scores are all 0 has weights 0.  A logit that is no
 * number counts as the lowest value: the others are chosen as without it, and its token's weights may be no numbers.  (The
 * softmax of a token with a logit of +infinity has no value: with a bias or groups its choice means nothing.) */
int rocm_wmma_gemm_route(int logits_type, int* chosen, float* weights, const void* logits,
                         const rocm_wmma_gemm_routing* routing, size_t M, size_t E, size_t k, void* stream);

/* dlogits (M x E, the logits' type) from dweights (M x k): the gradient of the weights; the choice has none, nor has
 * the bias.  chosen: route's; an expert outside 0 .. E - 1 has no gradient. */
int rocm_wmma_gemm_route_backward(int logits_type, void* dlogits, const float* dweights, const int* chosen,
                                  const void* logits, size_t M, size_t E, size_t k, int score, int renormalize, float scale,
                                  void* stream);

/* offsets (E + 1): where every expert's rows start when the choices are sorted by expert, within an expert in
 * their order; places (M x k): the row of every choice, -1 for one outside 0 .. E - 1 (it has no row); rows (M k x N of
 * rows_type): row places[t k + j] is row t of X (M x N).  rows may be NULL: then X is not read.  Rows from
 * offsets[E] on are left as they were.  The gradient of X is combine without weights of rows'. */
int rocm_wmma_gemm_dispatch(int rows_type, void* rows, int* offsets, int* places, const void* X, const int* chosen,
                            size_t E, size_t M, size_t N, size_t k, void* stream);

/* C (M x N): the sum over a token's choices of weights[t k + j] (NULL: 1) times row places[t k + j] of rows (M k x
 * N), plus residual (M x N of C's type, or NULL; may be C itself).  A place outside 0 .. M k - 1 adds nothing.  Summed
 * in fp32 in the order of the choices, rounded once.  out_type: rows_type or F32. */
int rocm_wmma_gemm_combine(int rows_type, int out_type, void* C, const void* rows, const int* places, const float* weights,
                           const void* residual, size_t M, size_t N, size_t k, void* stream);

/* drows (M k x N of rows_type, or NULL): weight times dC's row, for the rows that places name (each once); the others
 * are left as they were.  dweights (M x k, or NULL): the product of dC's row with the choice's, 0 for a
 * place outside 0 .. M k - 1.  dC: M x N of out_type; rows may be NULL where dweights is. */
int rocm_wmma_gemm_combine_backward(int rows_type, int out_type, void* drows, float* dweights, const void* dC,
                                    const void* rows, const int* places, const float* weights, size_t M, size_t N, size_t k,
                                    void* stream);

/* ---------------------------------------------------------------------------------------
 * A projection onto a vocabulary with its loss: additions with no counterpart in the reference.
 *
 * Logits z = A B of M states (A: M x K, row-major) over N entries (B: K x N, layout_b as for a linear layer: 1, weights stored
 * N x K, or 0), which are never kept: they are worked out piece by piece, and again for the gradient.  A and B have the
 * element F16 or BF16, loss, lse and dloss are fp32 and have one value a row.  lse: log sum_v e^(z_v / temperature)
 * (temperature 1 for cross entropy), which the backward pass reads.  Softmax, sums and losses are worked out in fp32.  M up to
 * 2^20, N and K up to 2^31 - 256; a size of 0 is no error.  Rows of A that are left out must hold numbers all the same (they are
 * multiplied by 0).  The calls enqueue on *stream and return; they work in the library's scratch buffer and return
 * ROCM_WMMA_GEMM_ERR_SCRATCH where it cannot be had (on a capturing stream: make one eager call first; operands whose rows do
 * not start on 16 bytes are copied, and the whole has to fit 16 GiB).
 * --------------------------------------------------------------------------------------- */

/* loss_t = lse_t - z_t,target; 0 for a row whose target lies outside 0 .. N - 1 (it is left out).  targets: M values of 32 bits, or
 * of 64 with wide_targets 1. */
int rocm_wmma_gemm_linear_cross_entropy(int element, float* loss, float* lse, const void* A, const void* B,
                                        const void* targets, int wide_targets, size_t M, size_t N, size_t K, int layout_b,
                                        void* stream);

/* dz = dloss (softmax(z) - [v = target]), 0 in rows that are left out; dA = dz B^T (M x K), dB = A^T dz in B's layout; a NULL result is
 * not computed.  accumulate 1: dB is added to.  type_idx: the types of dA and dB, and of A and B.  dz is rounded to A's
 * type before it is multiplied, in units of 2^-14 of the largest |dloss| of the rows that are not left out. */
int rocm_wmma_gemm_linear_cross_entropy_backward(int type_idx, void* dA, void* dB, const float* dloss, const float* lse,
                                                 const void* A, const void* B, const void* targets, int wide_targets, size_t M,
                                                 size_t N, size_t K, int layout_b, int accumulate, void* stream);

/* Most entries of a row's list. */
#define ROCM_WMMA_GEMM_MAX_ENTRIES 256

/* Distillation from the k entries of every row that a teacher lists, with its logits (teacher: M x k, fp32): q = softmax(teacher /
 * temperature) over the row's list, p = softmax(z / temperature) over all N, loss = temperature^2 sum_j q_j (log q_j - log p_entry j).
 * entries: M x k of 32 or (wide_entries 1) 64 bits; one outside 0 .. N - 1 is not in the list; a row with an empty list is left
 * out: its loss is 0.  picked (M x k, fp32) receives the logits z of the entries, which the backward pass reads. */
int rocm_wmma_gemm_linear_distillation(int element, float* loss, float* lse, float* picked, const void* A, const void* B,
                                       const void* entries, int wide_entries, const float* teacher, size_t M, size_t N,
                                       size_t K, size_t k, float temperature, int layout_b, void* stream);

/* dz = dloss temperature (p - q), with the shares of an entry that is listed more than once added up; the rest as above. */
int rocm_wmma_gemm_linear_distillation_backward(int type_idx, void* dA, void* dB, const float* dloss, const float* lse,
                                                const float* picked, const void* A, const void* B, const void* entries,
                                                int wide_entries, const float* teacher, size_t M, size_t N, size_t K, size_t k,
                                                float temperature, int layout_b, int accumulate, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ROCM_WMMA_GEMM_C_H */
