// The kernels from a router's logits to rows sorted by expert and back: the choice of the experts with its
// gradient, the sort of the choices with the copy of their rows, the weighted sum of the experts' rows with its
// gradients.  All are bound by memory, or by the latency of a launch where there are few tokens.
#ifndef ROCM_WMMA_GEMM_ROUTING_HPP
#define ROCM_WMMA_GEMM_ROUTING_HPP

#include "product_common.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

constexpr int route_lanes   = 16; // of a token
constexpr int most_choices  = 32; // experts of a token
constexpr int most_parts    = 16; // groups of experts
constexpr int most_dispatch = max_groups; // experts

// ------------------------------------------------------------------ sixteen lanes together

// The value of the lane that `control` names within the row of 16 lanes.
template<int CONTROL, class T>
__device__ __forceinline__ T from_row(T v)
{
    if constexpr(sizeof(T) == 8)
    {
        const unsigned long long b  = __builtin_bit_cast(unsigned long long, v);
        const unsigned int       lo = __builtin_amdgcn_update_dpp(0, (int)b, CONTROL, 0xf, 0xf, false);
        const unsigned int       hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CONTROL, 0xf, 0xf, false);
        return __builtin_bit_cast(T, (unsigned long long)hi << 32 | lo);
    }
    else
    {
        const int b = __builtin_bit_cast(int, v);
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, b, CONTROL, 0xf, 0xf, false));
    }
}

// Joins the values of 1, 2, 4, 8 or 16 neighbouring lanes, in every one of them: neighbours, pairs, then the mirror
// images in 8 and in 16 lanes (whose values are equal within 4 and 8 by then).
template<class T, class Join>
__device__ __forceinline__ T join_row(T v, int lanes, Join join)
{
    v = lanes > 1 ? join(v, from_row<0xb1>(v)) : v; // quad_perm 1 0 3 2
    v = lanes > 2 ? join(v, from_row<0x4e>(v)) : v; // quad_perm 2 3 0 1
    v = lanes > 4 ? join(v, from_row<0x141>(v)) : v; // row_half_mirror
    v = lanes > 8 ? join(v, from_row<0x140>(v)) : v; // row_mirror
    return v;
}

template<class T>
__device__ __forceinline__ T sum_of_row(T v)
{
    return join_row(v, route_lanes, [](T a, T b) { return a + b; });
}

// The value of lane `from` of the token's sixteen.
template<class T>
__device__ __forceinline__ T of_lane(T v, int from)
{
    const int lane = (int)(threadIdx.x & 48) | from;
    if constexpr(sizeof(T) == 8)
    {
        const unsigned long long b  = __builtin_bit_cast(unsigned long long, v);
        const unsigned int       lo = __shfl((int)b, lane), hi = __shfl((int)(b >> 32), lane);
        return __builtin_bit_cast(T, (unsigned long long)hi << 32 | lo);
    }
    else
    {
        return __builtin_bit_cast(T, __shfl(__builtin_bit_cast(int, v), lane));
    }
}

// ------------------------------------------------------------------ the choice

struct route_args
{
    int*         chosen; // tokens x k
    float*       weights; // tokens x k
    const void*  logits; // tokens x experts
    const float* bias; // nullptr, or one an expert: added for the choice alone
    const unsigned char* mask; // nullptr, or one a token: 0 goes nowhere
    long long    tokens;
    int          experts, k;
    int          groups, size; // of experts: experts = groups * size
    int          kept, best; // groups that a token may choose from; how many of its best make a group's score
    int          spread, chunk; // lanes of a group, and experts of a lane (spread * chunk >= size, spread * groups <= 16)
    int          renormalize;
    float        scale;
};

// Consecutive elements of a row, `count` of COUNT, as fp32.  WHOLE: all of them, on an address that pieces of them start
// on; else the others repeat the last one's address (a load is always in the row).
template<class T, int COUNT, bool WHOLE>
__device__ __forceinline__ void load_run(const T* from, int count, int last, float (&to)[COUNT])
{
    if constexpr(WHOLE)
    {
        constexpr int PIECE = COUNT * (int)sizeof(T) < 16 ? COUNT : 16 / (int)sizeof(T);
        typedef T     piece_t __attribute__((ext_vector_type(PIECE)));
#pragma unroll
        for(int i = 0; i < COUNT; i += PIECE)
        {
            const piece_t v = *reinterpret_cast<const piece_t*>(from + i);
#pragma unroll
            for(int e = 0; e < PIECE; ++e)
            {
                to[i + e] = (float)v[e];
            }
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < COUNT; ++i)
        {
            to[i] = (float)from[i < count ? i : last];
        }
    }
}

// e^t in fp64: t = n ln 2 + r with |r| <= ln 2 / 2, e^r by its series (the first term left out is 4e-18 of it), times 2^n.
// Half the instructions of the library's, which also serves what is far from here.
__device__ __forceinline__ double power_of_e(double t)
{
    constexpr double over_ln2 = 1.4426950408889634074, ln2 = 0.693147180559945309417, ln2_rest = 2.3190468138462996e-17;
    const double     n = __builtin_rint(t * over_ln2);
    const double     r = __builtin_fma(-n, ln2_rest, __builtin_fma(-n, ln2, t));
    double           p = 1.0 / 6227020800.0; // 1 / 13!
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const double e = __builtin_ldexp(p, (int)n);
    return t < -745.0 ? 0.0 : e; // (also of -infinity; no number stays none)
}

// 1 / d for d of ordinary size: the hardware's 2^-24 or better, doubled in digits twice.
__device__ __forceinline__ double one_over(double d)
{
    double y = __builtin_amdgcn_rcp(d);
    y        = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}

// 1 / (1 + e^-x); 0 below 1e-304, where 1 over it leaves fp64's ordinary numbers.
__device__ __forceinline__ double sigmoid(double x)
{
    const double e = power_of_e(-x);
    return x < -700.0 ? 0.0 : one_over(1.0 + e);
}

// A choice as one number that v_max_f64 orders: the value, whose last 9 bits tell the expert, so that of equal
// values the lower expert is more.  (Values that differ by less than 2^-43 of themselves may count as equal: 9 bits of 52; logits, which
// have 24 bits, are told apart.)  No number counts as the lowest value.
constexpr int choice_bits = 511;
__device__ __forceinline__ double choice_key(double value, int expert)
{
    constexpr double most = 1.7976931348623157e308;
    // (of a number and none, the maximum is the number; 0 is added for the sign of -0)
    value = __builtin_fmin(__builtin_fmax(value, -most), most) + 0.0;
    const unsigned long long b  = __builtin_bit_cast(unsigned long long, value);
    const int                hi = (int)(b >> 32);
    // below 0 the larger bits are the smaller number
    const unsigned int lo = ((unsigned int)b & ~(unsigned int)choice_bits)
                            | (unsigned int)((choice_bits - expert) ^ (hi >> 31 & choice_bits));
    return __builtin_bit_cast(double, (unsigned long long)(unsigned int)hi << 32 | lo);
}
__device__ __forceinline__ int expert_of_key(double key)
{
    const unsigned long long b = __builtin_bit_cast(unsigned long long, key);
    return choice_bits - (((int)b & choice_bits) ^ ((int)(b >> 32) >> 31 & choice_bits));
}

// Falling order by Batcher's merge of odd and even places: 63 exchanges for 16 keys.
template<int COUNT>
__device__ __forceinline__ void sort_falling(double (&key)[COUNT])
{
#pragma unroll
    for(int p = 1; p < COUNT; p *= 2)
    {
#pragma unroll
        for(int q = p; q >= 1; q /= 2)
        {
#pragma unroll
            for(int j = q % p; j + q < COUNT; j += 2 * q)
            {
#pragma unroll
                for(int i = 0; i < q; ++i)
                {
                    if(i + j + q < COUNT && (i + j) / (2 * p) == (i + j + q) / (2 * p))
                    {
                        const double a = key[i + j], b = key[i + j + q];
                        key[i + j]     = __builtin_fmax(a, b);
                        key[i + j + q] = __builtin_fmin(a, b);
                    }
                }
            }
        }
    }
}

// Sixteen lanes a token, CHUNK experts a lane (args.chunk of them used; WHOLE: all, in every lane), at most MOST choices.
//
// Mathematics: scores s = softmax(x) or 1 / (1 + e^-x); the k experts of the largest s + bias (of the largest x where there is
// no bias: the same order) among the experts of the `kept` groups whose `best` largest s + bias sum to most; weights scale s,
// or scale s over the sum of the chosen s.  Everything that decides is held in fp64, so that the choice is the definition's
// and not that of fp32's roundings; fp64 runs at the fp32 rate here.
//
// Bound by the instructions: 8191 tokens over 256 experts in groups are 2 waves for every SIMD, whose 16 scores a lane, their sort and
// eight rounds of a maximum over 16 lanes (four DPP steps) are some 1100 instructions: 7.9 us a call (8.4 MB, 1.1 TB/s).
template<class InT, int CHUNK, bool SIGMOID, bool WHOLE, int MOST>
__device__ __forceinline__ void route_token(const route_args& args, long long token, int lane)
{
    const InT* const x     = static_cast<const InT*>(args.logits) + token * args.experts;
    const int        group = lane / args.spread, within = lane % args.spread * args.chunk;
    int              first = group * args.size + within; // this lane's experts: first .. first + count - 1
    int              count = args.size - within;
    count                  = count < args.chunk ? count : args.chunk;
    count                  = group < args.groups && count > 0 ? count : 0;
    first                  = count > 0 ? first : 0;
    const int last         = count > 0 ? count - 1 : 0;
    const double least = -__builtin_inf();
    float        logit[CHUNK];
    load_run<InT, CHUNK, WHOLE>(x + first, count, last, logit);
    auto is = [&](int i) { return WHOLE || i < count; };
    const bool by_score = args.bias != nullptr || args.groups > 1;
    // softmax: its largest logit and sum, where the scores need them.  A logit that is no number adds nothing to the sum, so that
    // the others are chosen by their scores; the weights' sum is none with it.
    double top = 0.0, over_total = 1.0, over_weights = 1.0;
    if constexpr(!SIGMOID)
    {
        float most = -__builtin_inff();
#pragma unroll
        for(int i = 0; i < CHUNK; ++i)
        {
            most = is(i) ? __builtin_fmaxf(most, logit[i]) : most;
        }
        most = join_row(most, route_lanes, [](float a, float b) { return __builtin_fmaxf(a, b); });
        top  = most > -__builtin_inff() ? (double)most : 0.0; // (no finite logit: all scores are 0)
        if(by_score || !args.renormalize)
        {
            double sum = 0.0;
            int    bad = 0;
#pragma unroll
            for(int i = 0; i < CHUNK; ++i)
            {
                // (of a number and none, the maximum is the number)
                sum += is(i) ? power_of_e(__builtin_fmax((double)logit[i] - top, least)) : 0.0;
                bad |= is(i) && logit[i] != logit[i] ? 1 : 0;
            }
            sum          = sum_of_row(sum);
            bad          = join_row(bad, route_lanes, [](int a, int b) { return a | b; });
            over_total   = sum == 0.0 ? 1.0 : 1.0 / sum;
            over_weights = bad ? __builtin_nan("") : over_total;
        }
    }
    auto score = [&](float l, double over) { return SIGMOID ? sigmoid((double)l) : power_of_e((double)l - top) * over; };
    double key[CHUNK];
    double high = least, second = least; // the lane's two best values
    if(by_score)
    {
        float bias[CHUNK];
        if(args.bias != nullptr)
        {
            load_run<float, CHUNK, WHOLE>(args.bias + first, count, last, bias);
        }
        else
        {
#pragma unroll
            for(int i = 0; i < CHUNK; ++i)
            {
                bias[i] = 0.0f;
            }
        }
#pragma unroll
        for(int i = 0; i < CHUNK; ++i)
        {
            const double s = score(logit[i], over_total) + (double)bias[i];
            const double v = is(i) ? __builtin_fmax(s, least) : least; // (no number: the lowest)
            second         = __builtin_fmax(second, __builtin_fmin(high, v));
            high           = __builtin_fmax(high, v);
            key[i]         = is(i) ? choice_key(args.bias != nullptr ? s : (double)logit[i], first + i) : least;
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < CHUNK; ++i)
        {
            key[i] = is(i) ? choice_key((double)logit[i], first + i) : least;
        }
    }
    if(args.groups > 1)
    {
        // the group's two best, over its lanes
        const int spread = args.spread;
        auto      meet   = [&](double h, double s) {
            second = __builtin_fmax(__builtin_fmin(high, h), __builtin_fmax(second, s));
            high   = __builtin_fmax(high, h);
        };
        if(spread > 1)
        {
            meet(from_row<0xb1>(high), from_row<0xb1>(second));
        }
        if(spread > 2)
        {
            meet(from_row<0x4e>(high), from_row<0x4e>(second));
        }
        if(spread > 4)
        {
            meet(from_row<0x141>(high), from_row<0x141>(second));
        }
        // (infinite biases: of a sum that is none, the lowest, or the group would be one more than `kept`)
        const double of_group = __builtin_fmax(args.best > 1 && args.size > 1 ? high + second : high, least);
        int          better   = 0;
        for(int g = 0; g < args.groups; ++g)
        {
            const double other = of_lane(of_group, g * spread);
            better += other > of_group || (other == of_group && g < group);
        }
        if(better >= args.kept)
        {
#pragma unroll
            for(int i = 0; i < CHUNK; ++i)
            {
                key[i] = least;
            }
        }
    }
    // Every lane's keys in falling order; k times the largest of the lanes' first ones, whose lane moves its others up.  (No two
    // keys that an expert has are equal.)
    constexpr int DEPTH = CHUNK < MOST ? CHUNK : MOST; // keys of a lane that can be chosen
    sort_falling(key);
    int  mine[MOST > route_lanes ? 2 : 1] = {};
    auto choose_one = [&](int j, int depth) {
        const double most = join_row(key[0], route_lanes, [](double a, double b) { return __builtin_fmax(a, b); });
        const bool   own  = key[0] == most;
#pragma unroll
        for(int i = 0; i + 1 < DEPTH; ++i)
        {
            if(i < depth)
            {
                key[i] = own ? key[i + 1] : key[i];
            }
        }
        key[DEPTH - 1] = own && depth >= DEPTH - 1 ? least : key[DEPTH - 1];
        const int e = expert_of_key(most);
        mine[0]     = lane == j ? e : mine[0];
        if constexpr(MOST > route_lanes)
        {
            mine[1] = lane + route_lanes == j ? e : mine[1];
        }
    };
    if constexpr(MOST <= 8)
    {
#pragma unroll
        for(int j = 0; j < MOST; ++j)
        {
            if(j < args.k)
            {
                choose_one(j, MOST - 1 - j < DEPTH - 1 ? MOST - 1 - j : DEPTH - 1); // (as many as may still be chosen)
            }
        }
    }
    else
    {
        for(int j = 0; j < args.k; ++j)
        {
            choose_one(j, DEPTH - 1);
        }
    }
    // lane j: the j-th and the (16 + j)-th choice
    const bool real = args.mask == nullptr || args.mask[token] != 0;
    double     s[MOST > route_lanes ? 2 : 1], total = 0.0;
#pragma unroll
    for(int h = 0; h < (MOST > route_lanes ? 2 : 1); ++h)
    {
        s[h] = lane + h * route_lanes < args.k ? score((float)x[mine[h]], over_weights) : 0.0;
        total += s[h];
    }
    double factor = args.scale;
    if(args.renormalize)
    {
        total  = sum_of_row(total);
        factor = total == 0.0 ? 0.0 : factor / total;
    }
#pragma unroll
    for(int h = 0; h < (MOST > route_lanes ? 2 : 1); ++h)
    {
        const int j = lane + h * route_lanes;
        if(j < args.k)
        {
            args.chosen[token * args.k + j]  = real ? mine[h] : -1;
            args.weights[token * args.k + j] = real ? (float)(factor * s[h]) : 0.0f;
        }
    }
}

// (all lanes of a token leave the loop together)
template<class InT, int CHUNK, bool SIGMOID, bool WHOLE, int MOST>
__global__ void __launch_bounds__(256) route(const route_args args)
{
    constexpr int each = 256 / route_lanes; // tokens of a workgroup
    for(long long token = (long long)blockIdx.x * each + threadIdx.x / route_lanes; token < args.tokens;
        token += (long long)gridDim.x * each)
    {
        route_token<InT, CHUNK, SIGMOID, WHOLE, MOST>(args, token, threadIdx.x % route_lanes);
    }
}

struct route_back_args
{
    void*        dlogits; // tokens x experts, of the logits' type
    const float* dweights; // tokens x k
    const int*   chosen; // tokens x k
    const void*  logits;
    long long    tokens;
    int          experts, k, renormalize, chunk; // experts of a lane
    float        scale;
};

// What a lane's two choices get by sigmoid scores (see route_back_token); a choice that is none has a logit of -infinity and a
// gradient of 0.
__device__ __forceinline__ void sigmoid_gradients(const route_back_args& args, const float (&logit)[2], const float (&dw)[2],
                                                  float (&own)[2])
{
    double s[2], rest[2], ds[2]; // 1 / (1 + e^-x) and 1 / (1 + e^x), each with all its digits; 0 as in sigmoid()
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        const double x = (double)logit[h], e = power_of_e(-__builtin_fabs(x)), near_one = one_over(1.0 + e), small = e * near_one;
        s[h]    = x < -700.0 ? 0.0 : x < 0.0 ? small : near_one;
        rest[h] = x < 0.0 ? near_one : small;
        ds[h]   = (double)args.scale * (double)dw[h];
    }
    double dot = 0.0;
    if(args.renormalize)
    {
        const double sum = sum_of_row(s[0] + s[1]), over = sum == 0.0 ? 0.0 : 1.0 / sum;
        s[0] *= over;
        s[1] *= over;
        dot = sum_of_row(s[0] * ds[0] + s[1] * ds[1]);
    }
    own[0] = (float)(s[0] * (ds[0] - dot) * rest[0]);
    own[1] = (float)(s[1] * (ds[1] - dot) * rest[1]);
}

// The gradient of the weights by the logits; the choice itself has none.  With ds_j = scale (dw_j - D) / sum, D = sum_i dw_i
// w_i / scale, (renormalised; else scale dw_j): sigmoid dx_j = ds_j s_j (1 - s_j) for the chosen, 0 for the others; softmax
// dx_e = s_e (ds_e - sum_j s_j ds_j), where the sum is 0 if the weights are renormalised, so that the logits
// that were not chosen are not even read.  Softmax's largest score of the chosen is 1 before it is divided by anything, so
// fp32 holds all of it.  A sigmoid's scores may all be far below fp32's least number, and their shares of the sum are ordinary
// numbers all the same: they are worked out in fp64, as for the weights, and nothing but the result is rounded to fp32.
// Sixteen lanes a token, CHUNK experts a lane; a choice outside the experts has no gradient, one that is listed twice has both.
// Bound by the latency of a token's chain (its choices, their logits, the joins over 16 lanes, the places in LDS): 16384 tokens of
// 128 experts in bf16, 8 choices each, take 6.4 us, 9 MB at 1.4 TB/s; 6.5 us by sigmoid (6.1 with
// its scores in fp32, which gave 0 and infinities for logits of -80 and below).
template<class InT, int CHUNK, bool SIGMOID, bool WHOLE>
__device__ __forceinline__ void route_back_token(const route_back_args& args, long long token, int lane, float* row)
{
    const InT* const x  = static_cast<const InT*>(args.logits) + token * args.experts;
    InT* const       dx = static_cast<InT*>(args.dlogits) + token * args.experts;
    int              e[2];
    float            dw[2], logit[2];
    float            most = -__builtin_inff();
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        const int j = lane + h * route_lanes;
        e[h]        = j < args.k ? args.chosen[token * args.k + j] : -1;
        e[h]        = e[h] >= 0 && e[h] < args.experts ? e[h] : -1;
        dw[h]       = e[h] >= 0 ? args.dweights[token * args.k + j] : 0.0f;
        logit[h]    = e[h] >= 0 ? (float)x[e[h]] : -__builtin_inff();
        most        = __builtin_fmaxf(most, logit[h]);
    }
    const bool none  = sum_of_row((e[0] >= 0 ? 1 : 0) + (e[1] >= 0 ? 1 : 0)) == 0; // (a token that went nowhere)
    const bool dense = !SIGMOID && !args.renormalize && !none;
    const int  first = lane * args.chunk; // this lane's experts
    int        count = args.experts - first;
    count            = count < args.chunk ? (count > 0 ? count : 0) : args.chunk;
    float top = 0.0f, total = 1.0f;
    float p[CHUNK]; // dense: the scores of the lane's experts
    if constexpr(!SIGMOID)
    {
        if(dense)
        {
            load_run<InT, CHUNK, WHOLE>(x + (count > 0 ? first : 0), count, count > 0 ? count - 1 : 0, p);
#pragma unroll
            for(int i = 0; i < CHUNK; ++i)
            {
                most = WHOLE || i < count ? __builtin_fmaxf(most, p[i]) : most;
            }
        }
        top = join_row(most, route_lanes, [](float a, float b) { return __builtin_fmaxf(a, b); });
        top = top > -__builtin_inff() ? top : 0.0f;
        if(dense)
        {
            float sum = 0.0f;
#pragma unroll
            for(int i = 0; i < CHUNK; ++i)
            {
                p[i] = WHOLE || i < count ? expf(p[i] - top) : 0.0f;
                sum += p[i];
            }
            sum   = sum_of_row(sum);
            total = sum == 0.0f ? 1.0f : sum;
        }
    }
    // what every chosen logit gets, and what all get
    float own[2], all = 0.0f;
    if constexpr(SIGMOID)
    {
        sigmoid_gradients(args, logit, dw, own);
    }
    else
    {
        float s[2], ds[2];
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            s[h]  = e[h] < 0 ? 0.0f : expf(logit[h] - top) / total;
            ds[h] = args.scale * dw[h];
        }
        if(args.renormalize)
        {
            const float sum  = sum_of_row(s[0] + s[1]);
            const float rest = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float dot  = sum_of_row(ds[0] * s[0] * rest + ds[1] * s[1] * rest);
            ds[0]            = (ds[0] - dot) * rest;
            ds[1]            = (ds[1] - dot) * rest;
        }
        own[0] = s[0] * ds[0];
        own[1] = s[1] * ds[1];
        all    = dense ? sum_of_row(s[0] * ds[0] + s[1] * ds[1]) : 0.0f;
    }
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        own[h] = e[h] < 0 ? 0.0f : own[h];
    }
    // The choices' parts go to their experts' places in LDS, one after the other (of equal ones all count, in their order; the
    // sixteen lanes are of one wave, which LDS serves in order).
    volatile float* const places = row;
#pragma unroll
    for(int i = 0; i < CHUNK; ++i)
    {
        if(i < count)
        {
            places[first + i] = 0.0f;
        }
    }
    bool twice = false;
    for(int j = 0; j < args.k; ++j)
    {
        const int at = of_lane(j < route_lanes ? e[0] : e[1], j % route_lanes);
        twice        = twice || (at >= 0 && ((e[0] == at && lane != j) || (e[1] == at && lane + route_lanes != j)));
    }
    if(__ballot(twice) == 0)
    {
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            if(e[h] >= 0)
            {
                places[e[h]] = own[h];
            }
        }
    }
    else
    {
        for(int j = 0; j < args.k; ++j)
        {
            const int h = j < route_lanes ? 0 : 1;
            if(lane == j % route_lanes && e[h] >= 0)
            {
                places[e[h]] = places[e[h]] + own[h];
            }
        }
    }
    float d[CHUNK];
#pragma unroll
    for(int i = 0; i < CHUNK; ++i)
    {
        d[i] = i < count ? places[first + i] : 0.0f;
        d[i] = dense ? d[i] - all * (p[i] / total) : d[i];
    }
    if constexpr(WHOLE)
    {
        constexpr int PIECE = CHUNK * (int)sizeof(InT) < 16 ? CHUNK : 16 / (int)sizeof(InT);
        typedef InT   piece_t __attribute__((ext_vector_type(PIECE)));
#pragma unroll
        for(int i = 0; i < CHUNK; i += PIECE)
        {
            piece_t o;
#pragma unroll
            for(int v = 0; v < PIECE; ++v)
            {
                o[v] = to_out<InT>(d[i + v]);
            }
            *reinterpret_cast<piece_t*>(dx + first + i) = o;
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < CHUNK; ++i)
        {
            if(i < count)
            {
                dx[first + i] = to_out<InT>(d[i]);
            }
        }
    }
}

template<class InT, int CHUNK, bool SIGMOID, bool WHOLE>
__global__ void __launch_bounds__(256) route_backward(const route_back_args args)
{
    constexpr int    each = 256 / route_lanes;
    __shared__ float rows[each][route_lanes * CHUNK];
    for(long long token = (long long)blockIdx.x * each + threadIdx.x / route_lanes; token < args.tokens;
        token += (long long)gridDim.x * each)
    {
        route_back_token<InT, CHUNK, SIGMOID, WHOLE>(args, token, threadIdx.x % route_lanes, rows[threadIdx.x / route_lanes]);
    }
}

// ------------------------------------------------------------------ the sort

// A stable counting sort of the choices by expert, 1024 threads a block, 64 choices a wave at a time: the lanes
// with one expert find each other by nine ballots, one for each bit of its number, and their leader counts them in its
// wave's row of the histogram.  Nothing depends on the order in which waves or blocks run.
constexpr int sort_waves = 16, sort_round = sort_waves * 64, sort_rounds = 4, sort_block = sort_round * sort_rounds; // choices

// Rows of this many bytes are written past the caches: they are not in the 256 MB memory-side cache when they are read next.
// With a reader behind them, 256 MB of rows: 124.4 us against 125.5, 512 MB 253 against 266; but 128 MB 69 against 59, and
// the gradients of 128 MB, 256 MB and 512 MB 77 against 79, 182 against 189 and 353 against 360.
constexpr long long streamed_bytes = 256ll << 20;

// (a template argument: the compiler joins the two stores of a branch, without the hint)
template<bool STREAMED, class Piece>
__device__ __forceinline__ void put(Piece* to, const Piece& v)
{
    if constexpr(STREAMED)
    {
        __builtin_nontemporal_store(v.v, &to->v);
    }
    else
    {
        to->v = v.v;
    }
}

// 16 bytes, 2, or 8 elements, that may start on any element: accesses of vectors need no alignment here.  (Structures: the
// alignment of a plain vector type gets lost where templates take it.)
struct piece16
{
    typedef u32x4 vector __attribute__((aligned(2)));
    vector        v;
};
struct piece2
{
    unsigned short v;
};
template<class T>
struct eight
{
    typedef T vector __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    vector    v;
};
static_assert(alignof(piece16) == 2 && sizeof(piece16) == 16 && alignof(eight<float>) == 4 && sizeof(eight<_Float16>) == 16, "anywhere");

struct sort_tables
{
    int counts[sort_waves][max_groups]; // of a wave, then what lies before it in its block
    int first[max_groups + 1]; // of an expert, over the block
};

// The ranks of a block's choices within their expert and block, in rank[]; the block's counts by expert in
// tables.first[0 .. experts - 1].  Choices outside the experts have rank -1.
template<int ROUNDS>
__device__ __forceinline__ void rank_choices(const int* chosen, long long begin, long long end, int experts, sort_tables& tables,
                                             int (&expert)[ROUNDS], int (&rank)[ROUNDS])
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for(int r = 0; r < ROUNDS; ++r)
    {
        const long long at = begin + (wave * ROUNDS + r) * 64 + lane;
        expert[r]          = at < end ? chosen[at] : -1;
    }
    for(int e = lane; e < experts; e += 64)
    {
        tables.counts[wave][e] = 0; // (its own wave's: LDS serves a wave in order)
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for(int r = 0; r < ROUNDS; ++r)
    {
        const int       e  = expert[r];
        const bool      is = e >= 0 && e < experts;
        unsigned long long same = __ballot(is);
#pragma unroll
        for(int bit = 0; bit < 9; ++bit)
        {
            const bool               set = (e >> bit & 1) != 0;
            const unsigned long long b   = __ballot(set);
            same &= set ? b : ~b;
        }
        expert[r] = is ? e : -1;
        rank[r]   = -1;
        if(is)
        {
            // (every lane reads its expert's count before the leader adds: one wave, LDS in order)
            volatile int* const count  = &tables.counts[wave][e];
            const int           before = __popcll(same & ((1ull << lane) - 1ull));
            const int           sofar  = *count;
            rank[r]                    = sofar + before;
            if(before == 0)
            {
                *count = sofar + __popcll(same);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for(int e = threadIdx.x; e < experts; e += 1024)
    {
        int sum = 0;
#pragma unroll
        for(int w = 0; w < sort_waves; ++w)
        {
            const int c         = tables.counts[w][e];
            tables.counts[w][e] = sum;
            sum += c;
        }
        tables.first[e] = sum;
    }
    __syncthreads();
#pragma unroll
    for(int r = 0; r < ROUNDS; ++r)
    {
        rank[r] += expert[r] >= 0 ? tables.counts[wave][expert[r]] : 0;
    }
}

// first[0 .. experts - 1]: counts, then their exclusive sums, and the sum of all in first[experts].  One wave.
__device__ __forceinline__ void scan_experts(int* first, int experts)
{
    if(threadIdx.x < 64)
    {
        const int lane  = threadIdx.x;
        int       carry = 0;
        for(int base = 0; base < experts; base += 64)
        {
            const int e   = base + lane;
            const int own = e < experts ? first[e] : 0;
            int       sum = own;
#pragma unroll
            for(int d = 1; d < 64; d *= 2)
            {
                const int u = __shfl_up(sum, d);
                sum += lane >= d ? u : 0;
            }
            if(e < experts)
            {
                first[e] = carry + sum - own;
            }
            carry += __shfl(sum, 63);
        }
        if(lane == 0)
        {
            first[experts] = carry;
        }
    }
    __syncthreads();
}

struct dispatch_args
{
    void*       rows; // tokens * k x row_bytes
    int*        offsets; // experts + 1
    int*        places; // tokens x k
    const void* x; // tokens x row_bytes
    const int*  chosen; // tokens x k
    int*        counts; // blocks x experts: of a block, then where its first choice of an expert goes
    long long   slots; // tokens * k
    long long   tokens;
    long long   row_bytes;
    int         experts, k, blocks;
    int         copy; // 0: rows are not wanted
};

// The pieces begin .. end - 1 of a token's row to the places of its choices (place: of choice `lane`).  The last piece ends with
// the row: it may overlap the one before, whose bytes are the same.
template<class Piece, bool STREAMED>
__device__ __forceinline__ void copy_row(const dispatch_args& args, long long token, int place, long long begin, long long end)
{
    const char* const from = static_cast<const char*>(args.x) + token * args.row_bytes;
    char* const       to   = static_cast<char*>(args.rows);
    const long long   last = args.row_bytes - (long long)sizeof(Piece);
    auto start = [&](long long piece) { return piece * (long long)sizeof(Piece) < last ? piece * (long long)sizeof(Piece) : last; };
    // (four pieces of a lane on their way at a time; every lane stays in the loop, as the others read its place)
    for(; begin < end; begin += 256)
    {
        const long long at = begin + (threadIdx.x & 63);
        Piece           v[4];
#pragma unroll
        for(int u = 0; u < 4; ++u)
        {
            v[u].v = at + 64 * u < end ? reinterpret_cast<const Piece*>(from + start(at + 64 * u))->v : decltype(v[u].v){};
        }
        for(int j = 0; j < args.k; ++j)
        {
            const int p = __builtin_amdgcn_readlane(place, j);
            if(p >= 0)
            {
                char* const row = to + p * args.row_bytes;
#pragma unroll
                for(int u = 0; u < 4; ++u)
                {
                    if(at + 64 * u < end)
                    {
                        put<STREAMED>(reinterpret_cast<Piece*>(row + start(at + 64 * u)), v[u]);
                    }
                }
            }
        }
    }
}

template<class Piece>
__device__ __forceinline__ long long pieces_of_row(const dispatch_args& args)
{
    return (args.row_bytes + (long long)sizeof(Piece) - 1) / (long long)sizeof(Piece);
}

// All of it in one launch, for up to ROUNDS * 1024 choices: every workgroup sorts all of them for itself and copies its share
// of the rows, 64 pieces of a row a wave.  32 tokens of 8 choices, rows of 8 KB: 6.3 us, where two launches took 11.0.
template<int ROUNDS, class Piece>
__global__ void __launch_bounds__(1024) dispatch_few(const dispatch_args args)
{
    __shared__ sort_tables tables;
    __shared__ int         places[ROUNDS * sort_round];
    int                    expert[ROUNDS], rank[ROUNDS];
    rank_choices<ROUNDS>(args.chosen, 0, args.slots, args.experts, tables, expert, rank);
    scan_experts(tables.first, args.experts);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for(int r = 0; r < ROUNDS; ++r)
    {
        const int at = (wave * ROUNDS + r) * 64 + lane;
        places[at]   = expert[r] < 0 ? -1 : tables.first[expert[r]] + rank[r];
        if(blockIdx.x == 0 && at < args.slots)
        {
            args.places[at] = places[at];
        }
    }
    if(blockIdx.x == 0)
    {
        for(int e = threadIdx.x; e <= args.experts; e += 1024)
        {
            args.offsets[e] = tables.first[e];
        }
    }
    if(!args.copy)
    {
        return;
    }
    __syncthreads();
    const long long pieces = pieces_of_row<Piece>(args), runs = (pieces + 63) / 64, all = args.tokens * runs;
    // (neighbouring runs on different compute units)
    for(long long run = blockIdx.x + (long long)gridDim.x * wave; run < all; run += (long long)gridDim.x * sort_waves)
    {
        const long long token = run / runs, begin = (run - token * runs) * 64;
        const int       place = lane < args.k ? places[token * args.k + lane] : -1;
        copy_row<Piece, false>(args, token, place, begin, pieces < begin + 64 ? pieces : begin + 64);
    }
}

// The counts of every block, and the ranks within it in places, until it is known what lies before.
__global__ void __launch_bounds__(1024) dispatch_rank(const dispatch_args args)
{
    __shared__ sort_tables tables;
    int                    expert[sort_rounds], rank[sort_rounds];
    const long long        begin = (long long)blockIdx.x * sort_block;
    rank_choices<sort_rounds>(args.chosen, begin, args.slots, args.experts, tables, expert, rank);
    for(int e = threadIdx.x; e < args.experts; e += 1024)
    {
        args.counts[(long long)blockIdx.x * args.experts + e] = tables.first[e];
    }
#pragma unroll
    for(int r = 0; r < sort_rounds; ++r)
    {
        const long long at = begin + ((threadIdx.x >> 6) * sort_rounds + r) * 64 + (threadIdx.x & 63);
        if(at < args.slots)
        {
            args.places[at] = expert[r] < 0 ? -1 : rank[r];
        }
    }
}

// Where every block's choices of every expert begin (in counts), and the offsets.  One workgroup; for tables that are too
// large for dispatch_rows to add up.
__global__ void __launch_bounds__(1024) dispatch_scan(const dispatch_args args)
{
    __shared__ int first[max_groups + 1];
    for(int e = threadIdx.x; e < args.experts; e += 1024)
    {
        int sum = 0;
#pragma unroll 8
        for(int b = 0; b < args.blocks; ++b)
        {
            sum += args.counts[(long long)b * args.experts + e];
        }
        first[e] = sum;
    }
    __syncthreads();
    scan_experts(first, args.experts);
    for(int e = threadIdx.x; e <= args.experts; e += 1024)
    {
        args.offsets[e] = first[e];
    }
    for(int e = threadIdx.x; e < args.experts; e += 1024)
    {
        int at = first[e];
#pragma unroll 8
        for(int b = 0; b < args.blocks; ++b)
        {
            int* const here  = args.counts + (long long)b * args.experts + e;
            const int  count = *here;
            *here            = at;
            at += count;
        }
    }
}

// Adds what lies before a block's choices of an expert to their ranks, and copies the rows.  A workgroup takes `each`
// tokens in a row, whose choices lie in one block or in two neighbouring ones.  SCANNED: counts already say where the blocks' begin;
// else every workgroup adds up the (small) table.  A wave a token.  Bound by memory: 8191 tokens of 6 choices, rows of 4 KB, 235 MB: 54
// us at 4.4 TB/s behind dispatch_rank's 5.8.
template<class Piece, bool SCANNED, bool STREAMED>
__global__ void __launch_bounds__(256) dispatch_rows(const dispatch_args args, int each)
{
    __shared__ int  first[max_groups + 1], base[2][max_groups];
    const long long token0 = (long long)blockIdx.x * each;
    const int       block0 = (int)(token0 * args.k / sort_block);
    if constexpr(SCANNED)
    {
        for(int e = threadIdx.x; e < args.experts; e += 256)
        {
            base[0][e] = args.counts[(long long)block0 * args.experts + e];
            base[1][e] = block0 + 1 < args.blocks ? args.counts[(long long)(block0 + 1) * args.experts + e] : 0;
        }
    }
    else
    {
        for(int e = threadIdx.x; e < args.experts; e += 256)
        {
            int all = 0, before = 0, own = 0;
#pragma unroll 8
            for(int b = 0; b < args.blocks; ++b)
            {
                const int count = args.counts[b * args.experts + e];
                all += count;
                before += b < block0 ? count : 0;
                own += b == block0 ? count : 0;
            }
            first[e]   = all;
            base[0][e] = before;
            base[1][e] = before + own;
        }
        __syncthreads();
        scan_experts(first, args.experts);
        for(int e = threadIdx.x; e < args.experts; e += 256)
        {
            base[0][e] += first[e];
            base[1][e] += first[e];
        }
        if(blockIdx.x == 0)
        {
            for(int e = threadIdx.x; e <= args.experts; e += 256)
            {
                args.offsets[e] = first[e];
            }
        }
    }
    __syncthreads();
    const int       lane   = threadIdx.x & 63;
    const long long token1 = token0 + each < args.tokens ? token0 + each : args.tokens;
    for(long long token = token0 + (threadIdx.x >> 6); token < token1; token += 4)
    {
        const long long slot  = token * args.k + lane;
        int             place = -1;
        if(lane < args.k)
        {
            place = args.places[slot];
            if(place >= 0)
            {
                place += base[slot / sort_block - block0][args.chosen[slot]];
                args.places[slot] = place;
            }
        }
        if(args.copy)
        {
            copy_row<Piece, STREAMED>(args, token, place, 0, pieces_of_row<Piece>(args));
        }
    }
}

// ------------------------------------------------------------------ the sum

struct combine_args
{
    void*        out; // tokens x cols
    const void*  rows; // tokens * k x cols
    const int*   places; // tokens x k
    const float* weights; // nullptr: 1
    const void*  residual; // nullptr, or tokens x cols of out's type
    long long    tokens, cols, slots;
    int          k;
    // backward
    void*        drows; // nullptr: not wanted
    float*       dweights; // nullptr: not wanted
    const void*  dout;
};

// out = sum over the choices of weight * row (+ residual), in fp32 in the order of the choices, rounded once.  Eight columns a
// thread, the last ones of a row one by one; blockIdx.x: the token, blockIdx.y: 256 pieces of its row.  Bound by memory: 8192 tokens of
// 4 rows of 8 KB, a twentieth of them masked, 322 MB, take 61 us (5.3 TB/s).
template<class InT, class OutT>
__global__ void __launch_bounds__(256) combine(const combine_args args, int block0)
{
    const long long col = ((long long)(block0 + blockIdx.y) * 256 + threadIdx.x) * 8;
    if(col >= args.cols)
    {
        return;
    }
    const bool whole = col + 8 <= args.cols;
    const int  count = whole ? 8 : (int)(args.cols - col);
    for(long long token = blockIdx.x; token < args.tokens; token += gridDim.x)
    {
        float sum[8] = {};
        const int*   places  = args.places + token * args.k;
        const float* weights = args.weights != nullptr ? args.weights + token * args.k : nullptr;
        const InT*   rows    = static_cast<const InT*>(args.rows) + col;
        const long long at   = token * args.cols + col;
        OutT* const  out     = static_cast<OutT*>(args.out) + at;
        const OutT*  added   = args.residual != nullptr ? static_cast<const OutT*>(args.residual) + at : nullptr;
        if(whole)
        {
#pragma unroll 8
            for(int j = 0; j < args.k; ++j)
            {
                const int p = places[j];
                if(p >= 0 && p < args.slots)
                {
                    const float      w = weights != nullptr ? weights[j] : 1.0f;
                    const eight<InT> y{reinterpret_cast<const eight<InT>*>(rows + p * args.cols)->v};
#pragma unroll
                    for(int v = 0; v < 8; ++v)
                    {
                        sum[v] += w * (float)y.v[v];
                    }
                }
            }
            if(added != nullptr)
            {
                const eight<OutT> r{reinterpret_cast<const eight<OutT>*>(added)->v};
#pragma unroll
                for(int v = 0; v < 8; ++v)
                {
                    sum[v] += (float)r.v[v];
                }
            }
            eight<OutT> o;
#pragma unroll
            for(int v = 0; v < 8; ++v)
            {
                o.v[v] = to_out<OutT>(sum[v]);
            }
            reinterpret_cast<eight<OutT>*>(out)->v = o.v;
            continue;
        }
        for(int v = 0; v < count; ++v)
        {
            float s = 0.0f;
            for(int j = 0; j < args.k; ++j)
            {
                const int p = places[j];
                if(p >= 0 && p < args.slots)
                {
                    s += (weights != nullptr ? weights[j] : 1.0f) * (float)rows[p * args.cols + v];
                }
            }
            out[v] = to_out<OutT>(added != nullptr ? s + (float)added[v] : s);
        }
    }
}

// The gradients: of a row, weight * dout; of a weight, the product of dout with its row.  A wave a choice: the k waves
// of a token share dout in the caches.  Bound by memory: the same sizes, 577 MB with both gradients, take 118 us (4.9 TB/s).
template<class InT, class OutT, bool STREAMED>
__global__ void __launch_bounds__(256) combine_backward(const combine_args args)
{
    const int       lane  = threadIdx.x & 63;
    const long long whole = args.cols / 8 * 8, own = whole + lane; // this lane's column of the last ones
    for(long long slot = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); slot < args.slots; slot += (long long)gridDim.x * 4)
    {
        const int  p  = args.places[slot];
        const bool is = p >= 0 && p < args.slots;
        float      dot = 0.0f;
        if(is)
        {
            const float       w  = args.weights != nullptr ? args.weights[slot] : 1.0f;
            const OutT* const d0 = static_cast<const OutT*>(args.dout) + slot / args.k * args.cols;
            const InT* const  y0 = static_cast<const InT*>(args.rows) + p * args.cols;
            InT* const        to = static_cast<InT*>(args.drows) + p * args.cols;
#pragma unroll 4
            for(long long col = lane * 8; col < whole; col += 512)
            {
                const eight<OutT> d{reinterpret_cast<const eight<OutT>*>(d0 + col)->v};
                if(args.dweights != nullptr)
                {
                    const eight<InT> y{reinterpret_cast<const eight<InT>*>(y0 + col)->v};
#pragma unroll
                    for(int v = 0; v < 8; ++v)
                    {
                        dot += (float)d.v[v] * (float)y.v[v];
                    }
                }
                if(args.drows != nullptr)
                {
                    eight<InT> o;
#pragma unroll
                    for(int v = 0; v < 8; ++v)
                    {
                        o.v[v] = to_out<InT>(w * (float)d.v[v]);
                    }
                    put<STREAMED>(reinterpret_cast<eight<InT>*>(to + col), o);
                }
            }
            if(own < args.cols)
            {
                const float d = (float)d0[own];
                dot += args.dweights != nullptr ? d * (float)y0[own] : 0.0f;
                if(args.drows != nullptr)
                {
                    to[own] = to_out<InT>(w * d);
                }
            }
        }
        if(args.dweights != nullptr)
        {
#pragma unroll
            for(int d = 1; d < 64; d *= 2)
            {
                dot += __shfl_xor(dot, d);
            }
            if(lane == 0)
            {
                args.dweights[slot] = dot;
            }
        }
    }
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_ROUTING_HPP
