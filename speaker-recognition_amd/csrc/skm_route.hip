// skm_route.hip -- routing of rows to the best few of E experts (components of a mixture, linear transforms): choice
// and weights, their gradient, the order in which the experts' products take the rows, and the weighted sum of what
// they return.  gfx950 only.
#include "skm_ops.h"

#define ROUTE_MAX_E 4096
#define ROUTE_MAX_K 64
#define ROUTE_MAX_G 64
#define ROUTE_MAX_ROWS (SKM_MAX_GROUPS * 4)     // of one launch: a workgroup has 4 rows at least

struct RouteArgs {
    const void *x;          // logits [T][ldx]
    long T, ldx;
    int E, k;
    const float *bias;      // [E] or NULL
    int groups, group_k, group_top;
    int sigmoid, renorm;
    float scale;
    int32_t *ids;           // [T][k]
    float *w;               // [T][k]
};

// weights' numerators of the chosen places: t_j proportional to p_j, the same factor for the whole row, without
// overflow or underflow of the largest one.  M: softmax the largest chosen logit, sigmoid min(0, that).
//   softmax: exp(x - M)      sigmoid: exp(x - M) / (1 + exp(x)) for x <= 0 (= sigmoid(x) exp(-M)), sigmoid(x) above
template <typename A>
__device__ __forceinline__ A route_share(A x, A M, int sigmoid)
{
    if (!sigmoid) return exp(x - M);
    if (x <= (A)0) return exp(x - M) / ((A)1 + exp(x));
    return (A)1 / ((A)1 + exp(-x));
}

// a lane's value from another lane of its 16 (CTRL 0x120 + n: n lanes on)
template <int CTRL, typename V>
__device__ __forceinline__ V dpp_ror(V v)
{
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp_ror(double v)
{
    const long long i = __builtin_bit_cast(long long, v);
    const int lo = dpp_ror<CTRL>((int)i), hi = dpp_ror<CTRL>((int)(i >> 32));
    return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ double read_lane(double v, int lane)
{
    const long long i = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_readlane((int)i, lane), hi = __builtin_amdgcn_readlane((int)(i >> 32), lane);
    return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
template <typename F>
__device__ __forceinline__ double wave_reduce(double v, F f)
{
    v = f(v, dpp_ror<0x128>(v));
    v = f(v, dpp_ror<0x124>(v));
    v = f(v, dpp_ror<0x122>(v));
    v = f(v, dpp_ror<0x121>(v));
    return f(f(read_lane(v, 0), read_lane(v, 16)), f(read_lane(v, 32), read_lane(v, 48)));
}
__device__ __forceinline__ double wave_max(double v)
{
    return wave_reduce(v, [](double a, double b) { return b > a ? b : a; });
}
__device__ __forceinline__ double wave_sum(double v)
{
    return wave_reduce(v, [](double a, double b) { return a + b; });
}
// the larger value, at equal ones the lower place; every lane gets the result
__device__ __forceinline__ void wave_best(double &v, int &at)
{
#define ROUTE_BEST(OV, OA)                              \
    {                                                   \
        const double ov = OV;                           \
        const int oa = OA;                              \
        if (ov > v || (ov == v && oa < at)) {           \
            v = ov;                                     \
            at = oa;                                    \
        }                                               \
    }
    ROUTE_BEST(dpp_ror<0x128>(v), dpp_ror<0x128>(at))
    ROUTE_BEST(dpp_ror<0x124>(v), dpp_ror<0x124>(at))
    ROUTE_BEST(dpp_ror<0x122>(v), dpp_ror<0x122>(at))
    ROUTE_BEST(dpp_ror<0x121>(v), dpp_ror<0x121>(at))
    const double wv = v;
    const int wa = at;
    v = read_lane(wv, 0);
    at = __builtin_amdgcn_readlane(wa, 0);
    ROUTE_BEST(read_lane(wv, 16), __builtin_amdgcn_readlane(wa, 16))
    ROUTE_BEST(read_lane(wv, 32), __builtin_amdgcn_readlane(wa, 32))
    ROUTE_BEST(read_lane(wv, 48), __builtin_amdgcn_readlane(wa, 48))
#undef ROUTE_BEST
}

// One wave, one row, everything in float64: lane l holds the experts l, l + 64, ...
// The order of the experts is what must not depend on rounding: two choices that differ by less than a float32
// rounding are told apart here.  -inf as a key = not to be chosen.
template <typename T, int NV>
__device__ void route_row(const RouteArgs &a, long row, int lane)
{
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const double inf = __builtin_inf();
    double key[NV];
    double top = -inf;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + 64 * i;
        key[i] = e < a.E ? (double)x[e] : -inf;
        bad |= key[i] != key[i];
        top = key[i] > top ? key[i] : top;
    }
    top = wave_max(top);
    bad |= !a.sigmoid && top == inf;
    double total = 1.0;
    if (!a.sigmoid && (a.bias || a.groups > 1 || !a.renorm)) {
        total = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) total += key[i] == -inf ? 0.0 : exp(key[i] - top);
        total = wave_sum(total);
    }
    if (a.bias || a.groups > 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (key[i] == -inf) continue;
            const int e = lane + 64 * i;
            double p = a.sigmoid ? 1.0 / (1.0 + exp(-key[i])) : exp(key[i] - top) / total;
            if (a.bias) p += (double)a.bias[e];
            bad |= p != p;
            key[i] = p;
        }
    }
    if (__any(bad)) {                       // NaN: no choice, and the weights say so
        if (lane < a.k) {
            a.ids[row * a.k + lane] = -1;
            a.w[row * a.k + lane] = __builtin_nanf("");
        }
        return;
    }
    if (a.groups > 1) {
        const int per = a.E / a.groups;
        double mine = -inf;
        for (int g = 0; g < a.groups; ++g) {
            double f1 = -inf, f2 = -inf;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = lane + 64 * i;
                if (e >= g * per && e < (g + 1) * per) {
                    if (key[i] > f1) { f2 = f1; f1 = key[i]; }
                    else if (key[i] > f2) f2 = key[i];
                }
            }
            const auto merge = [&](double o1, double o2) {
                const double lo = f1 < o1 ? f1 : o1, two = f2 > o2 ? f2 : o2;
                f1 = f1 > o1 ? f1 : o1;
                f2 = lo > two ? lo : two;
            };
            merge(dpp_ror<0x128>(f1), dpp_ror<0x128>(f2));
            merge(dpp_ror<0x124>(f1), dpp_ror<0x124>(f2));
            merge(dpp_ror<0x122>(f1), dpp_ror<0x122>(f2));
            merge(dpp_ror<0x121>(f1), dpp_ror<0x121>(f2));
            const double w1 = f1, w2 = f2;
            f1 = read_lane(w1, 0);
            f2 = read_lane(w2, 0);
            merge(read_lane(w1, 16), read_lane(w2, 16));
            merge(read_lane(w1, 32), read_lane(w2, 32));
            merge(read_lane(w1, 48), read_lane(w2, 48));
            const double s = (a.group_top == 1 || f2 == -inf) ? f1 : f1 + f2;
            if (lane == g) mine = s;
        }
        int ahead = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double s = read_lane(mine, g);
            ahead += (s > mine || (s == mine && g < lane)) ? 1 : 0;
        }
        const unsigned long long stay = __ballot(lane < a.groups && ahead < a.group_k);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + 64 * i;
            if (e >= a.E) continue;
            if (!((stay >> (e / per)) & 1)) key[i] = -inf;
            else if (!a.bias) key[i] = (double)x[e];        // within what stays the logits themselves give the order
        }
    }
    int my_id = -1;
    for (int j = 0; j < a.k; ++j) {
        double best = -inf;
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i] > best) {
                best = key[i];
                at = lane + 64 * i;
            }
        wave_best(best, at);
        if (best == -inf) break;            // uniform: nothing is left for any further place
        if (lane == j) my_id = at;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 64 * i == at) key[i] = -inf;
    }
    const double xs = my_id >= 0 ? (double)x[my_id] : -inf;
    double t = 0.0;
    if (a.renorm) {
        double M = wave_max(xs);
        if (a.sigmoid && M > 0.0) M = 0.0;
        if (my_id >= 0) t = route_share(xs, M, a.sigmoid);
        const double s = wave_sum(t);
        if (s > 0.0) t /= s;
    } else if (my_id >= 0) {
        t = a.sigmoid ? 1.0 / (1.0 + exp(-xs)) : exp(xs - top) / total;
    }
    if (lane < a.k) {
        a.ids[row * a.k + lane] = my_id;
        a.w[row * a.k + lane] = (float)(t * (double)a.scale);
    }
}

// Every row in float64: what the fast kernel has no form for (float64 logits that need probabilities, many groups).
template <typename T, int NV>
__global__ __launch_bounds__(256) void k_route_wide(RouteArgs a)
{
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row < a.T) route_row<T, NV>(a, row, lane);
}

// reductions over the L = 16 or 64 lanes of a row; every lane gets the result
template <int L, typename V, typename F>
__device__ __forceinline__ V row_reduce(V v, F f)
{
    v = f(v, dpp_ror<0x128>(v));
    v = f(v, dpp_ror<0x124>(v));
    v = f(v, dpp_ror<0x122>(v));
    v = f(v, dpp_ror<0x121>(v));
    if (L == 64) {
        const int i = __builtin_bit_cast(int, v);
        const V a = __builtin_bit_cast(V, __builtin_amdgcn_readlane(i, 0)), b = __builtin_bit_cast(V, __builtin_amdgcn_readlane(i, 16));
        const V c = __builtin_bit_cast(V, __builtin_amdgcn_readlane(i, 32)), d = __builtin_bit_cast(V, __builtin_amdgcn_readlane(i, 48));
        v = f(f(a, b), f(c, d));
    }
    return v;
}
template <int L> __device__ __forceinline__ unsigned row_max(unsigned v)
{
    return row_reduce<L>(v, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
template <int L> __device__ __forceinline__ float row_max(float v)
{
    return row_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L> __device__ __forceinline__ float row_sum(float v)
{
    return row_reduce<L>(v, [](float a, float b) { return a + b; });
}

// order of float32 numbers as unsigned ones (0 is below all of them), and back
__device__ __forceinline__ unsigned order_bits(float x)
{
    const unsigned u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(unsigned k)
{
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// v[0 .. N) in descending order (Batcher's odd-even merge sort)
template <int N>
__device__ __forceinline__ void sort_down(unsigned *v)
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j <= N - 1 - k; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const unsigned a = v[i + j], b = v[i + j + k];
                        v[i + j] = a > b ? a : b;
                        v[i + j + k] = a > b ? b : a;
                    }
}
// the 8 largest of two descending runs of 8, descending, in a
__device__ __forceinline__ void merge_down8(unsigned *a, const unsigned *b)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = a[i] > b[7 - i] ? a[i] : b[7 - i];       // rises and falls once
#pragma unroll
    for (int k = 4; k >= 1; k /= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & k)) {
                const unsigned x = a[i], y = a[i + k];
                a[i] = x > y ? x : y;
                a[i + k] = x > y ? y : x;
            }
}

// One row per L lanes (16: four rows a wave), lane l holds the experts l, l + L, ...: NV of them.
//   A choice is a 32-bit key: the float32 number in an order-preserving form, its last log2(NV) bits replaced by the place
//   in the lane (lower place = larger), so that one v_max keeps the expert with it.  A lane sorts its keys and keeps the 8
//   largest; in each round the largest head of the row comes from four DPP steps, the lowest lane that holds it from a
//   ballot, and that lane moves up.  A lane that has given all 8 leaves the row in doubt.
//   The order itself is that of 64 bits.  Half-precision logits without a bias are exact in the key.  Otherwise one more
//   than k is taken, groups that are as near on either side of the choice are settled by their float64 scores, neighbours
//   are compared without the cut bits, and where two are not further apart than what float32
//   arithmetic and (the last one taken and the first that was not) the cut bits can have moved them, the row's choices are
//   ranked again by their float64 values -- for random logits about one row in a thousand.  Only where the one after that
//   is as near, and for NaN and infinities, the whole wave does the row again in float64 (route_row): that costs 6 us at
//   least, for one row.
//   Error of p: exp of a difference d <= 0 by exp2(d log2 e): (3 |d| + 2) 2^-24 of it, |d| exp(d) <= 0.37; the sum S of E
//   terms: (NV + 6) additions and the terms' errors, in all (NV + 48) 2^-24 / S bounds it; 1 / (1 + exp(-x)):
//   p (1 - p) |x| <= 0.23 and an approximate reciprocal, 8 2^-24.  Error of c = p + bias: that and |c| 2^-24; of the key: |c| 2^-(23 - bits).
// GROUPED: with groups of experts (without, those take registers that the rows in flight need).
// Bound by the vector ALU (sort of the keys, k + 1 steps of the row's largest head, each waiting for the one before), not
// by memory: 16384 x 256 float32, 4 of 8 groups, bias: 23 us (0.8 TB/s; vector ALU 73 % of the cycles in which a CU has
// waves); 32768 x 128 bf16 with a bias 18 us (94 %); 50001 x 512 float64, k = 20, 70 us (3.0 TB/s); one row 3.5 us, the
// launch.
template <typename T, int NV, int L, bool GROUPED>
__global__ __launch_bounds__(256, NV <= 16 ? 4 : NV == 32 ? (L == 16 ? 3 : 2) : 1) void k_route(RouteArgs a)
{
    constexpr int R = 64 / L, BITS = NV == 1 ? 0 : NV == 2 ? 1 : NV == 4 ? 2 : NV == 8 ? 3 : NV == 16 ? 4 : NV == 32 ? 5 : 6;
    constexpr bool HALF = sizeof(T) == 2;
    constexpr int PL = (ROUTE_MAX_K + L - 1) / L;       // places of a lane
    constexpr int NV64 = (NV * L + 63) / 64;
    __shared__ int32_t chosen[4 * R][ROUTE_MAX_K + 2], ranked[4 * R][ROUTE_MAX_K];
    __shared__ double value[4 * R][ROUTE_MAX_K + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % L, sub = lane / L;
    const long row0 = ((long)blockIdx.x * 4 + wave) * R;
    if (row0 >= a.T) return;                            // whole waves
    const long row = row0 + sub < a.T ? row0 + sub : a.T - 1;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const float inf = __builtin_inff();
    float c[NV];
    bool bad = false;
    float top = -inf;
    // an expert that is not to be chosen has c = -inf, here and below
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = l + L * i;
        const T v = e < a.E ? x[e] : (T)-inf;
        c[i] = (float)v + 0.f;              // -0 and 0 are the same number
        if (sizeof(T) == 8) bad |= c[i] == -inf && v != (T)-inf;        // masked is what is -inf in float64
        bad |= c[i] != c[i];
        top = fmaxf(top, c[i]);
    }
    bad |= !a.sigmoid && top == inf;
    float total = 1.f, err = 0.f;
    if (!a.sigmoid && (a.bias || GROUPED || !a.renorm)) {
        top = row_max<L>(top);
        total = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) total += c[i] == -inf ? 0.f : __expf(c[i] - top);
        total = row_sum<L>(total);
        err = (float)(NV + 48) * 5.9604645e-8f / total;
    } else if (a.sigmoid) {
        err = 8.f * 5.9604645e-8f;
    }
    if (a.bias || GROUPED) {                // c becomes the probability, with the bias
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float p = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-c[i])) : __expf(c[i] - top) * inv;
            c[i] = c[i] == -inf ? -inf : p;
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = l + L * i;
                const float b = e < a.E ? a.bias[e] : -inf;
                c[i] = c[i] == -inf ? -inf : c[i] + b;
                bad |= c[i] != c[i];
            }
        }
    }
    bool doubt = false;
    if constexpr (GROUPED) {
        // the two largest c of a group in every lane of the row; lane g keeps those of group g
        const int per = a.E / a.groups;
        const unsigned inv = per > 1 ? (unsigned)(((1ull << 32) + per - 1) / per) : 0;
        float s1 = -inf, s2 = -inf, f1 = -inf, f2 = -inf;
        const auto take = [&](float v) {
            f2 = fmaxf(f2, fminf(f1, v));
            f1 = fmaxf(f1, v);
        };
        const auto give = [&](int g) {      // over the lanes of the row; lane g keeps the result
#define ROUTE_TOP2(CTRL)                                            \
    {                                                               \
        const float o1 = dpp_ror<CTRL>(f1), o2 = dpp_ror<CTRL>(f2); \
        f2 = fmaxf(fmaxf(f2, o2), fminf(f1, o1));                   \
        f1 = fmaxf(f1, o1);                                         \
    }
            ROUTE_TOP2(0x128) ROUTE_TOP2(0x124) ROUTE_TOP2(0x122) ROUTE_TOP2(0x121)
#undef ROUTE_TOP2
            if (L == 64) {
#pragma unroll
                for (int m = 32; m > 8; m >>= 1) {
                    const float o1 = __shfl_xor(f1, m), o2 = __shfl_xor(f2, m);
                    f2 = fmaxf(fmaxf(f2, o2), fminf(f1, o1));
                    f1 = fmaxf(f1, o1);
                }
            }
            if (l == g) {
                s1 = f1;
                s2 = f2;
            }
            f1 = f2 = -inf;
        };
        if (per % L == 0) {                 // a group is per / L places of every lane
            int left = per / L, g = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                take(c[i]);
                if (--left == 0 && g < a.groups) {
                    give(g++);
                    left = per / L;
                }
            }
        } else {
            for (int g = 0; g < a.groups; ++g) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int e = l + L * i;
                    const int ge = per > 1 ? (int)__umulhi((unsigned)e, inv) : e;
                    take(ge == g ? c[i] : -inf);
                }
                give(g);
            }
        }
        const bool pair = a.group_top == 2 && s2 != -inf;
        const float score = pair ? s1 + s2 : s1;
        // what two scores can have been moved against each other
        float near = s1 == -inf ? 0.f : 4.f * err + 2.3841858e-7f * (fabsf(s1) + (pair ? fabsf(s2) : 0.f));
        near = row_max<L>(near);
        int ahead = 0;
        bool kept;
        unsigned long long all;
        if (L == 16) {                      // the other groups' scores by turning the row's lanes
#define ROUTE_TURNS(SEE)                                                                                              \
    SEE(1) SEE(2) SEE(3) SEE(4) SEE(5) SEE(6) SEE(7) SEE(8) SEE(9) SEE(10) SEE(11) SEE(12) SEE(13) SEE(14) SEE(15)
#define ROUTE_AHEAD(N)                                                                                                 \
    {                                                                                                                  \
        const float o = dpp_ror<0x120 + N>(score);                                                                     \
        const int g = dpp_ror<0x120 + N>(l);                                                                           \
        ahead += g < a.groups && (o > score || (o == score && g < l)) ? 1 : 0;                                         \
    }
            ROUTE_TURNS(ROUTE_AHEAD)
            kept = l < a.groups && ahead < a.group_k;
            bool open = false;              // near a group on the other side of the choice
#define ROUTE_NEAR(N)                                                                                                  \
    {                                                                                                                  \
        const float o = dpp_ror<0x120 + N>(score);                                                                     \
        const int g = dpp_ror<0x120 + N>(l);                                                                           \
        const bool okept = dpp_ror<0x120 + N>((int)kept) != 0;  /* by all lanes: one that sits out is not read */      \
        open |= l < a.groups && g < a.groups && okept != kept && fabsf(score - o) <= near;                             \
    }
            ROUTE_TURNS(ROUTE_NEAR)
            const unsigned long long rows = __ballot(open);
            if (rows) {                     // uniform: the open groups' scores in float64, the best of them for what is left
                unsigned todo = (unsigned)((rows | rows >> 16 | rows >> 32 | rows >> 48) & 0xFFFFull);
                double total64 = 1.0;
                const double top64 = (double)top;
                if (!a.sigmoid) {
                    double t = 0.0;
#pragma unroll 4
                    for (int e = l; e < a.E; e += 16) t += exp((double)x[e] - top64);
                    t = t + dpp_ror<0x128>(t);
                    t = t + dpp_ror<0x124>(t);
                    t = t + dpp_ror<0x122>(t);
                    t = t + dpp_ror<0x121>(t);
                    total64 = t;
                }
                const double dinf = __builtin_inf();
                double best64 = -dinf;
                while (todo) {
                    const int g = __ffs((int)todo) - 1;
                    todo &= todo - 1;
                    double d1 = -dinf, d2 = -dinf;
                    for (int e = g * per + l; e < (g + 1) * per; e += 16) {
                        const double v = (double)x[e], b = a.bias ? (double)a.bias[e] : 0.0;
                        const double p = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - top64) / total64;
                        const double w = v == -dinf || b == -dinf ? -dinf : p + b;
                        d2 = fmax(d2, fmin(d1, w));
                        d1 = fmax(d1, w);
                    }
#define ROUTE_TOP2(CTRL)                                              \
    {                                                                 \
        const double o1 = dpp_ror<CTRL>(d1), o2 = dpp_ror<CTRL>(d2);  \
        d2 = fmax(fmax(d2, o2), fmin(d1, o1));                        \
        d1 = fmax(d1, o1);                                            \
    }
                    ROUTE_TOP2(0x128) ROUTE_TOP2(0x124) ROUTE_TOP2(0x122) ROUTE_TOP2(0x121)
#undef ROUTE_TOP2
                    if (l == g) best64 = a.group_top == 2 && d2 != -dinf ? d1 + d2 : d1;
                }
                int settled = 0, before = 0;
#define ROUTE_SETTLE(N)                                                                                                \
    {                                                                                                                  \
        const double o = dpp_ror<0x120 + N>(best64);                                                                   \
        const int g = dpp_ror<0x120 + N>(l);                                                                           \
        const bool oopen = dpp_ror<0x120 + N>((int)open) != 0, okept = dpp_ror<0x120 + N>((int)kept) != 0;             \
        settled += okept && !oopen ? 1 : 0;                                                                            \
        before += oopen && (o > best64 || (o == best64 && g < l)) ? 1 : 0;                                             \
    }
                ROUTE_TURNS(ROUTE_SETTLE)
                if (open) kept = before < a.group_k - settled;
            }
#undef ROUTE_TURNS
#undef ROUTE_AHEAD
#undef ROUTE_NEAR
#undef ROUTE_SETTLE
            all = __ballot(kept);
        } else {
            for (int g = 0; g < a.groups; ++g) {
                const float o = __shfl(score, g);
                ahead += (o > score || (o == score && g < l)) ? 1 : 0;
            }
            kept = l < a.groups && ahead < a.group_k;
            all = __ballot(kept);
            for (int g = 0; g < a.groups; ++g) {
                const float o = __shfl(score, g);
                bad |= l < a.groups && (((all >> g) & 1) != 0) != kept && fabsf(score - o) <= near;
            }
        }
        const unsigned long long stay = L == 64 ? all : (all >> (sub * L)) & 0xFFFFull;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = l + L * i;
            const int ge = per > 1 ? (int)__umulhi((unsigned)e, inv) : e;
            if (!a.bias) c[i] = e < a.E ? (float)x[e] + 0.f : -inf;     // the order goes by the logits
            if (ge >= a.groups || !((stay >> (ge & 63)) & 1)) c[i] = -inf;
        }
    }
    constexpr int DEEP = NV < 8 ? NV : 8;
    unsigned key[NV < 8 ? 8 : NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        key[i] = c[i] == -inf ? 0u : (order_bits(c[i] + 0.f) & ~(unsigned)(NV - 1)) | (unsigned)(NV - 1 - i);
    sort_down<DEEP>(key);
#pragma unroll
    for (int i = 8; i < NV; i += 8) {
        sort_down<8>(key + i);
        merge_down8(key, key + i);
    }
    const bool exact = HALF && !a.bias;
    int32_t *mine = chosen[wave * R + sub];
    const int take_n = exact ? a.k : a.k + 1;
    for (int j = l; j < take_n + 1; j += L) mine[j] = -1;
    wave_sync();
    unsigned last = 0, after = 0;           // keys of place k - 1 and k
    int given = 0;
    for (int j = 0; j < take_n; ++j) {
        const unsigned best = row_max<L>(key[0]);
        const unsigned long long who = __ballot(key[0] == best);
        const int first = L == 64 ? __ffsll((long long)who) - 1 : __ffs((int)((who >> (sub * L)) & 0xFFFFu)) - 1;
        last = j == a.k ? last : best;
        after = best;
        if (l == first && best != 0) {
            mine[j] = l + L * (NV - 1 - (int)(best & (unsigned)(NV - 1)));
            ++given;
#pragma unroll
            for (int i = 0; i + 1 < DEEP; ++i) key[i] = key[i + 1];
            key[DEEP - 1] = 0;
        }
    }
    bad |= NV > DEEP && given == DEEP;
    wave_sync();
    if (!exact) {
        const unsigned m = ~(unsigned)(NV - 1);
        // whether a choice b may belong in front of a
        const auto close = [&](unsigned ka, unsigned kb) {
            if (kb == 0) return false;
            if (!a.bias) return ((ka ^ kb) & m) == 0;
            const float f = order_value(ka & m), g = order_value(kb & m);
            return f - g <= 2.f * err + fmaxf(fabsf(f), fabsf(g)) * (1.1920929e-7f * (float)(1 + 2 * NV));
        };
        bad |= close(last, row_max<L>(key[0]));
        doubt |= close(last, after);
        double *val = value[wave * R + sub];
        const float inv = 1.f / total;
        for (int j = l; j < a.k; j += L) {
            const int i = mine[j];
            if (i < 0) continue;
            const T v = x[i];
            float f = (float)v;
            if (a.bias) f = (a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-f)) : __expf(f - top) * inv) + a.bias[i];
            val[j] = a.bias ? (double)f : (double)v;
        }
        wave_sync();
        for (int j = l; j + 1 < a.k; j += L) {
            const int i0 = mine[j], i1 = mine[j + 1];
            if (i1 < 0) continue;
            const double v0 = val[j], v1 = val[j + 1];
            if (a.bias) doubt |= !((float)(v0 - v1) > 2.f * err + 2.3841858e-7f * fmaxf(fabsf((float)v0), fabsf((float)v1)));
            else doubt |= !(v0 > v1 || (v0 == v1 && i0 < i1));
        }
        const unsigned long long rows = __ballot(doubt);
        if (rows) {                         // uniform
            double total64 = 1.0, top64 = 0.0;
            if (a.bias && !a.sigmoid) {
                top64 = (double)top;
                double t = 0.0;
#pragma unroll 4
                for (int e = l; e < a.E; e += L) t += exp((double)x[e] - top64);
                t = t + dpp_ror<0x128>(t);
                t = t + dpp_ror<0x124>(t);
                t = t + dpp_ror<0x122>(t);
                t = t + dpp_ror<0x121>(t);
                if (L == 64) t = (read_lane(t, 0) + read_lane(t, 16)) + (read_lane(t, 32) + read_lane(t, 48));
                total64 = t;
            }
            if (a.bias) {
                for (int j = l; j < take_n; j += L) {
                    const int i = mine[j];
                    if (i < 0) continue;
                    const double v = (double)x[i];
                    val[j] = (a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - top64) / total64) + (double)a.bias[i];
                }
            } else if (l == a.k % L && mine[a.k] >= 0) {
                val[a.k] = (double)x[mine[a.k]];
            }
            int32_t *to = ranked[wave * R + sub];
            for (int j = l; j < a.k; j += L) to[j] = -1;
            wave_sync();
            for (int j = l; j < take_n; j += L) {
                const int i = mine[j];
                if (i < 0) continue;
                const double v = val[j];
                int rank = 0;
                for (int o = 0; o < take_n; ++o) {
                    const int io = mine[o];
                    rank += io >= 0 && (val[o] > v || (val[o] == v && io < i)) ? 1 : 0;
                }
                if (rank < a.k) to[rank] = i;
            }
            wave_sync();
            // a row without doubt has the same order
            for (int j = l; j < a.k; j += L) mine[j] = to[j];
            wave_sync();
        }
    }
    // weights: lane l has the places l, l + L, ...
    int id[PL];
    float t[PL];
    if (a.renorm) {
        T xs[PL];
        float M = -inf;
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            const int j = l + q * L;
            id[q] = j < a.k ? mine[j] : -1;
            xs[q] = id[q] >= 0 ? x[id[q]] : (T)-inf;
            if (sizeof(T) < 8) M = fmaxf(M, (float)xs[q]);
        }
        float sum = 0.f;
        if (sizeof(T) == 8) {               // without a bias: the first choice is the largest
            const int lead = mine[0];
            double Md = lead >= 0 ? (double)x[lead] : 0.0;
            if (a.sigmoid && Md > 0.0) Md = 0.0;
#pragma unroll
            for (int q = 0; q < PL; ++q) {
                const double v = (double)xs[q];
                t[q] = id[q] < 0 ? 0.f : !a.sigmoid ? expf((float)(v - Md))
                                       : v <= 0.0   ? expf((float)(v - Md)) / (1.f + expf((float)v))
                                                    : 1.f / (1.f + expf((float)-v));
                sum += t[q];
            }
        } else {
            M = row_max<L>(M);
            if (a.sigmoid && M > 0.f) M = 0.f;
#pragma unroll
            for (int q = 0; q < PL; ++q) {
                t[q] = id[q] >= 0 ? route_share((float)xs[q], M, a.sigmoid) : 0.f;
                sum += t[q];
            }
        }
        sum = row_sum<L>(sum);
        const float f = sum > 0.f ? a.scale / sum : 0.f;
#pragma unroll
        for (int q = 0; q < PL; ++q) t[q] *= f;
    } else {
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            const int j = l + q * L;
            id[q] = j < a.k ? mine[j] : -1;
            const float xs = id[q] >= 0 ? (float)x[id[q]] : -inf;
            t[q] = id[q] < 0 ? 0.f : a.scale * (a.sigmoid ? 1.f / (1.f + expf(-xs)) : expf(xs - top) / total);
        }
    }
    const unsigned long long again = __ballot(bad);
    const unsigned long long rowmask = (L == 64 ? ~0ull : 0xFFFFull << (sub * L));
    if (row0 + sub < a.T && !(again & rowmask)) {
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            const int j = l + q * L;
            if (j < a.k) {
                a.ids[row * a.k + j] = id[q];
                a.w[row * a.k + j] = t[q];
            }
        }
    }
    if (!again) return;
    for (int s = 0; s < R; ++s)             // one after the other
        if (row0 + s < a.T && (again & (L == 64 ? ~0ull : 0xFFFFull << (s * L)))) route_row<T, NV64>(a, row0 + s, lane);
}

struct RouteBackArgs {
    const void *x;
    long T, ldx;
    int E, k;
    const int32_t *ids;
    const float *g;         // dL/dweights [T][k]
    int sigmoid, renorm;
    float scale;
    void *dx;               // [T][E] in the type of x
};

// One wave per row.  Lane j < k holds place j: its logit, its share and d_j, what it adds to the gradient of its
// logit.  Only softmax without renormalisation has a gradient beside the chosen places (- p_i sum_j p_j u_j):
//   renorm   with s_j = t_j / sum t (t of route_share), G = sum_j s_j g_j:
//            softmax d_j = scale s_j (g_j - G)          sigmoid d_j = scale s_j (1 - p_j) (g_j - G)
//   else     sigmoid d_j = scale g_j p_j (1 - p_j)      softmax d_j = scale g_j p_j, dx_i = sum d_j - p_i sum_j d_j
// so all the other variants read k logits of a row and not E.
template <typename T, typename A>
__global__ __launch_bounds__(256) void k_route_backward(RouteBackArgs a)
{
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.T) return;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *dx = static_cast<T *>(a.dx) + row * a.E;
    const A inf = (A)__builtin_inf();
    int id = -1;
    A xs = -inf, g = 0;
    if (lane < a.k) {
        id = a.ids[row * a.k + lane];
        if (id < 0 || id >= a.E) id = -1;
        else {
            xs = (A)x[id];
            g = (A)a.g[row * a.k + lane];
            if (xs == -inf) id = -1;
        }
    }
    const bool there = id >= 0;
    A d = 0, D = 0, top = 0, total = 1;
    if (a.renorm) {
        A M = wave_max(there ? xs : -inf);
        if (a.sigmoid && M > (A)0) M = 0;
        A t = there ? route_share(xs, M, a.sigmoid) : (A)0;
        const A s = wave_sum(t);
        t = s > (A)0 ? t / s : t;
        const A G = wave_sum(there ? t * g : (A)0);
        d = there ? (A)a.scale * t * (g - G) : (A)0;
        if (a.sigmoid && there) d *= (A)1 / ((A)1 + exp(xs));
    } else if (a.sigmoid) {
        if (there) d = (A)a.scale * g / ((A)1 + exp(-xs)) / ((A)1 + exp(xs));
    } else {
        top = -inf;
        for (int e = lane; e < a.E; e += 64) top = (A)x[e] > top ? (A)x[e] : top;
        top = wave_max(top);
        if (top == -inf) top = 0;
        total = 0;
        for (int e = lane; e < a.E; e += 64) total += exp((A)x[e] - top);
        total = wave_sum(total);
        if (there) d = (A)a.scale * g * exp(xs - top) / total;
        D = wave_sum(d);
    }
    for (int e0 = 0; e0 < a.E; e0 += 64) {
        const int e = e0 + lane;
        A v = 0;
        if (D != (A)0 && e < a.E) v = -D * exp((A)x[e] - top) / total;
        for (int j = 0; j < a.k; ++j) {                 // in the order of the places: the same bits every time
            const int at = __builtin_amdgcn_readlane(id, j);
            const A dj = (A)read_lane((double)d, j);
            if (at == e) v += dj;
        }
        if (e < a.E) dx[e] = (T)v;
    }
}

// The same for rows of up to EMAX experts: 16 lanes a row, four rows a wave.  What the chosen places add goes through a
// row in LDS (places with the same expert are added first, in their order, by the first of them), so that the row leaves
// in 16-byte stores; a wave per row with a comparison per place and element took three times as long (32768 x 128
// bf16, k = 8: 21.6 us against 7.1).
template <typename T, int EMAX>
__global__ __launch_bounds__(256) void k_route_backward16(RouteBackArgs a)
{
    constexpr int PL = ROUTE_MAX_K / 16, V = 16 / sizeof(T);
    __shared__ float buf[16][EMAX + 4];
    __shared__ int32_t sid[16][ROUTE_MAX_K];
    __shared__ float sd[16][ROUTE_MAX_K];
    const int lane = threadIdx.x & 63, l = lane & 15, slot = threadIdx.x >> 4;
    const long row0 = (long)blockIdx.x * 16 + slot;
    if ((long)blockIdx.x * 16 + (threadIdx.x >> 6) * 4 >= a.T) return;      // whole waves
    const bool live = row0 < a.T;
    const long row = live ? row0 : a.T - 1;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *dx = static_cast<T *>(a.dx) + row * a.E;
    const float inf = __builtin_inff();
    int id[PL];
    float xs[PL], g[PL], d[PL], top = -inf;
#pragma unroll
    for (int q = 0; q < PL; ++q) {
        const int j = l + 16 * q;
        id[q] = -1;
        xs[q] = -inf;
        g[q] = d[q] = 0.f;
        if (j < a.k) {
            const int i = a.ids[row * a.k + j];
            if (i >= 0 && i < a.E) {
                xs[q] = (float)x[i];
                if (xs[q] != -inf) {
                    id[q] = i;
                    g[q] = a.g[row * a.k + j];
                }
            }
        }
        top = fmaxf(top, xs[q]);
    }
    float D = 0.f, total = 1.f;
    if (a.renorm) {
        float M = row_max<16>(top);
        if (a.sigmoid && M > 0.f) M = 0.f;
        float sum = 0.f, t[PL];
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            t[q] = id[q] >= 0 ? route_share(xs[q], M, a.sigmoid) : 0.f;
            sum += t[q];
        }
        sum = row_sum<16>(sum);
        float G = 0.f;
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            t[q] = sum > 0.f ? t[q] / sum : t[q];
            G += t[q] * g[q];
        }
        G = row_sum<16>(G);
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            d[q] = id[q] >= 0 ? a.scale * t[q] * (g[q] - G) : 0.f;
            if (a.sigmoid && id[q] >= 0) d[q] *= 1.f / (1.f + expf(xs[q]));
        }
    } else if (a.sigmoid) {
#pragma unroll
        for (int q = 0; q < PL; ++q)
            if (id[q] >= 0) d[q] = a.scale * g[q] / (1.f + expf(-xs[q])) / (1.f + expf(xs[q]));
    } else {
        top = -inf;
        for (int e = l; e < a.E; e += 16) top = fmaxf(top, (float)x[e]);
        top = row_max<16>(top);
        if (top == -inf) top = 0.f;
        total = 0.f;
        for (int e = l; e < a.E; e += 16) total += expf((float)x[e] - top);
        total = row_sum<16>(total);
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            if (id[q] >= 0) d[q] = a.scale * g[q] * expf(xs[q] - top) / total;
            D += d[q];
        }
        D = row_sum<16>(D);
    }
#pragma unroll
    for (int q = 0; q < PL; ++q) {
        const int j = l + 16 * q;
        if (j < a.k) {
            sid[slot][j] = id[q];
            sd[slot][j] = d[q];
        }
    }
    for (int e = l * 4; e < a.E; e += 64) *reinterpret_cast<float4 *>(&buf[slot][e]) = make_float4(0.f, 0.f, 0.f, 0.f);
    wave_sync();
#pragma unroll
    for (int q = 0; q < PL; ++q) {
        if (16 * q >= a.k) break;
        float sum = 0.f;
        bool first = true;
        for (int o = 0; o < a.k; ++o) {
            const bool same = sid[slot][o] == id[q];
            sum += same ? sd[slot][o] : 0.f;
            first &= !(same && o < l + 16 * q);
        }
        if (id[q] >= 0 && first) buf[slot][id[q]] = sum;
    }
    wave_sync();
    if (!live) return;
    typedef T vt __attribute__((ext_vector_type(V)));
    for (int e = l * V; e < a.E; e += 16 * V) {
        float v[V];
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = e + q < a.E ? buf[slot][e + q] : 0.f;
        if (D != 0.f) {
#pragma unroll
            for (int q = 0; q < V; ++q)
                if (e + q < a.E) v[q] -= D * expf((float)x[e + q] - top) / total;
        }
        if (e + V <= a.E) {
            vt o;
#pragma unroll
            for (int q = 0; q < V; ++q) o[q] = (T)v[q];
            store_any(dx + e, o);
        } else {
#pragma unroll
            for (int q = 0; q < V; ++q)
                if (e + q < a.E) dx[e + q] = (T)v[q];
        }
    }
}

template <typename T>
static void route_back_go(const RouteBackArgs &a, hipStream_t st)
{
    // 16 lanes a row up to 512 experts: 16384 x 512 bf16, k 8, 9.7 us, a wave a row 20.5.  Softmax without renormalisation has
    // a gradient at every expert and would be better off with a wave a row from there on (35 against 31 us; 16384 x 1024 60
    // against 80), the others with 16 lanes for longer (16384 x 1024: 35 against 14.5).
    const dim3 grid((unsigned)((a.T + 15) / 16)), block(256);
    if (a.E <= 128) hipLaunchKernelGGL((k_route_backward16<T, 128>), grid, block, 0, st, a);
    else if (a.E <= 512) hipLaunchKernelGGL((k_route_backward16<T, 512>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_route_backward<T, float>), dim3((unsigned)((a.T + 3) / 4)), block, 0, st, a);
}

template <typename T, int NV, int L>
static void route_go(const RouteArgs &a, hipStream_t st)
{
    const long per = 4 * (64 / L);
    const dim3 grid((unsigned)((a.T + per - 1) / per)), block(256);
    if constexpr (sizeof(T) < 8) {
        if (a.groups > 1) {
            hipLaunchKernelGGL((k_route<T, NV, L, true>), grid, block, 0, st, a);
            return;
        }
    }
    hipLaunchKernelGGL((k_route<T, NV, L, false>), grid, block, 0, st, a);
}

template <typename T, int NV>
static void route_go_wide(const RouteArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((k_route_wide<T, NV>), dim3((unsigned)((a.T + 3) / 4)), dim3(256), 0, st, a);
}

template <typename T>
static void route_launch(const RouteArgs &a, hipStream_t st)
{
    // 16 lanes a row up to 512 experts (32 of them a lane), the whole wave above: 16384 x 512 float32, k 8, 15.5 us (a wave a
    // row 20.4), 16384 x 1024 42.7 (16 lanes 54.3), bf16 12.6 (16.3) and 31.4 (35.8); 50001 x 512 float64, k 20, 69 (75).
    // In float64 throughout: probabilities of float64 logits; more groups than a row has lanes.
    const bool wide = (sizeof(T) == 8 && (a.bias || a.groups > 1 || (!a.renorm && !a.sigmoid))) || a.groups > (a.E <= 512 ? 16 : 64);
    if (wide) {
        if (a.E <= 64) route_go_wide<T, 1>(a, st);
        else if (a.E <= 256) route_go_wide<T, 4>(a, st);
        else if (a.E <= 1024) route_go_wide<T, 16>(a, st);
        else route_go_wide<T, 64>(a, st);
        return;
    }
    if (a.E <= 16) route_go<T, 1, 16>(a, st);
    else if (a.E <= 32) route_go<T, 2, 16>(a, st);
    else if (a.E <= 64) route_go<T, 4, 16>(a, st);
    else if (a.E <= 128) route_go<T, 8, 16>(a, st);
    else if (a.E <= 256) route_go<T, 16, 16>(a, st);
    else if (a.E <= 512) route_go<T, 32, 16>(a, st);
    else if (a.E <= 1024) route_go<T, 16, 64>(a, st);
    else if (a.E <= 2048) route_go<T, 32, 64>(a, st);
    else route_go<T, 64, 64>(a, st);
}

extern "C" int skm_route(void *ctx_, const void *x, int dtype, long T, int E, long ldx, int k, int scores,
                         const float *bias, int groups, int group_k, int group_top, int renorm, float scale,
                         int32_t *ids, float *weights, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && skm_dt_size(dtype) && T >= 0 && E >= 1 && ldx >= E && (T == 0 || (x && ids && weights)),
                "skm_route: bad argument");
    SKM_REQUIRE(scores == SKM_ROUTE_SOFTMAX || scores == SKM_ROUTE_SIGMOID, "skm_route: unknown scores %d", scores);
    SKM_REQUIRE(k >= 1 && k <= E, "skm_route: k = %d of %d experts", k, E);
    SKM_REQUIRE(groups >= 1 && E % groups == 0 && group_k >= 1 && group_k <= groups,
                "skm_route: %d of %d groups over %d experts", group_k, groups, E);
    SKM_REQUIRE(k <= E / groups * group_k, "skm_route: k = %d of the %d experts that %d groups hold", k,
                E / groups * group_k, group_k);
    SKM_REQUIRE(group_top == 1 || group_top == 2, "skm_route: group_top is 1 or 2");
    if (E > ROUTE_MAX_E || k > ROUTE_MAX_K || groups > ROUTE_MAX_G || T > 4L * 0x7FFFFFFF) {
        skm_set_error("skm_route: built for %d experts, k = %d, %d groups", ROUTE_MAX_E, ROUTE_MAX_K, ROUTE_MAX_G);
        return SKM_ERR_UNSUPPORTED;
    }
    if (T == 0) return SKM_OK;
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_route", st);
    for (long t = 0; t < T; t += ROUTE_MAX_ROWS) {
        const RouteArgs a{static_cast<const char *>(x) + t * ldx * skm_dt_size(dtype), T - t < ROUTE_MAX_ROWS ? T - t : ROUTE_MAX_ROWS,
                          ldx, E, k, bias, groups, group_k, group_top, scores == SKM_ROUTE_SIGMOID, renorm != 0, scale,
                          ids + t * k, weights + t * k};
        switch (dtype) {
        case SKM_DT_F32: route_launch<float>(a, st); break;
        case SKM_DT_BF16: route_launch<bf16_t>(a, st); break;
        case SKM_DT_F16: route_launch<f16_t>(a, st); break;
        default: route_launch<double>(a, st); break;
        }
        SKM_HIP(hipGetLastError());
    }
    return SKM_OK;
}

extern "C" int skm_route_backward(void *ctx_, const void *x, int dtype, long T, int E, long ldx, int k, int scores,
                                  int renorm, float scale, const int32_t *ids, const float *dweights, void *dx,
                                  void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && skm_dt_size(dtype) && T >= 0 && E >= 1 && ldx >= E && (T == 0 || (x && ids && dweights && dx)),
                "skm_route_backward: bad argument");
    SKM_REQUIRE(scores == SKM_ROUTE_SOFTMAX || scores == SKM_ROUTE_SIGMOID, "skm_route_backward: unknown scores %d", scores);
    SKM_REQUIRE(k >= 1 && k <= E, "skm_route_backward: k = %d of %d experts", k, E);
    if (E > ROUTE_MAX_E || k > ROUTE_MAX_K || T > 4L * 0x7FFFFFFF) {
        skm_set_error("skm_route_backward: built for %d experts, k = %d", ROUTE_MAX_E, ROUTE_MAX_K);
        return SKM_ERR_UNSUPPORTED;
    }
    if (T == 0) return SKM_OK;
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_route_backward", st);
    for (long t = 0; t < T; t += ROUTE_MAX_ROWS) {
        const int size = skm_dt_size(dtype);
        const RouteBackArgs a{static_cast<const char *>(x) + t * ldx * size, T - t < ROUTE_MAX_ROWS ? T - t : ROUTE_MAX_ROWS,
                              ldx, E, k, ids + t * k, dweights + t * k, scores == SKM_ROUTE_SIGMOID, renorm != 0, scale,
                              static_cast<char *>(dx) + t * E * size};
        switch (dtype) {
        case SKM_DT_F32: route_back_go<float>(a, st); break;
        case SKM_DT_BF16: route_back_go<bf16_t>(a, st); break;
        case SKM_DT_F16: route_back_go<f16_t>(a, st); break;
        default:
            hipLaunchKernelGGL((k_route_backward<double, double>), dim3((unsigned)((a.T + 3) / 4)), dim3(256), 0, st, a);
            break;
        }
        SKM_HIP(hipGetLastError());
    }
    return SKM_OK;
}

// ------------------------------------------------------------------ plan: rows by expert, stable ------
// The (token, slot) pairs n = t * k + j with 0 <= id < E, by expert and within an expert by n: a counting sort.
// Every wave owns a run of `chunk` consecutive pairs; 1: its histogram; 2: where each (expert, wave) run starts;
// 3: the waves walk their runs again, 64 pairs at a time; the rank of a pair among its equals of the 64 comes from
// ballots over the bits of the id, so the order never depends on who is first.
//   offsets[E + 1]  first row of an expert, [E] = number of rows
//   pair[n]         row -> t * k + j               pos[n]  t * k + j -> row, -1 without an expert
//   first[E + 1]    first 128-row tile of an expert (its rows from a tile's start), [E] = number of tiles
//   tiles[.][4]     per tile: expert, first row, rows (<= 128), 0
//   more[.][4]      the same with 16 or 256 rows a tile (more_rows; 0: none), more_count[1]
// Latency, not bytes: 32764 pairs over 32 experts 5.6 + 8.1 + 7.3 us for the three kernels (0.4 MB), 32 pairs over 64
// experts 4.8 us in one.

#define PLAN_WAVES 4

struct PlanArgs {
    const int32_t *ids;
    long n;
    int E;
    int chunk;              // pairs per wave, a multiple of 64
    int nw;                 // waves (= runs)
    int32_t *hist;          // [nw][E]: counts, then first rows
    int32_t *offsets, *pair, *pos, *first, *tiles, *more, *more_count;
    int more_rows;
};

__device__ __forceinline__ void plan_clear(int32_t *h, int E, int lane)
{
    for (int e = lane; e < E; e += 64) h[e] = 0;
}

__device__ void plan_count(const PlanArgs &a, int run, int lane, int32_t *h)
{
    const long lo = (long)run * a.chunk, hi = lo + a.chunk < a.n ? lo + a.chunk : a.n;
    for (long i = lo + lane; i < hi; i += 64) {
        const int e = a.ids[i];
        if (e >= 0 && e < a.E) atomicAdd(&h[e], 1);         // LDS, integers: the order does not matter
    }
}

// h[e]: the row of this run's next pair of expert e
__device__ void plan_place(const PlanArgs &a, int run, int lane, int32_t *h)
{
    const long lo = (long)run * a.chunk, hi = lo + a.chunk < a.n ? lo + a.chunk : a.n;
    int bits = 1;
    while ((1 << bits) < a.E) ++bits;
    int ahead = lo + lane < hi ? a.ids[lo + lane] : -1;
    for (long i0 = lo; i0 < hi; i0 += 64) {
        const long i = i0 + lane;
        const int e = ahead;
        ahead = i + 64 < hi ? a.ids[i + 64] : -1;           // the next 64, under this step's work
        const bool ok = e >= 0 && e < a.E;
        unsigned long long same = __ballot(ok);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long one = __ballot(ok && ((e >> b) & 1));
            same &= ((e >> b) & 1) ? one : ~one;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int row = -1;
        if (ok) row = h[e] + rank;
        wave_sync();                    // all lanes have read before the last of each kind writes
        if (ok && rank == __popcll(same) - 1) h[e] = row + 1;
        wave_sync();
        if (i < hi) a.pos[i] = row;
        if (ok) a.pair[row] = (int32_t)i;
    }
}

// exclusive prefix over the experts of v (one value per thread and round of blockDim), all threads call it
__device__ int plan_scan_block(int v, int *sh, int &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int s = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(s, m);
        if (lane >= m) s += o;
    }
    if (lane == 63) sh[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < waves; ++w) {
        if (w < wave) before += sh[w];
        total += sh[w];
    }
    __syncthreads();
    return before + s - v;
}

// From the histograms of all runs to the first row of every (run, expert), and the tile tables.  One workgroup of `threads`
// (a power of two); `part` has room for that many numbers.  Up to that many experts the threads of one expert share its runs
// and its tiles.
__device__ void plan_scan(const PlanArgs &a, int32_t *hist, int *sh, int *part, int threads)
{
    int share = 1;                          // threads of an expert
    while (share * 2 * a.E <= threads && share < a.nw) share *= 2;
    const int wide = threads / share;       // experts at a time
    const int s = threadIdx.x / wide, el = threadIdx.x - s * wide;
    const int per = (a.nw + share - 1) / share;
    const int mr = a.more_rows ? a.more_rows : 1;
    int rows0 = 0, tiles0 = 0, more0 = 0;
    for (int e0 = 0; e0 < a.E; e0 += wide) {
        const int e = e0 + el;
        const int r0 = s * per, r1 = r0 + per < a.nw ? r0 + per : a.nw;
        int own = 0;
        if (e < a.E)
            for (int r = r0; r < r1; ++r) own += hist[(long)r * a.E + e];
        part[threadIdx.x] = own;
        __syncthreads();
        int count = 0, before = 0;
        for (int o = 0; o < share; ++o) {
            const int v = part[o * wide + el];
            before += o < s ? v : 0;
            count += v;
        }
        // only the first thread of an expert counts in the prefix sums; the others learn its result
        const int mine = s == 0 ? count : 0;
        int nrows, ntiles, nmore;
        int off = rows0 + plan_scan_block(mine, sh, nrows);
        int t0 = tiles0 + plan_scan_block((mine + 127) / 128, sh, ntiles);
        int s0 = more0 + plan_scan_block((mine + mr - 1) / mr, sh, nmore);
        rows0 += nrows;
        tiles0 += ntiles;
        more0 += nmore;
        if (share > 1) {
            if (s == 0) part[el] = off;
            __syncthreads();
            off = part[el];
            __syncthreads();
            if (s == 0) part[el] = t0;
            __syncthreads();
            t0 = part[el];
            __syncthreads();
            if (s == 0) part[el] = s0;
            __syncthreads();
            s0 = part[el];
        }
        __syncthreads();
        if (e < a.E) {
            if (s == 0) {
                a.offsets[e] = off;
                a.first[e] = t0;
            }
            int at = off + before;
            for (int r = r0; r < r1; ++r) {
                const int c = hist[(long)r * a.E + e];
                hist[(long)r * a.E + e] = at;
                at += c;
            }
            for (int t = s; t * 128 < count; t += share)
                *reinterpret_cast<int4 *>(a.tiles + (long)(t0 + t) * 4) =
                    make_int4(e, off + t * 128, count - t * 128 < 128 ? count - t * 128 : 128, 0);
            if (a.more_rows)
                for (int t = s; t * mr < count; t += share)
                    *reinterpret_cast<int4 *>(a.more + (long)(s0 + t) * 4) =
                        make_int4(e, off + t * mr, count - t * mr < mr ? count - t * mr : mr, 0);
        }
    }
    if (threadIdx.x == 0) {
        a.offsets[a.E] = rows0;
        a.first[a.E] = tiles0;
        if (a.more_rows) a.more_count[0] = more0;
    }
}

// few pairs: everything in one workgroup, the histograms in LDS (nw = PLAN_WAVES)
__global__ __launch_bounds__(64 * PLAN_WAVES) void k_plan_one(PlanArgs a)
{
    extern __shared__ int32_t lds[];
    __shared__ int sh[PLAN_WAVES], part[64 * PLAN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t *h = lds + (long)wave * a.E;
    plan_clear(h, a.E, lane);
    __syncthreads();
    plan_count(a, wave, lane, h);
    __syncthreads();
    plan_scan(a, lds, sh, part, 64 * PLAN_WAVES);
    __syncthreads();
    plan_place(a, wave, lane, h);
}

__global__ __launch_bounds__(64) void k_plan_count(PlanArgs a)
{
    extern __shared__ int32_t lds[];
    plan_clear(lds, a.E, threadIdx.x);
    __syncthreads();
    plan_count(a, blockIdx.x, threadIdx.x, lds);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += 64) a.hist[(long)blockIdx.x * a.E + e] = lds[e];
}

__global__ __launch_bounds__(1024) void k_plan_scan(PlanArgs a)
{
    __shared__ int sh[16], part[1024];
    plan_scan(a, a.hist, sh, part, 1024);
}

__global__ __launch_bounds__(64) void k_plan_place(PlanArgs a)
{
    extern __shared__ int32_t lds[];
    for (int e = threadIdx.x; e < a.E; e += 64) lds[e] = a.hist[(long)blockIdx.x * a.E + e];
    __syncthreads();
    plan_place(a, blockIdx.x, threadIdx.x, lds);
}

// Few enough for one workgroup: 4 runs of up to 1024 pairs, 32 KB of histograms.  Beyond that a workgroup walks its pairs
// longer than three launches take (32764 pairs of 32 experts in 16 waves: 48 us against 19).
static bool plan_is_one(long n, int E) { return n <= 4096 && E <= 2048; }

static int plan_runs(long n, int E, int *chunk)
{
    if (plan_is_one(n, E)) {
        *chunk = (int)((n + PLAN_WAVES - 1) / PLAN_WAVES + 63) / 64 * 64;
        return PLAN_WAVES;
    }
    long c = (n + 511) / 512;               // at most 512 runs
    if (c < 512) c = 512;
    c = (c + 63) / 64 * 64;
    *chunk = (int)c;
    return (int)((n + c - 1) / c);
}

extern "C" size_t skm_route_plan_workspace_bytes(long n, int E)
{
    if (n <= 0 || E <= 0 || plan_is_one(n, E)) return 0;
    int chunk;
    return (size_t)plan_runs(n, E, &chunk) * (size_t)E * 4;
}

extern "C" long skm_route_plan_tiles(long n, int E, int rows)
{
    if (n < 0 || E < 1 || rows < 1) return 0;
    return n / rows + (n < E ? n : E);      // every expert adds less than one tile to its full ones
}

extern "C" int skm_route_plan(void *ctx_, const int32_t *ids, long n, int E, int32_t *offsets, int32_t *pair,
                              int32_t *pos, int32_t *first, int32_t *tiles, int more_rows, int32_t *more_tiles,
                              int32_t *more_count, void *ws, size_t ws_bytes, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && n >= 0 && E >= 1 && offsets && first && (n == 0 || (ids && pair && pos && tiles)) &&
                    (!more_rows || ((more_rows == 16 || more_rows == 256) && more_count && (n == 0 || more_tiles))) &&
                    (((uintptr_t)tiles | (uintptr_t)more_tiles) & 15) == 0,
                "skm_route_plan: bad argument");
    if (E > ROUTE_MAX_E || n > 0x3FFFFFFF) {
        skm_set_error("skm_route_plan: built for %d experts and 2^30 - 1 pairs", ROUTE_MAX_E);
        return SKM_ERR_UNSUPPORTED;
    }
    if (ws_bytes < skm_route_plan_workspace_bytes(n, E) || (skm_route_plan_workspace_bytes(n, E) && !ws)) {
        skm_set_error("skm_route_plan: workspace too small");
        return SKM_ERR_WORKSPACE;
    }
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    PlanArgs a{ids, n, E, 0, 0, static_cast<int32_t *>(ws), offsets, pair, pos, first, tiles, more_tiles, more_count, more_rows};
    a.nw = plan_runs(n, E, &a.chunk);
    SkmProfScope ps(ctx, "k_plan", st);
    if (plan_is_one(n, E)) {
        hipLaunchKernelGGL(k_plan_one, dim3(1), dim3(64 * PLAN_WAVES), (size_t)PLAN_WAVES * E * 4, st, a);
    } else {                                // no pairs, no runs: only the scan, which writes the tables' zeros
        if (a.nw) hipLaunchKernelGGL(k_plan_count, dim3((unsigned)a.nw), dim3(64), (size_t)E * 4, st, a);
        hipLaunchKernelGGL(k_plan_scan, dim3(1), dim3(1024), 0, st, a);
        if (a.nw) hipLaunchKernelGGL(k_plan_place, dim3((unsigned)a.nw), dim3(64), (size_t)E * 4, st, a);
    }
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}

// ------------------------------------------------------------------ weighted sum of the experts' rows ------
struct CombineArgs {
    const void *rows;       // [.][N]
    const int32_t *pos;     // [T][k]
    const float *w;         // [T][k]
    long T;
    int k, N;
    void *out;              // [T][N]
    const void *dout;
    float *dw;
    long pair0;             // first pair of a launch (gradient)
};

// out[t] = sum_j w[t][j] rows[pos[t][j]], in the order of j, float32.  An empty place adds w * 0: nothing, or the NaN
// that a row without a choice carries in its weights.
// Bound by memory: 8191 tokens, 4 places, 2048 columns bf16 27.5 us, 168 MB at 6.1 TB/s (part of the rows is still in the
// cache).  A workgroup has one token (or, of short rows, several): its places and weights are the same for all lanes of a row, four
// rows are in flight.
template <typename TR, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_route_combine(CombineArgs a, int per, int tokens)
{
    typedef TR vr __attribute__((ext_vector_type(VEC)));
    typedef TO vo __attribute__((ext_vector_type(VEC)));
    const int sub = tokens > 1 ? threadIdx.x / per : 0;         // per: threads of a row, where a workgroup has several
    const long t = (long)blockIdx.x * tokens + sub;
    const int c = (tokens > 1 ? (int)threadIdx.x - sub * per : (int)(blockIdx.y * 256 + threadIdx.x)) * VEC;
    if (t >= a.T || sub >= tokens || c >= a.N) return;
    const int32_t *pos = a.pos + t * a.k;
    const float *w = a.w + t * a.k;
    const TR *rows = static_cast<const TR *>(a.rows) + c;
    TO *out = static_cast<TO *>(a.out) + t * a.N + c;
    if (c + VEC > a.N) {                    // the end of a row
        for (int q = 0; c + q < a.N; ++q) {
            float s = 0.f;
            for (int j = 0; j < a.k; ++j) s += w[j] * (pos[j] >= 0 ? (float)rows[(long)pos[j] * a.N + q] : 0.f);
            out[q] = (TO)s;
        }
        return;
    }
    float s[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) s[q] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += 4) {
        vr v[4];
        float f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = j0 + u < a.k ? pos[j0 + u] : -1;
            f[u] = j0 + u < a.k ? w[j0 + u] : 0.f;
#pragma unroll
            for (int q = 0; q < VEC; ++q) v[u][q] = (TR)0.f;
            if (p >= 0) v[u] = load_any<vr>(rows + (long)p * a.N);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < VEC; ++q) s[q] += f[u] * (float)v[u][q];
    }
    vo o;
#pragma unroll
    for (int q = 0; q < VEC; ++q) o[q] = (TO)s[q];
    store_any(out, o);
}

// dw[t][j] = <dout[t], rows[pos[t][j]]>: one wave per pair.  Bound by memory: 8192 tokens, 2 places, 2048 columns of float32
// rows 32 us, 168 MB at 5.2 TB/s.
template <typename TR, typename TO>
__global__ __launch_bounds__(256) void k_route_combine_backward(CombineArgs a)
{
    constexpr int VEC = 4;
    typedef TR vr __attribute__((ext_vector_type(VEC)));
    typedef TO vo __attribute__((ext_vector_type(VEC)));
    const int lane = threadIdx.x & 63;
    const long i = a.pair0 + (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.T * a.k) return;
    const int p = a.pos[i];
    float s = 0.f;
    if (p >= 0) {
        const TR *r = static_cast<const TR *>(a.rows) + (long)p * a.N;
        const TO *d = static_cast<const TO *>(a.dout) + (i / a.k) * a.N;
        float part[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) part[q] = 0.f;
        const int whole = a.N / VEC * VEC;
#pragma unroll 4
        for (int c = lane * VEC; c < whole; c += 64 * VEC) {
            const vr x = load_any<vr>(r + c);
            const vo y = load_any<vo>(d + c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) part[q] += (float)x[q] * (float)y[q];
        }
        if (whole + lane < a.N) s = (float)r[whole + lane] * (float)d[whole + lane];
#pragma unroll
        for (int q = 0; q < VEC; ++q) s += part[q];
        s = wave_sum(s);
    }
    if (lane == 0) a.dw[i] = s;
}

template <typename TR, typename TO>
static void combine_launch(const CombineArgs &a, hipStream_t st)
{
    // 16 bytes of the narrower type a thread
    constexpr int V = sizeof(TR) == 4 && sizeof(TO) == 4 ? 4 : 8;
    const int per = (a.N + V - 1) / V, tokens = per <= 128 ? 256 / per : 1;
    const long most = SKM_MAX_GROUPS * tokens;
    for (long t = 0; t < a.T; t += most) {
        CombineArgs b = a;
        b.pos += t * a.k;
        b.w += t * a.k;
        b.out = static_cast<TO *>(a.out) + t * a.N;
        b.T = a.T - t < most ? a.T - t : most;
        const dim3 grid((unsigned)((b.T + tokens - 1) / tokens), tokens > 1 ? 1u : (unsigned)((per + 255) / 256));
        hipLaunchKernelGGL((k_route_combine<TR, TO, V>), grid, dim3(256), 0, st, b, per, tokens);
    }
}

template <typename TR, typename TO>
static void combine_back_launch(const CombineArgs &a, hipStream_t st)
{
    const long pairs = a.T * a.k;
    CombineArgs b = a;
    for (b.pair0 = 0; b.pair0 < pairs; b.pair0 += SKM_MAX_GROUPS * 4) {
        const long groups = (pairs - b.pair0 + 3) / 4;
        hipLaunchKernelGGL((k_route_combine_backward<TR, TO>), dim3((unsigned)(groups < SKM_MAX_GROUPS ? groups : SKM_MAX_GROUPS)),
                           dim3(256), 0, st, b);
    }
}

#define COMBINE_TYPES(F, TR_CODE, TO_CODE)                                                                       \
    switch ((TR_CODE) * 4 + (TO_CODE)) {                                                                         \
    case SKM_DT_F32 * 4 + SKM_DT_F32: F<float, float>(a, st); break;                                             \
    case SKM_DT_F32 * 4 + SKM_DT_BF16: F<float, bf16_t>(a, st); break;                                           \
    case SKM_DT_F32 * 4 + SKM_DT_F16: F<float, f16_t>(a, st); break;                                             \
    case SKM_DT_BF16 * 4 + SKM_DT_F32: F<bf16_t, float>(a, st); break;                                           \
    case SKM_DT_BF16 * 4 + SKM_DT_BF16: F<bf16_t, bf16_t>(a, st); break;                                         \
    case SKM_DT_F16 * 4 + SKM_DT_F32: F<f16_t, float>(a, st); break;                                             \
    case SKM_DT_F16 * 4 + SKM_DT_F16: F<f16_t, f16_t>(a, st); break;                                             \
    default: skm_set_error("rows of type %d and result of type %d do not go together", (int)(TR_CODE), (int)(TO_CODE)); \
             return SKM_ERR_UNSUPPORTED;                                                                         \
    }

extern "C" int skm_route_combine(void *ctx_, const void *rows, int rows_dtype, const int32_t *pos, const float *weights,
                                 long T, int k, int N, void *out, int out_dtype, void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && T >= 0 && k >= 1 && N >= 1 && (T == 0 || (rows && pos && weights && out)),
                "skm_route_combine: bad argument");
    SKM_REQUIRE(T <= 0x7FFFFFFF && (N + 255) / 256 <= 65535, "skm_route_combine: too many elements");
    if (T == 0) return SKM_OK;
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_route_combine", st);
    const CombineArgs a{rows, pos, weights, T, k, N, out, nullptr, nullptr, 0};
    COMBINE_TYPES(combine_launch, rows_dtype, out_dtype)
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}

extern "C" int skm_route_combine_backward(void *ctx_, const void *rows, int rows_dtype, const int32_t *pos,
                                          const void *dout, int dout_dtype, long T, int k, int N, float *dweights,
                                          void *stream)
{
    SkmCtx *ctx = static_cast<SkmCtx *>(ctx_);
    SKM_REQUIRE(ctx && T >= 0 && k >= 1 && N >= 1 && (T == 0 || (rows && pos && dout && dweights)),
                "skm_route_combine_backward: bad argument");
    SKM_REQUIRE(T * k < 0x7FFFFFFFL * 4, "skm_route_combine_backward: too many pairs");
    if (T == 0) return SKM_OK;
    SkmDeviceGuard guard(ctx);
    hipStream_t st = (hipStream_t)stream;
    SkmProfScope ps(ctx, "k_route_combine_backward", st);
    const CombineArgs a{rows, pos, nullptr, T, k, N, nullptr, dout, dweights, 0};
    COMBINE_TYPES(combine_back_launch, rows_dtype, dout_dtype)
    SKM_HIP(hipGetLastError());
    return SKM_OK;
}
