// select.hip - routing to experts by a rule, from router logits.
//
//   s_e = softmax(x)_e or 1 / (1 + e^-x_e);  c_e = s_e + bias_e  (the choice values)
//   a group's value is the sum of its `group_top` largest c; the best n_group_used groups stay; of their experts the k largest
//   c are chosen (equal values: the lowest id), in that order;  w = s / max(sum of the chosen s, 2^-14) * scale
//
// Scores and choice values are those of 64 bits: two experts a 32-bit rounding apart would swap places with the compiler's
// choice of instructions. But few are that close. So a wavefront first scores its tokens in 32 bits and takes the k largest and
// a few more (choose_fast). Only these candidates' scores are computed in 64 bits, which gives their order and weights. The
// 32-bit scores settle the rest where the last group that stays is further from the next, and the k-th candidate from all that
// are none, than they can be off; a wavefront with a token where they are not does all of it in 64 bits (choose_exact). The
// chosen weights are rounded once, to fp32.
//
// 16 lanes (a DPP row) take a token, so a wavefront takes four, and lane l the experts l, l + 16, ..: a row's maximum is four
// DPP steps. A 32-bit choice value carries its expert in its lowest 8 bits, so that the maximum says whose it is; 64-bit ones keep
// all their bits, and a second maximum finds the lowest id among equal ones. In each of the k rounds the lane that owned the
// maximum takes it out of its values in LDS and finds its next one; the others keep theirs.
//
// Bound by vector instructions, 1445 a wavefront (the units are busy for 74% of the time), not by the 65 MB of 60000 tokens over
// 256 experts, which take 49 us with sigmoid scores, bias and 4 of 8 groups on MI355X; 512 such tokens take 8 us, or 15 where
// one wavefront does it over in 64 bits; one token over 128 experts 3.7. All in 64 bits (a softmax with a bias): 60000 tokens over
// 128 experts 29 us a call, where the same without a bias take 15.
#include <cfloat>
#include <type_traits>

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

constexpr int kSelLanes = 16;                 // per token
constexpr int kSelTokens = kWave / kSelLanes; // per wavefront

__device__ __forceinline__ double value_of(float x) { return x != x ? -INFINITY : (double) fminf(x, FLT_MAX); }

// e^z for |z| <= 800 to 1e-15 of its value: 2^n e^r with |r| <= ln 2 / 2, e^r by its series to r^12 (what is left out is below
// 2e-16 of it).
__device__ __forceinline__ double exp_of(double z) {
    const double n = rint(z * 1.4426950408889634);
    double r = fma(n, -0.6931471803691238, z); // ln 2 in two parts, the first of 33 bits (Cody and Waite)
    r = fma(n, -1.9082149292705877e-10, r);
    double p = 1.0 / 479001600;
    p = fma(p, r, 1.0 / 39916800);
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int) n);
}
// 1 / d for 1 <= d < 2e308: the hardware's estimate and two Newton steps.
__device__ __forceinline__ double inverse(double d) {
    double y = __builtin_amdgcn_rcp(d);
    y = fma(fma(-d, y, 1.0), y, y);
    return fma(fma(-d, y, 1.0), y, y);
}
__device__ __forceinline__ double sigmoid(double x) { return inverse(1.0 + exp_of(fmin(fmax(-x, -800.0), 709.5))); }

// Over the 16 lanes of a DPP row; every lane gets the result.
__device__ __forceinline__ double row_max(double v) {
    v = fmax(v, dpp_d<0xB1>(v));  // quad_perm [1,0,3,2]
    v = fmax(v, dpp_d<0x4E>(v));  // quad_perm [2,3,0,1]
    v = fmax(v, dpp_d<0x141>(v)); // row_half_mirror
    return fmax(v, dpp_d<0x140>(v)); // row_mirror
}
__device__ __forceinline__ double row_sum(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    return v + dpp_d<0x140>(v);
}

__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0xB1, 0xF, 0xF, false));
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x4E, 0xF, 0xF, false));
    v = max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x141, 0xF, 0xF, false));
    return max(v, (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x140, 0xF, 0xF, false));
}
__device__ __forceinline__ unsigned row_sum(unsigned v) {
    v += (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0xB1, 0xF, 0xF, false);
    v += (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x4E, 0xF, 0xF, false);
    v += (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x141, 0xF, 0xF, false);
    return v + (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, 0x140, 0xF, 0xF, false);
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    return fmaxf(v, dpp_f<0x140>(v));
}
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_f<0xB1>(v);
    v += dpp_f<0x4E>(v);
    v += dpp_f<0x141>(v);
    return v + dpp_f<0x140>(v);
}

// A choice value as it is ordered: -inf and NaN become a finite value below all others, so that they stay above what may not be
// chosen at all (-inf here).
__device__ __forceinline__ double ordered(double c) { return fmax(c, -0x1p1000); }

// A 32-bit choice value with its expert, as a whole number: the order-preserving key of c with the expert in place of its lowest 8
// bits; 0 is below all of them. value_below is at most 2^-14 |c| below c, and never above it.
__device__ __forceinline__ unsigned tagged(float c, int e) {
    const unsigned u = __float_as_uint(c), key = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (key & ~255u) | (255u - (unsigned) e);
}
__device__ __forceinline__ float value_below(unsigned t) {
    const unsigned key = t & ~255u;
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// How far a 32-bit choice value near v can be from the 64-bit one. A sigmoid is off by less than 3e-7: its argument's rounding
// |x| s (1 - s) 2^-23 < 3e-8, the exponential s (1 - s) 2^-23, 1 + t 2^-24, the inverse 2^-23 of s; a softmax score by less
// than that too (its sum by 2^-23 and its exponentials' errors); the sum with the bias by 2^-24 of itself. The rest, 2e-7 and
// 4e-7 |v|, covers the roundings of a group's sum and of the comparisons.
__device__ __forceinline__ float margin(float v) { return 5e-7f * (1.0f + fabsf(v)); }
constexpr int kSelMore = 3; // candidates beyond the k largest

// What a wavefront knows of its lane's token.
struct Lane {
    const float *x;
    int l;        // lane of the token
    double *vals; // LDS: the token's choice values, lane by lane, in either width
    double *s_g;  // with groups: their values (in 32 bits margins too), and which of them stay
    uint32_t *s_keep;
    int *s_id; // the chosen experts
};

// LDS of one wavefront: the choice values of each token, lane by lane, with groups their values and which of them stay, and the
// chosen ids.
template <int V>
__host__ __device__ constexpr size_t select_lds(int groups) {
    return kSelTokens * ((size_t) kSelLanes * (V + 2) * 8 + (size_t) groups * 8 + (groups ? 32 : 0) + kMaxK * 4);
}
// From one lane's choice values to the next's: two 64-bit or four 32-bit ones more than it has, against bank conflicts.
template <int V, typename T>
__host__ __device__ constexpr int stride_of() { return sizeof(T) == 8 ? V + 2 : V + 4; }
// Orders a wavefront's LDS writes before its later reads by other lanes (they execute in order; the compiler has to as well).
__device__ __forceinline__ void lds_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The two largest choice values of group g of a token, from LDS; lanes_per lanes (a power of two) take a group together.
template <int V, typename T>
__device__ __forceinline__ void best_two(const T *vals, int g, int per, int part, int lanes_per, T &a, T &b) {
    a = b = -INFINITY;
#pragma unroll 4
    for (int j = part; j < per; j += lanes_per) {
        const int e = g * per + j;
        const T v = vals[(e % kSelLanes) * stride_of<V, T>() + e / kSelLanes];
        const T low = a < v ? a : v;
        b = b < low ? low : b;
        a = a < v ? v : a;
    }
    auto join = [&](T oa, T ob) {
        const T low = a < oa ? a : oa, high = b < ob ? ob : b;
        a = a < oa ? oa : a;
        b = low < high ? high : low;
    };
    auto dpp = [](T v, auto ctrl) {
        if constexpr (sizeof(T) == 8) return dpp_d<decltype(ctrl)::value>(v);
        else return dpp_f<decltype(ctrl)::value>(v);
    };
    if (lanes_per >= 2) join(dpp(a, std::integral_constant<int, 0xB1>()), dpp(b, std::integral_constant<int, 0xB1>()));
    if (lanes_per >= 4) join(dpp(a, std::integral_constant<int, 0x4E>()), dpp(b, std::integral_constant<int, 0x4E>()));
    if (lanes_per >= 8) join(dpp(a, std::integral_constant<int, 0x141>()), dpp(b, std::integral_constant<int, 0x141>()));
    if (lanes_per >= 16) join(dpp(a, std::integral_constant<int, 0x140>()), dpp(b, std::integral_constant<int, 0x140>()));
}
// Which of the lane's experts may not be chosen (bit i: expert l + 16 i), from the choice values c. stays(values, g): whether
// group g stays, 1 or 0, or -1 where that is not settled; settled then becomes false. Behind 32-bit values stand how far they can be
// off: the margins of their summands, which may be far larger than their sum.
template <int V, typename T, typename F>
__device__ __forceinline__ unsigned left_out(const SelectParams &P, const Lane &L, const T (&c)[V], bool &settled, F stays) {
    const int per = P.E / P.n_group;
    const unsigned inv = (65536u + per - 1) / per; // e / per = e * inv >> 16 for e < 256
    T *const vals = reinterpret_cast<T *>(L.vals), *const values = reinterpret_cast<T *>(L.s_g);
    lds_in_order();
#pragma unroll
    for (int i = 0; i < V; i++) vals[L.l * stride_of<V, T>() + i] = c[i];
    if (L.l < 8) L.s_keep[L.l] = 0;
    lds_in_order();
    int lanes_per = 1;
    while (lanes_per * 2 * P.n_group <= kSelLanes) lanes_per *= 2;
    const int at_once = kSelLanes / lanes_per;
    for (int g0 = 0; g0 < P.n_group; g0 += at_once) { // all lanes stay in step for the DPP joins
        const int g = g0 + L.l / lanes_per;
        T a, b;
        best_two<V>(vals, min(g, P.n_group - 1), per, L.l % lanes_per, lanes_per, a, b);
        const T v = P.group_top == 2 ? a + b : a;
        if (g < P.n_group && L.l % lanes_per == 0) {
            values[g] = v != v ? (T) -INFINITY : v;
            if constexpr (sizeof(T) == 4) values[P.n_group + g] = P.group_top == 2 ? margin(a) + margin(b) : margin(a);
        }
    }
    lds_in_order();
    for (int g = L.l; g < P.n_group; g += kSelLanes) {
        const int s = stays(values, g);
        if (s > 0) atomicOr(&L.s_keep[g / 32], 1u << (g % 32));
        settled = settled && s >= 0;
    }
    lds_in_order();
    unsigned out = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const unsigned g = (L.l + kSelLanes * i) * inv >> 16;
        out |= (~L.s_keep[g / 32] >> (g % 32) & 1u) << i;
    }
    return out;
}

// The k largest of the tagged values t (the lanes' own, 0 for one that may not be chosen), into s_id; returns the next.
template <int V>
__device__ __forceinline__ unsigned take_largest(const Lane &L, const unsigned (&t)[V], int k) {
    unsigned *const mine = reinterpret_cast<unsigned *>(L.vals) + L.l * stride_of<V, unsigned>();
    lds_in_order();
    unsigned best = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        mine[i] = t[i];
        best = best < t[i] ? t[i] : best;
    }
    for (int j = 0; j < k; j++) {
        // (where groups are not settled there may be none left: expert 0 stands in, and choose_exact does it over)
        const unsigned top = row_max(best);
        const int e = top == 0 ? 0 : (int) (255u - (top & 255u));
        if (L.l == e % kSelLanes) {
            L.s_id[j] = e;
            mine[e / kSelLanes] = 0;
            unsigned v[V];
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = mine[i];
            best = v[0];
#pragma unroll
            for (int i = 1; i < V; i++) best = best < v[i] ? v[i] : best;
        }
    }
    lds_in_order();
    return row_max(best);
}

// The k largest of the 64-bit values c (ordered(); -inf for one that may not be chosen), of equal ones the lowest id first, into
// s_id in that order. The ids stand apart from the values: in their lowest 8 bits they would make values 2^-45 of themselves apart
// equal, as saturated sigmoids are.
template <int V>
__device__ __forceinline__ void take_largest(const Lane &L, const double (&c)[V], int k) {
    double *const mine = L.vals + L.l * stride_of<V, double>();
    lds_in_order();
    double v[V], best = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        mine[i] = v[i] = c[i];
        best = fmax(best, c[i]);
    }
    for (int j = 0; j < k; j++) {
        const double top = row_max(best);
        int at = V; // the lane's first value that is the largest
#pragma unroll
        for (int i = V - 1; i >= 0; i--) at = v[i] == top ? i : at;
        const int e = 255 - (int) row_max(at < V ? 255u - (unsigned) (L.l + kSelLanes * at) : 0u);
        if (L.l == e % kSelLanes) {
            L.s_id[j] = e;
            mine[e / kSelLanes] = -INFINITY;
            best = -INFINITY;
#pragma unroll
            for (int i = 0; i < V; i++) best = fmax(best, v[i] = mine[i]);
        }
    }
    lds_in_order();
}

// The lane's logits and biases; -inf past the last expert.
template <int V>
__device__ __forceinline__ void load_lane(const SelectParams &P, const Lane &L, float (&xv)[V], float (&bv)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        xv[i] = L.x[min(L.l + kSelLanes * i, P.E - 1)];
        bv[i] = 0.0f;
    }
    if (P.bias) {
#pragma unroll
        for (int i = 0; i < V; i++) bv[i] = P.bias[min(L.l + kSelLanes * i, P.E - 1)];
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (L.l + kSelLanes * i >= P.E) xv[i] = -INFINITY;
}

// All in 64 bits: s_id gets the chosen experts in order. A softmax's scores are e^(x - top) scale.
template <int V, bool SIGMOID, bool GROUPS>
__device__ __forceinline__ void choose_exact(const SelectParams &P, const Lane &L, double &top, double &scale) {
    float xv[V], bv[V];
    load_lane(P, L, xv, bv);
    double c[V];
    top = 0.0;
    scale = 1.0;
    if constexpr (SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = sigmoid(value_of(xv[i]));
    } else {
        top = value_of(xv[0]);
#pragma unroll
        for (int i = 1; i < V; i++) top = fmax(top, value_of(xv[i]));
        top = row_max(top);
        if (top == -INFINITY) top = 0.0;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            c[i] = exp_of(fmax(value_of(xv[i]) - top, -800.0));
            sum += c[i];
        }
        sum = row_sum(sum);
        scale = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) c[i] *= scale;
    }
    unsigned out = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        c[i] += (double) bv[i];
        if (c[i] != c[i]) c[i] = -INFINITY;
        out |= (L.l + kSelLanes * i < P.E ? 0u : 1u) << i;
    }
    if constexpr (GROUPS) {
        bool settled = true;
        out |= left_out<V>(P, L, c, settled, [&](const double *v, int g) {
            const double mine = v[g];
            int rank = 0;
            for (int j = 0; j < P.n_group; j++) rank += v[j] > mine || (v[j] == mine && j < g);
            return rank < P.n_group_used ? 1 : 0;
        });
    }
#pragma unroll
    for (int i = 0; i < V; i++) c[i] = out >> i & 1u ? -INFINITY : ordered(c[i]);
    take_largest<V>(L, c, P.k);
}

// In 32 bits: s_id gets the n largest, in no order that counts; returns whether what stays by groups is settled, and a bound of
// all choice values that are none of the n (in units of 1 / sum for a softmax with groups, of logits for one without). For
// sigmoid scores, and for softmax ones without bias that are renormalised (the weights then need no exact sum over all).
struct Fast {
    bool settled;
    float rest, most, sum; // most, sum: a softmax's largest logit and sum of e^(x - most)
};
template <int V, bool SIGMOID, bool GROUPS>
__device__ __forceinline__ Fast choose_fast(const SelectParams &P, const Lane &L, int n) {
    float xv[V], bv[V];
    load_lane(P, L, xv, bv);
    constexpr float kLog2e = 1.44269504088896341f;
    float c[V], most = 0.0f, sum = 1.0f;
    bool settled = true;
    if constexpr (SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(xv[i] * -kLog2e)) + bv[i];
    } else {
        most = xv[0];
#pragma unroll
        for (int i = 1; i < V; i++) most = fmaxf(most, xv[i]);
        most = row_max(most);
        settled = fabsf(most) < 1e30f;
        if constexpr (GROUPS) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) {
                c[i] = __builtin_amdgcn_exp2f((xv[i] - most) * kLog2e);
                sum += c[i];
            }
            sum = row_sum(sum);
            const float inv = 1.0f / sum;
#pragma unroll
            for (int i = 0; i < V; i++) c[i] *= inv;
        } else {
            // the order of the logits is that of the scores
#pragma unroll
            for (int i = 0; i < V; i++) c[i] = xv[i];
        }
    }
    unsigned out = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const bool in = L.l + kSelLanes * i < P.E;
        out |= (in ? 0u : 1u) << i;
        settled = settled && (c[i] < 1e30f || !in); // no NaN, nothing too large for the margins
    }
    if constexpr (GROUPS) {
        out |= left_out<V>(P, L, c, settled, [&](const float *v, int g) {
            const float mine = v[g], mine_m = v[P.n_group + g];
            int above = 0, near = 0;
            for (int j = 0; j < P.n_group; j++) {
                const float m = mine_m + v[P.n_group + j];
                above += v[j] > mine + m;
                near += !(v[j] < mine - m);
            }
            return near <= P.n_group_used ? 1 : above >= P.n_group_used ? 0 : -1; // `near` counts the group itself
        });
    }
    unsigned t[V];
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = out >> i & 1u ? 0u : tagged(c[i], L.l + kSelLanes * i);
    const unsigned next = take_largest<V>(L, t, n);
    const float v = value_below(next);
    return {settled, next == 0 ? -INFINITY : v + fabsf(v) * 0x1p-14f + 2.0f * margin(v), most, sum};
}

// The candidates' scores and their ranks by 64-bit choice value; lane l's are s_id[l], s_id[l + 16], ..
template <int MOST>
struct Ranked {
    double s[MOST], sum; // sum: of the k best of the token
    int rank[MOST];
};
template <bool SIGMOID, int MOST>
__device__ __forceinline__ Ranked<MOST> rank_candidates(const SelectParams &P, const Lane &L, int n, double top, double scale) {
    Ranked<MOST> r;
    lds_in_order();
#pragma unroll
    for (int q = 0; q < MOST; q++) {
        const int j = L.l + kSelLanes * q;
        if (j < n) {
            const int e = L.s_id[j];
            const double v = value_of(L.x[e]);
            if constexpr (SIGMOID) r.s[q] = sigmoid(v);
            else r.s[q] = exp_of(fmax(v - top, -800.0)) * scale;
            L.vals[j] = ordered(P.bias ? r.s[q] + (double) P.bias[e] : r.s[q]);
        }
        if (kSelLanes * (q + 1) >= n) break;
    }
    lds_in_order();
    unsigned ranks = 0;
#pragma unroll
    for (int q = 0; q < MOST; q++) {
        const int j = L.l + kSelLanes * q;
        if (j < n) {
            r.rank[q] = 0;
            const double mine = L.vals[j];
            for (int i = 0; i < n; i++) r.rank[q] += L.vals[i] > mine;
            ranks += (unsigned) r.rank[q];
        }
        if (kSelLanes * (q + 1) >= n) break;
    }
    // of equal values the lowest id is first; there are some where the ranks add up to less than 0 + 1 + .. + n - 1 (comparing ids
    // with every value costs 60000 tokens 5 us)
    if (__any(row_sum(ranks) != (unsigned) (n * (n - 1) / 2))) {
#pragma unroll
        for (int q = 0; q < MOST; q++) {
            const int j = L.l + kSelLanes * q;
            if (j < n) {
                const double mine = L.vals[j];
                const int e = L.s_id[j];
                for (int i = 0; i < n; i++) r.rank[q] += L.vals[i] == mine && L.s_id[i] < e;
            }
            if (kSelLanes * (q + 1) >= n) break;
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < MOST; q++) {
        if (L.l + kSelLanes * q < n && r.rank[q] < P.k) sum += r.s[q];
        if (kSelLanes * (q + 1) >= n) break;
    }
    r.sum = row_sum(sum);
    return r;
}
template <int MOST>
__device__ __forceinline__ void write_out(const SelectParams &P, const Lane &L, const Ranked<MOST> &r, int64_t t, int n, double f) {
    f *= (double) P.scale;
#pragma unroll
    for (int q = 0; q < MOST; q++) {
        const int j = L.l + kSelLanes * q;
        if (j < n && r.rank[q] < P.k) {
            P.ids[t * P.k + r.rank[q]] = L.s_id[j];
            P.weights[t * P.k + r.rank[q]] = (float) (r.s[q] * f);
        }
        if (kSelLanes * (q + 1) >= n) break;
    }
}

// V: experts per lane, 16 V >= E
template <int V, bool SIGMOID, bool GROUPS>
__global__ __launch_bounds__(kWave) void select_kernel(SelectParams P) {
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int kMost = kMaxK / kSelLanes; // candidates of a lane
    const int l = threadIdx.x % kSelLanes, row = threadIdx.x / kSelLanes, groups = GROUPS ? P.n_group : 0;
    Lane L;
    L.l = l;
    unsigned char *at = lds;
    L.vals = reinterpret_cast<double *>(at) + row * kSelLanes * (V + 2);
    at += kSelTokens * kSelLanes * (V + 2) * 8;
    L.s_g = reinterpret_cast<double *>(at) + row * groups;
    at += (size_t) kSelTokens * groups * 8;
    L.s_keep = reinterpret_cast<uint32_t *>(at) + row * 8;
    at += GROUPS ? kSelTokens * 32 : 0;
    L.s_id = reinterpret_cast<int *>(at) + row * kMaxK;
    const int64_t first = (int64_t) blockIdx.x * kSelTokens, t = min(first + row, (int64_t) P.T - 1);
    const bool live = first + row < P.T; // rows past the last token compute it again and store nothing
    L.x = P.logits + t * P.ld;

    Ranked<kMost> r;
    if (SIGMOID || (P.renorm && !P.bias)) {
        const int n = min(min(P.k + kSelMore, kMaxK), GROUPS ? P.n_group_used * (P.E / P.n_group) : P.E);
        const Fast F = choose_fast<V, SIGMOID, GROUPS>(P, L, n);
        r = rank_candidates<SIGMOID, kMost>(P, L, n, (double) F.most, 1.0);
        bool settled = F.settled;
#pragma unroll
        for (int q = 0; q < kMost; q++) {
            const int j = l + kSelLanes * q;
            if (j < n && r.rank[q] == P.k - 1 && n < P.E) {
                // the last one that stays, against all that are no candidates
                float v = SIGMOID ? (float) L.vals[j] : GROUPS ? (float) r.s[q] * (1.0f / F.sum) : L.x[L.s_id[j]];
                settled = settled && v - margin(v) > F.rest;
                // of a softmax also: not so small that 64 bits make it the same as others
                if constexpr (!SIGMOID) settled = settled && r.s[q] > 1e-290;
            }
            if (kSelLanes * (q + 1) >= n) break;
        }
        // the scores' sum is held above 2^-14, which a softmax's best k without groups always are (k / E at least)
        if constexpr (!SIGMOID && GROUPS) settled = settled && r.sum > (double) (0x1p-12f * F.sum);
        if (__all(settled)) {
            if (live) write_out(P, L, r, t, n, P.renorm ? 1.0 / (SIGMOID ? fmax(r.sum, 0x1p-14) : r.sum) : 1.0);
            return;
        }
    }
    double top, scale;
    choose_exact<V, SIGMOID, GROUPS>(P, L, top, scale);
    r = rank_candidates<SIGMOID, kMost>(P, L, P.k, top, scale);
    if (live) write_out(P, L, r, t, P.k, P.renorm ? 1.0 / fmax(r.sum, 0x1p-14) : 1.0);
}

template <int V>
hipError_t launch_select_v(const SelectParams &P, hipStream_t st, const LaunchTiming *tm) {
    const bool groups = P.n_group_used < P.n_group;
    // one wavefront per work-group: with four, 60000 tokens took the same time and 512 4% more (all scores in 64 bits then: 71 us,
    // and 10.6 instead of 10.2)
    const dim3 grid((P.T + kSelTokens - 1) / kSelTokens), block(kWave);
    const size_t lds = select_lds<V>(groups ? P.n_group : 0);
    if (P.sigmoid)
        return groups ? launch(select_kernel<V, true, true>, grid, block, lds, st, tm, P) : launch(select_kernel<V, true, false>, grid, block, lds, st, tm, P);
    return groups ? launch(select_kernel<V, false, true>, grid, block, lds, st, tm, P) : launch(select_kernel<V, false, false>, grid, block, lds, st, tm, P);
}

}  // namespace

hipError_t launch_select(const SelectParams &P, hipStream_t st, const LaunchTiming *tm) {
    if (P.T <= 0) return hipSuccess;
    if (P.E <= 64) return launch_select_v<4>(P, st, tm);
    if (P.E <= 128) return launch_select_v<8>(P, st, tm);
    return launch_select_v<16>(P, st, tm);
}

}  // namespace lstk
