// select.hip - routing to experts by a rule, from router logits.
//
//   s_e = softmax(x)_e or 1 / (1 + e^-x_e);  c_e = s_e + bias_e  (the choice values)
//   a group's value is the sum of its `group_top` largest c; the best n_group_used groups stay; of their experts the k largest
//   c are chosen (equal values: the lowest id), in that order;  w = s / max(sum of the chosen s, 2^-14) * scale
//
// Scores and choice values are held in 64 bits: two experts a 32-bit rounding apart would swap places with the compiler's
// choice of instructions. The chosen weights are rounded once, to fp32.
//
// 16 lanes (a DPP row) take a token, so a wavefront takes four, and lane l the experts l, l + 16, ..: a row's maximum is four
// DPP steps. A choice value carries its expert in its lowest 8 mantissa bits (2^-44 of it), so that the maximum says whose it
// is and of equal values the lowest id is the largest. In each of the k rounds the lane that owned the maximum takes it out of
// its values in LDS and finds its next one; the others keep theirs.
#include <cfloat>

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
    double r = fma(n, -0.6931471803691238, z); // ln 2 in two parts, the first of 33 bits
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

// A choice value with its expert: larger is earlier. -inf becomes a finite value below all others, so that it stays above what
// may not be chosen at all (-inf here).
__device__ __forceinline__ double tagged(double c, int e) {
    c = fmin(fmax(c, -0x1p1023), 0x1p1023); // (a NaN becomes -2^1023)
    const unsigned long long u = __builtin_bit_cast(unsigned long long, c);
    return __builtin_bit_cast(double, (u & ~255ull) | (u >> 63 ? (unsigned) e : 255u - (unsigned) e));
}
__device__ __forceinline__ int expert_of(double t) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, t);
    return (int) (u >> 63 ? u & 255u : 255u - (u & 255u));
}

// LDS of one wavefront: the choice values of each token, lane by lane (two more a lane against bank conflicts), the chosen
// ids, and with groups their values and which of them stay.
template <int V>
__host__ __device__ constexpr size_t select_lds(int k, int groups) {
    return kSelTokens * ((size_t) kSelLanes * (V + 2) * 8 + (size_t) groups * 8 + (groups ? 32 : 0) + (size_t) k * 4);
}
// Orders a wavefront's LDS writes before its later reads by other lanes (they execute in order; the compiler has to as well).
__device__ __forceinline__ void lds_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// V: experts per lane, 16 V >= E
template <int V, bool SIGMOID, bool GROUPS>
__global__ __launch_bounds__(kWave) void select_kernel(SelectParams P) {
    extern __shared__ __align__(16) unsigned char s_all[];
    const int l = threadIdx.x % kSelLanes, row = threadIdx.x / kSelLanes;
    unsigned char *lds = s_all;
    double *const s_c = reinterpret_cast<double *>(lds) + (row * kSelLanes) * (V + 2); // the token's values: lane's at (V + 2) l
    double *const mine = s_c + l * (V + 2);
    lds += kSelTokens * kSelLanes * (V + 2) * 8;
    double *s_g = nullptr;
    uint32_t *s_keep = nullptr;
    if constexpr (GROUPS) {
        s_g = reinterpret_cast<double *>(lds) + row * P.n_group;
        lds += (size_t) kSelTokens * P.n_group * 8;
        s_keep = reinterpret_cast<uint32_t *>(lds) + row * 8;
        lds += kSelTokens * 32;
    }
    int *const s_id = reinterpret_cast<int *>(lds) + row * P.k;
    const int64_t first = (int64_t) blockIdx.x * kSelTokens;
    const int64_t t = min(first + row, (int64_t) P.T - 1); // rows past the last token compute it again and store nothing
    const float *x = P.logits + t * P.ld;

    float xv[V], bv[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = l + kSelLanes * i;
        xv[i] = e < P.E ? x[e] : -INFINITY;
        bv[i] = P.bias && e < P.E ? P.bias[e] : 0.0f;
    }
    double c[V], top = 0.0, scale = 1.0; // softmax: e^(x - top) * scale
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
#pragma unroll
    for (int i = 0; i < V; i++) {
        c[i] += (double) bv[i];
        if (c[i] != c[i]) c[i] = -INFINITY;
    }
    unsigned out = 0; // bit i: expert l + 16 i may not be chosen
#pragma unroll
    for (int i = 0; i < V; i++) out |= (l + kSelLanes * i < P.E ? 0u : 1u) << i;
    if constexpr (GROUPS) {
        const int per = P.E / P.n_group;
        const unsigned inv = (65536u + per - 1) / per; // e / per = e * inv >> 16 for e < 256
#pragma unroll
        for (int i = 0; i < V; i++) mine[i] = c[i];
        if (l < 8) s_keep[l] = 0;
        lds_in_order();
        for (int g = l; g < P.n_group; g += kSelLanes) {
            double a = -INFINITY, b = -INFINITY; // the two largest
            for (int j = 0; j < per; j++) {
                const int e = g * per + j;
                const double v = s_c[(e % kSelLanes) * (V + 2) + e / kSelLanes];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
            const double v = P.group_top == 2 ? a + b : a;
            s_g[g] = v != v ? -INFINITY : v;
        }
        lds_in_order();
        for (int g = l; g < P.n_group; g += kSelLanes) {
            const double v = s_g[g];
            int rank = 0;
            for (int j = 0; j < P.n_group; j++) {
                const double o = s_g[j];
                rank += o > v || (o == v && j < g);
            }
            if (rank < P.n_group_used) atomicOr(&s_keep[g / 32], 1u << (g % 32));
        }
        lds_in_order();
#pragma unroll
        for (int i = 0; i < V; i++) {
            const unsigned g = (l + kSelLanes * i) * inv >> 16;
            out |= (~s_keep[g / 32] >> (g % 32) & 1u) << i;
        }
    }
    double best = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const double v = out >> i & 1u ? -INFINITY : tagged(c[i], l + kSelLanes * i);
        mine[i] = v;
        best = fmax(best, v);
    }
    for (int j = 0; j < P.k; j++) {
        const int e = expert_of(row_max(best));
        if (l == e % kSelLanes) {
            s_id[j] = e;
            mine[e / kSelLanes] = -INFINITY;
            double v[V];
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = mine[i];
            best = v[0];
#pragma unroll
            for (int i = 1; i < V; i++) best = fmax(best, v[i]);
        }
    }
    lds_in_order();
    // the chosen experts' scores, 16 at a time
    double sum = 0.0;
    auto score = [&](int j) {
        const double v = value_of(x[s_id[j]]);
        if constexpr (SIGMOID) return sigmoid(v);
        else return exp_of(fmax(v - top, -800.0)) * scale;
    };
    for (int j = l; j < P.k; j += kSelLanes) {
        const double s = score(j);
        sum += s;
        mine[j / kSelLanes] = s;
    }
    sum = row_sum(sum);
    if (first + row >= P.T) return;
    const double f = (P.renorm ? 1.0 / fmax(sum, 0x1p-14) : 1.0) * (double) P.scale;
    for (int j = l; j < P.k; j += kSelLanes) {
        P.ids[t * P.k + j] = s_id[j];
        P.weights[t * P.k + j] = (float) (mine[j / kSelLanes] * f);
    }
}

template <int V>
hipError_t launch_select_v(const SelectParams &P, hipStream_t st, const LaunchTiming *tm) {
    const bool groups = P.n_group_used < P.n_group;
    // one wavefront per work-group: with four, 60000 tokens take the same 71 us and 512 take 10.6 instead of 10.2
    const dim3 grid((P.T + kSelTokens - 1) / kSelTokens), block(kWave);
    const size_t lds = select_lds<V>(P.k, groups ? P.n_group : 0);
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
