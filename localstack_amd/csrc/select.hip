// select.hip - routing to experts by a rule, from router logits.
//
//   s_e = softmax(x)_e or 1 / (1 + e^-x_e);  c_e = s_e + bias_e  (the choice values)
//   a group's value is the sum of its `group_top` largest c; the best n_group_used groups stay; of their experts the k largest
//   c are chosen (equal values: the lowest id), in that order;  w = s / max(sum of the chosen s, 2^-14) * scale
//
// Scores and choice values are held in 64 bits: two experts a 32-bit rounding apart would swap places with the compiler's
// choice of instructions. The chosen weights are rounded once, to fp32.
#include <cfloat>

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

constexpr int kSelWaves = kBlock / kWave; // tokens per work-group, one per wavefront

__device__ __forceinline__ double finite(float x) { return x != x ? -INFINITY : (double) fminf(x, FLT_MAX); }

__global__ __launch_bounds__(kBlock) void select_kernel(SelectParams P) {
    __shared__ double s_c[kSelWaves][kMaxEPL * kWave];
    __shared__ double s_g[kSelWaves][kMaxEPL * kWave];
    const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave;
    const int64_t t = (int64_t) blockIdx.x * kSelWaves + wv;
    const bool live = t < P.T;
    const float *x = P.logits + (live ? t : 0) * P.ld;
    double s[kMaxEPL], c[kMaxEPL];
    double top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxEPL; i++) {
        const int e = lane + kWave * i;
        s[i] = e < P.E ? finite(x[e]) : -INFINITY;
        top = fmax(top, s[i]);
    }
    if (P.sigmoid) {
#pragma unroll
        for (int i = 0; i < kMaxEPL; i++) s[i] = 1.0 / (1.0 + exp(-s[i]));
    } else {
        for (int d = 1; d < kWave; d *= 2) top = fmax(top, __shfl_xor(top, d, kWave));
        if (top == -INFINITY) top = 0.0;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kMaxEPL; i++) {
            s[i] = exp(s[i] - top);
            sum += s[i];
        }
        sum = wave_sum_d(sum);
#pragma unroll
        for (int i = 0; i < kMaxEPL; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    }
#pragma unroll
    for (int i = 0; i < kMaxEPL; i++) {
        const int e = lane + kWave * i;
        c[i] = P.bias && e < P.E ? s[i] + (double) P.bias[e] : s[i];
        if (c[i] != c[i]) c[i] = -INFINITY;
        s_c[wv][e] = c[i];
    }
    unsigned on = 0; // bit i: expert lane + 64 i may be chosen
    const int per = P.E / P.n_group;
#pragma unroll
    for (int i = 0; i < kMaxEPL; i++)
        if (lane + kWave * i < P.E) on |= 1u << i;
    if (P.n_group_used < P.n_group) {
        __syncthreads();
        for (int g = lane; g < P.n_group; g += kWave) {
            double a = -INFINITY, b = -INFINITY; // the two largest
            for (int j = 0; j < per; j++) {
                const double v = s_c[wv][g * per + j];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
            s_g[wv][g] = P.group_top == 2 ? a + b : a;
            if (s_g[wv][g] != s_g[wv][g]) s_g[wv][g] = -INFINITY;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMaxEPL; i++) {
            const int e = lane + kWave * i;
            if (e >= P.E) continue;
            const int g = e / per;
            const double v = s_g[wv][g];
            int rank = 0;
            for (int j = 0; j < P.n_group; j++) {
                const double o = s_g[wv][j];
                rank += o > v || (o == v && j < g);
            }
            if (rank >= P.n_group_used) on &= ~(1u << i);
        }
    }
    double sum = 0.0, mine = 0.0; // lane j keeps the score of the j-th chosen expert
    for (int j = 0; j < P.k; j++) {
        double v = -INFINITY, sv = 0.0;
        int e = INT_MAX;
#pragma unroll
        for (int i = 0; i < kMaxEPL; i++) {
            if ((on >> i & 1u) && (e == INT_MAX || c[i] > v)) {
                v = c[i];
                sv = s[i];
                e = lane + kWave * i;
            }
        }
        for (int d = 1; d < kWave; d *= 2) {
            const double ov = __shfl_xor(v, d, kWave), os = __shfl_xor(sv, d, kWave);
            const int oe = __shfl_xor(e, d, kWave);
            if (oe != INT_MAX && (e == INT_MAX || ov > v || (ov == v && oe < e))) {
                v = ov;
                sv = os;
                e = oe;
            }
        }
        sum += sv;
        if (lane == j) {
            mine = sv;
            if (live) P.ids[t * P.k + j] = e;
        }
        if (e % kWave == lane) on &= ~(1u << (e / kWave));
    }
    if (live && lane < P.k) P.weights[t * P.k + lane] = (float) ((P.renorm ? mine / fmax(sum, 0x1p-14) : mine) * (double) P.scale);
}

}  // namespace

hipError_t launch_select(const SelectParams &P, hipStream_t st, const LaunchTiming *tm) {
    if (P.T <= 0) return hipSuccess;
    return launch(select_kernel, dim3((P.T + kSelWaves - 1) / kSelWaves), dim3(kBlock), 0, st, tm, P);
}

}  // namespace lstk
