// sample.hip - one token per row of logits: temperature, top-k, min-p and top-p from given random numbers.
//
// With the row's values in descending order (equal values: the lowest index first) and w_i = e^((x_i - x_max) / T):
//   the first top_k values with w >= min_p stay (at least one);  M = their sum
//   of those the shortest run from the top whose sum reaches top_p M stays;  S = its sum
//   the token is the first whose running sum exceeds u S;  its probability w / S
//
// No row is sorted. Each weight is rounded to a whole multiple of 2^-44 of the largest (of rows below 2^20 values; half a
// step is 3e-14), so running sums are whole numbers that come out the same in any order, atomics included. A histogram of
// counts and weights over kSampleBins equal steps of (x_max - x) / T says in which bins the three cuts fall; only those
// bins' values are looked at one by one. Weights that round to zero cannot be drawn and take no part.
#include <cfloat>

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

typedef unsigned long long u64;

constexpr int kSmThreads = 1024;
constexpr double kUnit = 0x1p44;
// (x_max - x) / T that the bins cover; the last one starts at 31.2347, where the weight is 0.479 * 2^-44, so all that it
// holds rounds to zero
constexpr float kSmRange = 31.25f;
constexpr double kSmStep = 31.25 / kSampleBins; // of (x_max - x) / T per bin

__device__ __forceinline__ float value_of(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
// order-preserving key of a float
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f); // -0 and 0 are equal values
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// larger is earlier in the order
__device__ __forceinline__ u64 place_of(float x, uint32_t i) { return (u64) key_of(x) << 32 | (uint32_t) ~i; }

struct Row {
    float top;
    float step; // bins per unit of x
    double inv_t, min_p;
};
__device__ __forceinline__ int bin_of(const Row &r, float x) {
    const float d = r.top - x;
    return d == 0.0f ? 0 : (int) fminf(d * r.step, (float) (kSampleBins - 1));
}
// e^(-i kSmStep) 2^44, the weight at the edge of bin i: e^z = 2^n e^r with |r| <= ln 2 / 2, and e^r by its series to r^12
// (what is left out is below 2e-16 of it).
__device__ __forceinline__ double edge_weight(int i) {
    const double z = -kSmStep * (double) i;
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
    return ldexp(p, (int) n + 44);
}
// The weight of a value of bin `bin`, times 2^44 (the largest value's: 2^44 exactly): the edge's, times e^r for the rest, which
// is at most a bin wide (0.0153), by its series to r^6 (what is left out is below 4e-17; the bin's own fp32 rounding can put a
// value 2e-6 of a bin beyond its edges, which changes nothing).
__device__ __forceinline__ double weight_of(const Row &r, float x, int bin, double edge) {
    const double d = fma((double) bin, kSmStep, ((double) x - (double) r.top) * r.inv_t);
    double p = 1.0 / 720;
    p = fma(p, d, 1.0 / 120);
    p = fma(p, d, 1.0 / 24);
    p = fma(p, d, 1.0 / 6);
    p = fma(p, d, 0.5);
    p = fma(p, d, 1.0);
    p = fma(p, d, 1.0);
    return p * edge;
}
// A value's weight as a whole number; 0 for those of the last bin and for one that min-p drops. The values that min-p keeps
// are a run from the top, so the first top_k of them are those of the first top_k values that it keeps. The sum with 2^52
// rounds to a whole number, which is then its mantissa.
__device__ __forceinline__ u64 mass_of(const Row &r, float x, int bin, double edge) {
    const double w = weight_of(r, x, bin, edge);
    return bin < kSampleBins - 1 && w >= r.min_p ? __builtin_bit_cast(u64, w + 0x1p52) & 0xfffffffffffffull : 0;
}
__device__ __forceinline__ u64 mass_of(const Row &r, float x) {
    const int bin = bin_of(r, x);
    return mass_of(r, x, bin, edge_weight(bin));
}

__device__ __forceinline__ u64 wave_max_u64(u64 v) {
    for (int d = 1; d < kWave; d *= 2) {
        const u64 o = __shfl_xor(v, d, kWave);
        v = o > v ? o : v;
    }
    return v;
}

// The largest of the row's slices; best 0 where no value is above -inf.
__device__ __forceinline__ u64 best_of(const SampleParams &P, int b) {
    u64 v = 0;
    for (int s = threadIdx.x & (kWave - 1); s < P.slices; s += kWave) {
        const u64 o = P.best[(int64_t) b * P.slices + s];
        v = o > v ? o : v;
    }
    return wave_max_u64(v);
}
__device__ __forceinline__ Row row_of(const SampleParams &P, int b, u64 best) {
    Row r;
    const float t = P.temperature ? P.temperature[b] : 1.0f;
    r.top = of_key((uint32_t) (best >> 32));
    r.step = (float) kSampleBins / (kSmRange * t);
    r.inv_t = 1.0 / (double) t;
    const float p = P.min_p ? P.min_p[b] : 0.0f;
    r.min_p = p > 0.0f ? (double) fminf(p, 1.0f) * kUnit : 0.0;
    return r;
}
__device__ __forceinline__ bool greedy(const SampleParams &P, int b) { return P.temperature && !(P.temperature[b] > 0.0f); }

__device__ __forceinline__ uint32_t top_k_of(const SampleParams &P, int b) {
    const int k = P.top_k ? P.top_k[b] : 0;
    return k > 0 ? (uint32_t) k : UINT_MAX;
}

// A row is read as 16-byte quads on 16-byte addresses: quad j holds the values 4 j - off .. + 3, off = the row's offset from
// such an address. What lies outside the row reads as -inf.
struct Quads {
    const float *x;
    int off, n, first, end; // values of the row; the slice's quads
};
__device__ __forceinline__ Quads quads_of(const SampleParams &P, int b, int s) {
    Quads q;
    q.x = P.logits + (int64_t) b * P.ld;
    q.off = (int) (reinterpret_cast<uintptr_t>(q.x) / 4 % 4);
    q.n = P.n_vocab;
    q.first = s * P.slice;
    q.end = min((q.n + q.off + 3) / 4, q.first + P.slice);
    return q;
}
__device__ __forceinline__ float4 quad_at(const Quads &q, int j) {
    const int i = 4 * j - q.off;
    if (i >= 0 && i + 4 <= q.n) return *reinterpret_cast<const float4 *>(q.x + i);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = i + e >= 0 && i + e < q.n ? q.x[i + e] : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
}
// Calls f(value, index) for the slice's values that are above -inf. kSmAhead quads of a thread are in flight at once.
constexpr int kSmAhead = 4;
template <typename F>
__device__ __forceinline__ void each_value(const Quads &q, F f) {
    for (int j0 = q.first + (int) threadIdx.x; j0 < q.end; j0 += kSmAhead * kSmThreads) {
        float4 v[kSmAhead];
#pragma unroll
        for (int a = 0; a < kSmAhead; a++)
            if (j0 + a * kSmThreads < q.end) v[a] = quad_at(q, j0 + a * kSmThreads);
#pragma unroll
        for (int a = 0; a < kSmAhead; a++) {
            const int j = j0 + a * kSmThreads;
            if (j >= q.end) break;
            const float w[4] = {v[a].x, v[a].y, v[a].z, v[a].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = value_of(w[e]);
                if (x > -INFINITY) f(x, 4 * j - q.off + e);
            }
        }
    }
}

// Largest value of each slice, and cleared histograms and counters for the next launches.
__global__ __launch_bounds__(kSmThreads) void sample_max_kernel(SampleParams P) {
    __shared__ u64 s_best[kSmThreads / kWave];
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    float top = -INFINITY;
    int at = 0;
    each_value(quads_of(P, b, s), [&](float x, int i) {
        if (x > top) { // a thread's values come in rising order of index
            top = x;
            at = i;
        }
    });
    u64 best = top > -INFINITY ? place_of(top, at) : 0;
    for (int i = s * kSmThreads + tid; i < kSampleBins; i += P.slices * kSmThreads) {
        P.mass[(int64_t) b * kSampleBins + i] = 0;
        P.count[(int64_t) b * kSampleBins + i] = 0;
    }
    if (s == 0 && tid == 0) P.n_list[b] = P.n_done[b] = 0u;
    best = wave_max_u64(best);
    if ((tid & (kWave - 1)) == 0) s_best[tid / kWave] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kSmThreads / kWave; w++) best = s_best[w] > best ? s_best[w] : best;
        P.best[(int64_t) b * P.slices + s] = best;
    }
}

__global__ __launch_bounds__(kSmThreads) void sample_bins_kernel(SampleParams P) {
    __shared__ u64 s_mass[kSampleBins];
    __shared__ uint32_t s_count[kSampleBins];
    __shared__ double s_edge[kSampleBins];
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    if (greedy(P, b)) return;
    const u64 best = best_of(P, b);
    if (best == 0) return;
    const Row r = row_of(P, b, best);
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        s_mass[i] = 0;
        s_count[i] = 0;
        s_edge[i] = edge_weight(i);
    }
    __syncthreads();
    const bool ranked = top_k_of(P, b) != UINT_MAX; // the counts are asked for only where ranks cut
    each_value(quads_of(P, b, s), [&](float x, int) {
        const int bin = bin_of(r, x);
        const u64 m = mass_of(r, x, bin, s_edge[bin]);
        if (m == 0) return;
        atomicAdd(&s_mass[bin], m);
        if (ranked) atomicAdd(&s_count[bin], 1u);
    });
    __syncthreads();
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        if (s_mass[i] == 0) continue;
        atomicAdd(&P.mass[(int64_t) b * kSampleBins + i], s_mass[i]);
        if (ranked) atomicAdd(&P.count[(int64_t) b * kSampleBins + i], s_count[i]);
    }
}

// Inclusive running sums of a row's histogram, kept by the threads: bins per * tid .. + per - 1.
constexpr int kSmPer = kSampleBins / kSmThreads;
struct Sums {
    u64 mass[kSmPer], mass0; // through each bin, and before the first
    uint32_t count[kSmPer], count0;
};
struct Found { // a bin in which a running sum reaches its target
    int bin;
    u64 mass0, mass;
    uint32_t count0, count;
};
struct SumsLds {
    u64 wave_mass[kSmThreads / kWave];
    uint32_t wave_count[kSmThreads / kWave];
    Found found[2];
};
__device__ __forceinline__ Sums sums_of(const SampleParams &P, int b, SumsLds &L) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    Sums S;
    u64 ms = 0;
    uint32_t cs = 0;
#pragma unroll
    for (int i = 0; i < kSmPer; i++) {
        ms += P.mass[(int64_t) b * kSampleBins + tid * kSmPer + i];
        cs += P.count[(int64_t) b * kSampleBins + tid * kSmPer + i];
        S.mass[i] = ms;
        S.count[i] = cs;
    }
    u64 im = ms;
    uint32_t ic = cs;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 om = __shfl_up(im, d, kWave);
        const uint32_t oc = __shfl_up(ic, d, kWave);
        if (lane >= d) {
            im += om;
            ic += oc;
        }
    }
    if (lane == kWave - 1) {
        L.wave_mass[wv] = im;
        L.wave_count[wv] = ic;
    }
    __syncthreads();
    S.mass0 = im - ms;
    S.count0 = ic - cs;
    for (int w = 0; w < wv; w++) {
        S.mass0 += L.wave_mass[w];
        S.count0 += L.wave_count[w];
    }
#pragma unroll
    for (int i = 0; i < kSmPer; i++) {
        S.mass[i] += S.mass0;
        S.count[i] += S.count0;
    }
    return S;
}
// The first bins whose running sums reach two targets (found[0], found[1]); a target lies in [1, the whole sum].
template <bool BY_MASS>
__device__ __forceinline__ void reaching(const Sums &S, SumsLds &L, u64 t0, u64 t1) {
    __syncthreads(); // the last call's results have been read
    u64 m0 = S.mass0;
    uint32_t c0 = S.count0;
#pragma unroll
    for (int i = 0; i < kSmPer; i++) {
        const u64 before = BY_MASS ? m0 : c0, sum = BY_MASS ? S.mass[i] : S.count[i];
        const Found f{(int) threadIdx.x * kSmPer + i, m0, S.mass[i], c0, S.count[i]};
        if (before < t0 && t0 <= sum) L.found[0] = f;
        if (before < t1 && t1 <= sum) L.found[1] = f;
        m0 = S.mass[i];
        c0 = S.count[i];
    }
    __syncthreads();
}

// The run of the top: how much of M it has to reach, as a whole number in [1, M].
__device__ __forceinline__ u64 top_p_target(const SampleParams &P, int b, u64 M) {
    const float p = P.top_p ? P.top_p[b] : 1.0f;
    if (!(p < 1.0f)) return M;
    if (!(p > 0.0f)) return 1;
    const u64 t = (u64) ceil((double) p * (double) M);
    return t < 1 ? 1 : t > M ? M : t;
}
// The least whole running sum above u S, in [1, S].
__device__ __forceinline__ u64 draw_target(const SampleParams &P, int b, u64 S) {
    const double u = (double) P.u[b];
    if (!(u > 0.0)) return 1;
    if (u >= 1.0) return S;
    const u64 t = (u64) floor(u * (double) S) + 1;
    return t > S ? S : t;
}

// The bins where a cut may fall. What stays by rank ends in bin `cut`, inside it where `part` is set (else at its end, or
// nowhere). The sum of what stays, M, lies between those before and after that bin, so the run that top-p keeps ends in bins
// [p_lo, p_hi] (where top-p cuts at all), and the draw in [d_lo, d_hi].
struct Cuts {
    uint32_t k; // values that stay by rank
    bool part, by_p;
    Found cut;
    u64 sum; // of what stays by rank, where not `part`
    int p_lo, p_hi, d_lo, d_hi;
    __device__ __forceinline__ bool holds(int bin) const {
        return (bin >= d_lo && bin <= d_hi) || (part && bin == cut.bin) || (by_p && bin >= p_lo && bin <= p_hi);
    }
};
__device__ __forceinline__ Cuts cuts_of(const SampleParams &P, int b, const Sums &S, SumsLds &L) {
    Cuts c;
    u64 m_hi = 0;
    uint32_t n = 0;
    for (int w = 0; w < kSmThreads / kWave; w++) {
        m_hi += L.wave_mass[w];
        n += L.wave_count[w];
    }
    u64 m_lo = m_hi;
    c.k = top_k_of(P, b);
    c.part = false;
    if (c.k < n) {
        reaching<false>(S, L, c.k, c.k);
        c.cut = L.found[0];
        c.part = c.cut.count != c.k;
        m_hi = c.cut.mass;
        m_lo = !c.part ? m_hi : c.cut.mass0 > 0 ? c.cut.mass0 : 1;
    }
    c.sum = m_hi;
    u64 s_lo = m_lo, s_hi = m_hi;
    c.by_p = (P.top_p ? P.top_p[b] : 1.0f) < 1.0f;
    if (c.by_p) {
        reaching<true>(S, L, top_p_target(P, b, m_lo), top_p_target(P, b, m_hi));
        c.p_lo = L.found[0].bin;
        c.p_hi = L.found[1].bin;
        s_lo = L.found[0].mass0 > 0 ? L.found[0].mass0 : 1;
        s_hi = L.found[1].mass < m_hi ? L.found[1].mass : m_hi;
    }
    reaching<true>(S, L, draw_target(P, b, s_lo), draw_target(P, b, s_hi));
    c.d_lo = L.found[0].bin;
    c.d_hi = L.found[1].bin;
    return c;
}

// The gathered values, and the search among those of one bin.
constexpr int kSmKeep = 1024;           // gathered values that are kept in LDS; more are read from the list again
constexpr int kSmGather = 2 * kSmKeep; // of a work-group's own, before they go to the list together
struct Search {
    union {
        u64 place[kSmKeep];
        int gathered[kSmGather]; // (before the search) this work-group's indices
    };
    u64 mass[kSmKeep];
    u64 digit_mass[256];
    uint32_t digit_count[256];
    u64 hi, lo, at, mass0;
    uint32_t count0, left;
};
struct Reached {
    u64 place; // of the value at which the running sum reaches the target
    u64 mass0; // running sum before it
};
// The value of bin `f` at which the running sum of weights (BY_MASS) or of values reaches `target`, which lies in that bin.
// The places of the bin's values, as whole numbers, are told apart 8 bits at a time from the first bit in which they differ:
// a histogram of those bits over the values still in question, and the running sum over it from the top.
template <bool BY_MASS>
__device__ __forceinline__ Reached reach(const SampleParams &P, int b, const Row &r, Search &D, const Found &f, uint32_t n, u64 target) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const float *x = P.logits + (int64_t) b * P.ld;
    auto each = [&](auto &&take) {
        for (uint32_t i = tid; i < n; i += kSmThreads) {
            if (n <= (uint32_t) kSmKeep) {
                const u64 p = D.place[i];
                if (bin_of(r, of_key((uint32_t) (p >> 32))) == f.bin) take(p, D.mass[i]);
            } else {
                const int at = ld_dev(P.list + (int64_t) b * P.n_vocab + i);
                const float v = value_of(x[at]);
                if (bin_of(r, v) == f.bin) take(place_of(v, (uint32_t) at), mass_of(r, v));
            }
        }
    };
    __syncthreads();
    if (tid == 0) {
        D.hi = 0;
        D.lo = ~0ull;
        D.mass0 = f.mass0;
        D.count0 = f.count0;
    }
    __syncthreads();
    u64 hi = 0, lo = ~0ull;
    each([&](u64 p, u64) {
        hi = p > hi ? p : hi;
        lo = p < lo ? p : lo;
    });
    if (hi >= lo) {
        atomicMax(&D.hi, hi);
        atomicMin(&D.lo, lo);
    }
    __syncthreads();
    hi = D.hi;
    // places in question: those that share their bits from `bit` up with `at`
    u64 at = hi;
    int bit = hi == D.lo ? 0 : 64 - __clzll((long long) (hi ^ D.lo));
    while (bit > 0) {
        const int shift = bit > 8 ? bit - 8 : 0;
        const u64 above = bit < 64 ? ~0ull << bit : 0;
        for (int i = tid; i < 256; i += kSmThreads) {
            D.digit_mass[i] = 0;
            D.digit_count[i] = 0;
        }
        __syncthreads();
        each([&](u64 p, u64 m) {
            if ((p ^ at) & above) return;
            const int d = (int) (p >> shift & 255);
            atomicAdd(&D.digit_mass[d], m);
            atomicAdd(&D.digit_count[d], 1u);
        });
        __syncthreads();
        if (tid < kWave) {
            // lane l takes digits 255 - 4 l .. 252 - 4 l
            u64 m = 0;
            uint32_t c = 0;
            u64 dm[4];
            uint32_t dc[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                dm[i] = D.digit_mass[255 - 4 * lane - i];
                dc[i] = D.digit_count[255 - 4 * lane - i];
                m += dm[i];
                c += dc[i];
            }
            u64 im = m;
            uint32_t ic = c;
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const u64 om = __shfl_up(im, d, kWave);
                const uint32_t oc = __shfl_up(ic, d, kWave);
                if (lane >= d) {
                    im += om;
                    ic += oc;
                }
            }
            u64 m0 = D.mass0 + im - m;
            uint32_t c0 = D.count0 + ic - c;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const u64 before = BY_MASS ? m0 : c0, sum = BY_MASS ? m0 + dm[i] : c0 + dc[i];
                if (before < target && target <= sum) {
                    D.at = (at & above & ~(255ull << shift)) | (u64) (255 - 4 * lane - i) << shift;
                    D.left = dc[i];
                    D.mass0 = m0; // every lane has read the old sums: the wavefront runs in step
                    D.count0 = c0;
                }
                m0 += dm[i];
                c0 += dc[i];
            }
        }
        __syncthreads();
        at = D.at;
        bit = shift;
        if (D.left == 1) { // one value: its place
            each([&](u64 p, u64) {
                if (!((p ^ at) & ~0ull << shift)) D.hi = p;
            });
            __syncthreads();
            at = D.hi;
            break;
        }
    }
    return {at, D.mass0};
}

// Gathers the values in the bins where a cut may fall; the row's last work-group to be done finds the cuts among them and
// draws.
__global__ __launch_bounds__(kSmThreads) void sample_pick_kernel(SampleParams P) {
    __shared__ SumsLds L;
    __shared__ Search D;
    __shared__ uint32_t s_n, s_base;
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    const u64 best = best_of(P, b);
    if (best == 0 || greedy(P, b)) {
        if (s == 0 && tid == 0) {
            P.tokens[b] = best == 0 ? -1 : (int32_t) ~(uint32_t) best;
            if (P.probs) P.probs[b] = best == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    const Row r = row_of(P, b, best);
    if (tid == 0) s_n = 0;
    const Sums S = sums_of(P, b, L);
    const Cuts c = cuts_of(P, b, S, L);
    int *list = P.list + (int64_t) b * P.n_vocab;
    each_value(quads_of(P, b, s), [&](float x, int i) {
        const int bin = bin_of(r, x);
        if (!c.holds(bin) || mass_of(r, x, bin, edge_weight(bin)) == 0) return;
        const uint32_t at = atomicAdd(&s_n, 1u);
        if (at < (uint32_t) kSmGather) D.gathered[at] = i;
        else st_dev(list + atomicAdd(&P.n_list[b], 1u), i);
    });
    // one place in the list for all that fitted (a global counter's answer takes a microsecond: one each, and a wavefront that
    // meets 20 such values takes 20)
    __syncthreads();
    const uint32_t mine = min(s_n, (uint32_t) kSmGather);
    if (tid == 0 && mine > 0) s_base = atomicAdd(&P.n_list[b], mine);
    __syncthreads();
    for (uint32_t i = tid; i < mine; i += kSmThreads) st_dev(list + s_base + i, D.gathered[i]);
    // Hand-over without an L2 write-back: the entries are device-coherent stores, complete before the work-group counts itself
    // done, and read with device-coherent loads by the one that counts last.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s_n = atomicAdd(&P.n_done[b], 1u) + 1 == (uint32_t) P.slices ? atomicAdd(&P.n_list[b], 0u) : UINT_MAX;
    __syncthreads();
    const uint32_t n = s_n;
    if (n == UINT_MAX) return;
    if (n <= (uint32_t) kSmKeep) {
        const float *x = P.logits + (int64_t) b * P.ld;
        for (uint32_t i = tid; i < n; i += kSmThreads) {
            const int at = ld_dev(list + i);
            const float v = value_of(x[at]);
            D.place[i] = place_of(v, (uint32_t) at);
            D.mass[i] = mass_of(r, v);
        }
    }
    auto mass_at = [&](u64 place) { return mass_of(r, of_key((uint32_t) (place >> 32))); };
    u64 total = c.sum;
    if (c.part) {
        const Reached at = reach<false>(P, b, r, D, c.cut, n, c.k);
        total = at.mass0 + mass_at(at.place);
    }
    if (c.by_p) {
        const u64 target = top_p_target(P, b, total);
        reaching<true>(S, L, target, target);
        const Reached at = reach<true>(P, b, r, D, L.found[0], n, target);
        total = at.mass0 + mass_at(at.place);
    }
    const u64 target = draw_target(P, b, total);
    reaching<true>(S, L, target, target);
    const Reached at = reach<true>(P, b, r, D, L.found[0], n, target);
    if (tid == 0) {
        P.tokens[b] = (int32_t) ~(uint32_t) at.place;
        const float x = of_key((uint32_t) (at.place >> 32));
        const int bin = bin_of(r, x);
        if (P.probs) P.probs[b] = (float) (weight_of(r, x, bin, edge_weight(bin)) / (double) total);
    }
}

}  // namespace

size_t sample_plan(SampleParams &P, void *work) {
    // slices of at least 1024 quads, as many as bring the launches to 512 work-groups; a row out of line has a quad more
    const int quads = (P.n_vocab + 6) / 4;
    P.slices = std::max(1, std::min((quads + kSmThreads - 1) / kSmThreads, 256 / std::max(1, P.n_rows)));
    P.slice = (quads + P.slices - 1) / P.slices;
    size_t off = 0;
    auto take = [&](auto *&p, size_t n) {
        p = work ? reinterpret_cast<std::remove_reference_t<decltype(p)>>(static_cast<uint8_t *>(work) + off) : nullptr;
        off += (n * sizeof(*p) + 255) / 256 * 256;
    };
    const size_t rows = (size_t) P.n_rows;
    take(P.best, rows * P.slices);
    take(P.mass, rows * kSampleBins);
    take(P.count, rows * kSampleBins);
    take(P.n_list, rows);
    take(P.n_done, rows);
    take(P.list, rows * P.n_vocab);
    return off;
}

hipError_t launch_sample(const SampleParams &P, hipStream_t st) {
    if (P.n_rows <= 0) return hipSuccess;
    const dim3 all((unsigned) (P.n_rows * P.slices)), block(kSmThreads);
    hipError_t e;
    if ((e = launch(sample_max_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    if ((e = launch(sample_bins_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    return launch(sample_pick_kernel, all, block, 0, st, nullptr, P);
}

}  // namespace lstk
