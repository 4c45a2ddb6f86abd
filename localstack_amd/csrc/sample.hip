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
//
// Measured on MI355X: 64 rows of 151936 values (39 MB) 58 us in three launches of 9 (reading at 4.3 TB/s), 17 (the vector units
// are busy for 39% of it, mostly with the weights; the rest are waits, LDS atomics among them) and 32 us (18%; waits in turn:
// histogram, cuts, the row again, the row's last work-group); one such row 22 us.

#include <cfloat>
#include <type_traits>

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

typedef unsigned long long u64;

constexpr int kSmThreads = 512;
constexpr int kSmTarget = 512; // work-groups of a launch
constexpr int kSmHeld = 24;    // quads of a thread where a row takes one work-group: up to 49149 values
constexpr double kUnit = 0x1p44;
// (x_max - x) / T that the bins cover; the last one starts at 31.2347, where the weight is 0.479 * 2^-44, so all that it
// holds rounds to zero
constexpr double kSmRange = 31.25;
constexpr double kSmStep = kSmRange / kSampleBins; // of (x_max - x) / T per bin

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
    double top;   // the largest value
    double scale; // bins per unit of x
    double min_p; // in units of 2^-44
    float least;  // nothing below has a weight, -inf and NaN among it (a little lower than need be)
};
// The largest float that is at most x, or one a few steps lower; at least the lowest finite one.
__device__ __forceinline__ float float_below(double x) {
    const float f = (float) fmin(fmax(x, (double) -FLT_MAX), (double) FLT_MAX);
    return fmaxf(f - fabsf(f) * 0x1p-22f - FLT_MIN, -FLT_MAX);
}
// How many bins below the largest value x lies, up to the last bin's edge.
__device__ __forceinline__ double bins_below(const Row &r, float x) { return fmin((r.top - (double) x) * r.scale, (double) (kSampleBins - 1)); }
__device__ __forceinline__ int bin_of(const Row &r, float x) { return (int) bins_below(r, x); }
// e^(-i kSmStep) 2^44, the weight at the edge of bin i: e^z = 2^n e^r with |r| <= ln 2 / 2, and e^r by its series to r^12
// (what is left out is below 2e-16 of it).
__device__ __forceinline__ double edge_weight(int i) {
    const double z = -kSmStep * (double) i;
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
    return ldexp(p, (int) n + 44);
}
// The weight of a value `below` bins from the largest, times 2^44 (the largest value's: 2^44 exactly): that of its bin's edge,
// times e^-r for the rest of a bin r < kSmStep = 0.0153, by its series to r^5 (what is left out is below 1.8e-14).
__device__ __forceinline__ double weight_of(double below, int bin, double edge) {
    constexpr double h = kSmStep;
    const double f = below - (double) bin;
    double p = -h * h * h * h * h / 120;
    p = fma(p, f, h * h * h * h / 24);
    p = fma(p, f, -h * h * h / 6);
    p = fma(p, f, h * h / 2);
    p = fma(p, f, -h);
    p = fma(p, f, 1.0);
    return p * edge;
}
// A value's weight as a whole number; 0 for those of the last bin and for one that min-p drops. The values that min-p keeps
// are a run from the top, so the first top_k of them are those of the first top_k values that it keeps. The sum with 2^52
// rounds to a whole number, which is then its mantissa.
__device__ __forceinline__ u64 mass_of(const Row &r, double below, int bin, double edge) {
    const double w = weight_of(below, bin, edge);
    return bin < kSampleBins - 1 && w >= r.min_p ? __builtin_bit_cast(u64, w + 0x1p52) & 0xfffffffffffffull : 0;
}
__device__ __forceinline__ u64 mass_of(const Row &r, float x) {
    const double below = bins_below(r, x);
    return mass_of(r, below, (int) below, edge_weight((int) below));
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
// A row's settings, asked for together at a kernel's start (each would be a wait of its own where it is used).
struct Settings {
    float t, p, min_p, u;
    uint32_t k;
    bool greedy;
};
__device__ __forceinline__ Settings settings_of(const SampleParams &P, int b) {
    const float t = P.temperature ? P.temperature[b] : 1.0f, p = P.top_p ? P.top_p[b] : 1.0f, min_p = P.min_p ? P.min_p[b] : 0.0f;
    const int k = P.top_k ? P.top_k[b] : 0;
    const float u = P.u[b];
    return {t, p, min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f, u, k > 0 ? (uint32_t) k : UINT_MAX, !(t > 0.0f)};
}
__device__ __forceinline__ Row row_of(const Settings &how, u64 best) {
    Row r;
    r.top = (double) of_key((uint32_t) (best >> 32));
    r.scale = (double) kSampleBins / (kSmRange * (double) how.t);
    r.min_p = (double) how.min_p * kUnit;
    double range = kSmRange;
    if (how.min_p > 0.0f) range = fmin(range, 1e-6 - log((double) how.min_p));
    r.least = float_below(r.top - range * (double) how.t);
    return r;
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
// kSmAhead quads of a thread are in flight at once; the first ones may be asked for long before they are needed.
constexpr int kSmAhead = 4;
struct Ahead {
    float4 v[kSmAhead];
};
__device__ __forceinline__ Ahead ahead_of(const Quads &q, int j0) {
    Ahead a;
#pragma unroll
    for (int i = 0; i < kSmAhead; i++) {
        const int j = j0 + i * kSmThreads;
        a.v[i] = j < q.end ? quad_at(q, j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    return a;
}
// Calls f(value as stored, index) for the slice's values and some -inf beyond, a thread's in rising order of index; `a` =
// ahead_of(q, q.first + threadIdx.x).
template <typename F>
__device__ __forceinline__ void each_value(const Quads &q, Ahead a, F f) {
    for (int j0 = q.first + (int) threadIdx.x; j0 < q.end;) {
        const Ahead now = a;
        const int j1 = j0 + kSmAhead * kSmThreads;
        if (j1 < q.end) a = ahead_of(q, j1);
#pragma unroll
        for (int i = 0; i < kSmAhead; i++) {
            const int at = 4 * (j0 + i * kSmThreads) - q.off;
            f(now.v[i].x, at);
            f(now.v[i].y, at + 1);
            f(now.v[i].z, at + 2);
            f(now.v[i].w, at + 3);
        }
        j0 = j1;
    }
}

// Largest value of each slice, and cleared histograms and counters for the next launches.
__global__ __launch_bounds__(kSmThreads) void sample_max_kernel(SampleParams P) {
    __shared__ u64 s_best[kSmThreads / kWave];
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    float top = -INFINITY;
    int at = 0;
    const Quads q = quads_of(P, b, s);
    each_value(q, ahead_of(q, q.first + tid), [&](float x, int i) {
        x = x > FLT_MAX ? FLT_MAX : x;
        if (x > top) { // (a NaN is not)
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
    const Settings how = settings_of(P, b);
    if (how.greedy) return;
    const Quads q = quads_of(P, b, s);
    const Ahead ahead = ahead_of(q, q.first + tid);
    const bool ranked = how.k != UINT_MAX; // the counts are asked for only where ranks cut
    const u64 best = best_of(P, b);
    if (best == 0) return;
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        s_mass[i] = 0;
        s_count[i] = 0;
        s_edge[i] = edge_weight(i);
    }
    const Row r = row_of(how, best);
    __syncthreads();
    each_value(q, ahead, [&](float x, int) {
        if (!(x >= r.least)) return;
        const double below = bins_below(r, fminf(x, FLT_MAX));
        const int bin = (int) below;
        const u64 m = mass_of(r, below, bin, s_edge[bin]);
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
__device__ __forceinline__ Sums sums_of(const u64 *mass, const uint32_t *count, SumsLds &L) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    Sums S;
    u64 ms = 0;
    uint32_t cs = 0;
#pragma unroll
    for (int i = 0; i < kSmPer; i++) {
        ms += mass[tid * kSmPer + i];
        cs += count[tid * kSmPer + i];
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
__device__ __forceinline__ u64 top_p_target(const Settings &how, u64 M) {
    if (!(how.p < 1.0f)) return M;
    if (!(how.p > 0.0f)) return 1;
    const u64 t = (u64) ceil((double) how.p * (double) M);
    return t < 1 ? 1 : t > M ? M : t;
}
// The least whole running sum above u S, in [1, S].
__device__ __forceinline__ u64 draw_target(const Settings &how, u64 S) {
    if (!(how.u > 0.0f)) return 1;
    if (how.u >= 1.0f) return S;
    const u64 t = (u64) floor((double) how.u * (double) S) + 1;
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
__device__ __forceinline__ Cuts cuts_of(const Settings &how, const Sums &S, SumsLds &L) {
    Cuts c;
    u64 m_hi = 0;
    uint32_t n = 0;
    for (int w = 0; w < kSmThreads / kWave; w++) {
        m_hi += L.wave_mass[w];
        n += L.wave_count[w];
    }
    u64 m_lo = m_hi;
    c.k = how.k;
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
    c.by_p = how.p < 1.0f;
    if (c.by_p) {
        reaching<true>(S, L, top_p_target(how, m_lo), top_p_target(how, m_hi));
        c.p_lo = L.found[0].bin;
        c.p_hi = L.found[1].bin;
        s_lo = L.found[0].mass0 > 0 ? L.found[0].mass0 : 1;
        s_hi = L.found[1].mass < m_hi ? L.found[1].mass : m_hi;
    }
    reaching<true>(S, L, draw_target(how, s_lo), draw_target(how, s_hi));
    c.d_lo = L.found[0].bin;
    c.d_hi = L.found[1].bin;
    return c;
}

// The search among the gathered values. Up to kSmKeep of them are sorted by place (larger first) once, with the running sum of
// their weights; more are left in the list, and told apart there by digits.
constexpr int kSmKeep = 1024;
constexpr int kSmGather = kSmKeep; // places that a work-group gathers before they go to the list together
struct Search {
    union {
        struct {
            u64 place[kSmKeep], before[kSmKeep]; // sorted, and the sum of the weights before each
        };
        u64 gathered[kSmGather];
        struct {
            u64 digit_mass[256];
            uint32_t digit_count[256];
            u64 hi, lo, at;
            uint32_t count0, left;
        };
    };
    uint32_t rank[kSmThreads];
    u64 wave_mass[kSmThreads / kWave];
    u64 found, mass0; // answer
    int first;        // the bin's first value
};
struct Reached {
    u64 place; // of the value at which the running sum reaches the target
    u64 mass0; // running sum before it
};

// Sorts the places of `n` values (place(i), i < n <= kSmKeep) and sums their weights.
template <typename F>
__device__ __forceinline__ void sort_gathered(const Row &r, Search &D, int n, F place) {
    constexpr int E = kSmKeep / kSmThreads; // entries of a thread
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    u64 mine[E];
#pragma unroll
    for (int e = 0; e < E; e++) mine[e] = tid + e * kSmThreads < n ? place(tid + e * kSmThreads) : 0;
    __syncthreads(); // place() may read what is written now
    int size = 1;
    while (size < n) size *= 2;
    // up to kSmThreads values by counting, of each, those before it (the threads of a value share the count): 206 values 1 us,
    // 400 4 us, where the exchanges below take 7 and 10
    const bool by_count = size <= kSmThreads;
    if (by_count) {
        if (tid < size) {
            D.before[tid] = mine[0];
            D.rank[tid] = 0;
        }
        __syncthreads();
        const int parts = kSmThreads / size, each = (n + parts - 1) / parts, from = tid / size * each;
        const u64 own = D.before[tid % size];
        uint32_t rank = 0;
#pragma unroll 8
        for (int j = from; j < min(n, from + each); j++) rank += D.before[j] > own;
        if (own > 0) atomicAdd(&D.rank[tid % size], rank);
        __syncthreads();
        if (tid < n) D.place[D.rank[tid]] = mine[0];
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) D.place[tid + e * kSmThreads] = mine[e];
    }
    __syncthreads();
    for (int run = 2; run <= size && !by_count; run *= 2) {
        for (int step = run / 2; step > 0; step /= 2) {
            for (int p = tid; p < size / 2; p += kSmThreads) {
                const int i = 2 * p - (p & (step - 1)), j = i + step; // the pair's first and second place
                const u64 a = D.place[i], o = D.place[j];
                if ((a < o) == ((i & run) == 0)) {
                    D.place[i] = o;
                    D.place[j] = a;
                }
            }
            __syncthreads();
        }
    }
    u64 m[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = tid * E + e;
        m[e] = i < n ? mass_of(r, of_key((uint32_t) (D.place[i] >> 32))) : 0;
        sum += m[e];
    }
    u64 upto = sum;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 o = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += o;
    }
    if (lane == kWave - 1) D.wave_mass[wv] = upto;
    __syncthreads();
    upto -= sum;
    for (int w = 0; w < wv; w++) upto += D.wave_mass[w];
#pragma unroll
    for (int e = 0; e < E; e++) {
        D.before[tid * E + e] = upto;
        upto += m[e];
    }
    __syncthreads();
}

// The value of bin `f` at which the running sum of weights (BY_MASS) or of values reaches `target`, which lies in that bin.
template <bool BY_MASS>
__device__ __forceinline__ Reached reach_sorted(const Row &r, Search &D, const Found &f, int n, u64 target) {
    for (int i = threadIdx.x; i < n; i += kSmThreads) {
        auto bin_at = [&](int at) { return bin_of(r, of_key((uint32_t) (D.place[at] >> 32))); };
        if (bin_at(i) == f.bin && (i == 0 || bin_at(i - 1) != f.bin)) D.first = i;
    }
    __syncthreads();
    const int first = D.first;
    for (int i = threadIdx.x; i < n; i += kSmThreads) {
        const u64 place = D.place[i];
        const float x = of_key((uint32_t) (place >> 32));
        const u64 mass0 = f.mass0 + D.before[i] - D.before[first];
        const u64 before = BY_MASS ? mass0 : f.count0 + (uint32_t) (i - first);
        if (i >= first && bin_of(r, x) == f.bin && before < target && target <= before + (BY_MASS ? mass_of(r, x) : 1)) {
            D.found = place;
            D.mass0 = mass0;
        }
    }
    __syncthreads();
    const Reached out{D.found, D.mass0};
    __syncthreads();
    return out;
}

// The same among the n entries of the list: the places of the bin's values, as whole numbers, are told apart 8 bits at a time
// from the first bit in which they differ, by a histogram of those bits over the values still in question and the running sum
// over it from the top.
template <bool BY_MASS>
__device__ __forceinline__ Reached reach_in_list(const Row &r, const u64 *list, Search &D, const Found &f, uint32_t n,
                                                 u64 target) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    auto each = [&](auto &&take) {
        for (uint32_t i = tid; i < n; i += kSmThreads) {
            const u64 p = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const float v = of_key((uint32_t) (p >> 32));
            if (bin_of(r, v) == f.bin) take(p, v);
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
    each([&](u64 p, float) {
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
        each([&](u64 p, float v) {
            if ((p ^ at) & above) return;
            const int d = (int) (p >> shift & 255);
            atomicAdd(&D.digit_mass[d], mass_of(r, v));
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
            each([&](u64 p, float) {
                if (!((p ^ at) & ~0ull << shift)) D.hi = p;
            });
            __syncthreads();
            at = D.hi;
            break;
        }
    }
    return {at, D.mass0};
}

// The cuts and the draw. reach(by_mass, bin, target) is one of the two above.
template <typename F>
__device__ __forceinline__ void draw(const SampleParams &P, const Settings &how, int b, const Row &r, const Cuts &c, const Sums &S, SumsLds &L, F reach) {
    auto mass_at = [&](u64 place) { return mass_of(r, of_key((uint32_t) (place >> 32))); };
    u64 total = c.sum;
    if (c.part) {
        const Reached at = reach(std::false_type(), c.cut, c.k);
        total = at.mass0 + mass_at(at.place);
    }
    if (c.by_p) {
        const u64 target = top_p_target(how, total);
        reaching<true>(S, L, target, target);
        const Reached at = reach(std::true_type(), L.found[0], target);
        total = at.mass0 + mass_at(at.place);
    }
    const u64 target = draw_target(how, total);
    reaching<true>(S, L, target, target);
    const Reached at = reach(std::true_type(), L.found[0], target);
    if (threadIdx.x == 0) {
        P.tokens[b] = (int32_t) ~(uint32_t) at.place;
        const double below = bins_below(r, of_key((uint32_t) (at.place >> 32)));
        if (P.probs) P.probs[b] = (float) (weight_of(below, (int) below, edge_weight((int) below)) / (double) total);
    }
}

// The values from bin `lo` to bin `hi`, and a few steps more on either side.
struct Span {
    float least, most;
    __device__ __forceinline__ bool holds(float x) const { return x >= least && x <= most; } // (no NaN)
};
__device__ __forceinline__ Span span_of(const Row &r, int lo, int hi) {
    Span s;
    s.least = float_below(r.top - (double) (hi + 1) / r.scale);
    s.most = lo == 0 ? INFINITY : -float_below((double) lo / r.scale - r.top);
    return s;
}

// Gathers the values in the bins where a cut may fall; the row's last work-group to be done finds the cuts among them and
// draws.
__global__ __launch_bounds__(kSmThreads) void sample_pick_kernel(SampleParams P) {
    __shared__ SumsLds L;
    __shared__ Search D;
    __shared__ uint32_t s_n, s_base;
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    const Settings how = settings_of(P, b);
    const Quads q = quads_of(P, b, s);
    const Ahead ahead = ahead_of(q, q.first + tid);
    const u64 best = best_of(P, b);
    if (best == 0 || how.greedy) {
        if (s == 0 && tid == 0) {
            P.tokens[b] = best == 0 ? -1 : (int32_t) ~(uint32_t) best;
            if (P.probs) P.probs[b] = best == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    if (tid == 0) s_n = 0;
    const Sums S = sums_of(P.mass + (int64_t) b * kSampleBins, P.count + (int64_t) b * kSampleBins, L);
    const Row r = row_of(how, best);
    const Cuts c = cuts_of(how, S, L);
    u64 *list = P.list + (int64_t) b * P.n_vocab;
    auto write_through = [&](uint32_t at, u64 p) { __hip_atomic_store(list + at, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const Span drawn = span_of(r, c.d_lo, c.d_hi);
    const Span ranked = c.part ? span_of(r, c.cut.bin, c.cut.bin) : drawn, run = c.by_p ? span_of(r, c.p_lo, c.p_hi) : drawn;
    each_value(q, ahead, [&](float x, int i) {
        if (!(drawn.holds(x) || ranked.holds(x) || run.holds(x))) return;
        x = fminf(x, FLT_MAX);
        const double below = bins_below(r, x);
        const int bin = (int) below;
        if (!c.holds(bin) || mass_of(r, below, bin, edge_weight(bin)) == 0) return;
        const uint32_t at = atomicAdd(&s_n, 1u);
        if (at < (uint32_t) kSmGather) D.gathered[at] = place_of(x, (uint32_t) i);
        else write_through(atomicAdd(&P.n_list[b], 1u), place_of(x, (uint32_t) i));
    });
    // one place in the list for all that fitted (a global counter's answer takes a microsecond: one each, and a wavefront that
    // meets 20 such values takes 20)
    __syncthreads();
    const uint32_t mine = min(s_n, (uint32_t) kSmGather);
    if (tid == 0 && mine > 0) s_base = atomicAdd(&P.n_list[b], mine);
    __syncthreads();
    for (uint32_t i = tid; i < mine; i += kSmThreads) write_through(s_base + i, D.gathered[i]);
    // Hand-over without an L2 write-back: the entries are device-coherent stores, complete before the work-group counts itself
    // done, and read with device-coherent loads by the one that counts last.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s_n = atomicAdd(&P.n_done[b], 1u) + 1 == (uint32_t) P.slices ? atomicAdd(&P.n_list[b], 0u) : UINT_MAX;
    __syncthreads();
    const uint32_t n = s_n;
    if (n == UINT_MAX) return;
    if (n <= (uint32_t) kSmKeep) {
        sort_gathered(r, D, (int) n, [&](int i) { return __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
        draw(P, how, b, r, c, S, L, [&](auto by_mass, const Found &f, u64 target) { return reach_sorted<by_mass>(r, D, f, (int) n, target); });
    } else {
        draw(P, how, b, r, c, S, L, [&](auto by_mass, const Found &f, u64 target) { return reach_in_list<by_mass>(r, list, D, f, n, target); });
    }
}

// A row by one work-group, in one launch: the same steps with the histogram in LDS and the row, up to kSmHeld quads a thread,
// in registers, so that it is read once. 0.7 us per 1000 values: two wavefronts a SIMD do not cover each other's waits.
__global__ __launch_bounds__(kSmThreads) void sample_row_kernel(SampleParams P) {
    __shared__ u64 s_mass[kSampleBins];
    __shared__ uint32_t s_count[kSampleBins];
    __shared__ double s_edge[kSampleBins];
    __shared__ SumsLds L;
    __shared__ Search D;
    __shared__ uint32_t s_n;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    const Settings how = settings_of(P, b);
    const Quads q = quads_of(P, b, 0);
    float4 held[kSmHeld];
#pragma unroll
    for (int i = 0; i < kSmHeld; i++) {
        const int j = tid + i * kSmThreads;
        held[i] = j < q.end ? quad_at(q, j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    auto all_values = [&](auto &&f) {
#pragma unroll
        for (int i = 0; i < kSmHeld; i++) {
            if (i * kSmThreads >= q.end) break;
            const int at = 4 * (tid + i * kSmThreads) - q.off;
            f(held[i].x, at);
            f(held[i].y, at + 1);
            f(held[i].z, at + 2);
            f(held[i].w, at + 3);
        }
    };
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        s_mass[i] = 0;
        s_count[i] = 0;
        s_edge[i] = edge_weight(i);
    }
    if (tid == 0) s_n = 0;

    float top = -INFINITY;
    int top_at = 0;
    all_values([&](float x, int i) {
        x = x > FLT_MAX ? FLT_MAX : x;
        if (x > top) { // (a NaN is not)
            top = x;
            top_at = i;
        }
    });
    u64 best = wave_max_u64(top > -INFINITY ? place_of(top, top_at) : 0);
    if (lane == 0) L.wave_mass[wv] = best;
    __syncthreads();
    for (int w = 0; w < kSmThreads / kWave; w++) best = L.wave_mass[w] > best ? L.wave_mass[w] : best;
    __syncthreads();
    if (best == 0 || how.greedy) {
        if (tid == 0) {
            P.tokens[b] = best == 0 ? -1 : (int32_t) ~(uint32_t) best;
            if (P.probs) P.probs[b] = best == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    const Row r = row_of(how, best);
    const bool ranked = how.k != UINT_MAX;
    all_values([&](float x, int) {
        if (!(x >= r.least)) return;
        const double below = bins_below(r, fminf(x, FLT_MAX));
        const int bin = (int) below;
        const u64 m = mass_of(r, below, bin, s_edge[bin]);
        if (m == 0) return;
        atomicAdd(&s_mass[bin], m);
        if (ranked) atomicAdd(&s_count[bin], 1u);
    });
    __syncthreads();
    const Sums S = sums_of(s_mass, s_count, L);
    const Cuts c = cuts_of(how, S, L);
    u64 *const list = P.list + (int64_t) b * P.n_vocab;
    auto write_through = [&](uint32_t at, u64 p) { __hip_atomic_store(list + at, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const Span drawn = span_of(r, c.d_lo, c.d_hi);
    const Span cut = c.part ? span_of(r, c.cut.bin, c.cut.bin) : drawn, run = c.by_p ? span_of(r, c.p_lo, c.p_hi) : drawn;
    all_values([&](float x, int i) {
        if (!(drawn.holds(x) || cut.holds(x) || run.holds(x))) return;
        x = fminf(x, FLT_MAX);
        const double below = bins_below(r, x);
        const int bin = (int) below;
        if (!c.holds(bin) || mass_of(r, below, bin, s_edge[bin]) == 0) return;
        const uint32_t at = atomicAdd(&s_n, 1u);
        if (at < (uint32_t) kSmGather) D.gathered[at] = place_of(x, (uint32_t) i);
        else write_through(at, place_of(x, (uint32_t) i));
    });
    __syncthreads();
    const uint32_t n = s_n;
    if (n <= (uint32_t) kSmKeep) {
        sort_gathered(r, D, (int) n, [&](int i) { return D.gathered[i]; });
        draw(P, how, b, r, c, S, L, [&](auto by_mass, const Found &f, u64 target) { return reach_sorted<by_mass>(r, D, f, (int) n, target); });
    } else {
        for (int i = tid; i < kSmGather; i += kSmThreads) write_through(i, D.gathered[i]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        draw(P, how, b, r, c, S, L, [&](auto by_mass, const Found &f, u64 target) { return reach_in_list<by_mass>(r, list, D, f, n, target); });
    }
}

}  // namespace

size_t sample_plan(SampleParams &P, void *work) {
    // slices of at least 1024 quads, as many as bring the launches to kSmTarget work-groups; a row out of line has a quad more
    const int quads = (P.n_vocab + 6) / 4;
    // One work-group a row, in one launch, for rows of up to 16384 values, and where there are many for all that it can hold. Us
    // a call, so and in slices: one row of 1000 values 12 and 19, of 8192 16 and 21, of 32768 30 and 22; 256 rows of 5000 15 and
    // 30; 64 rows of 32768 32 and 31; 250 of 38000 40 and 50.
    P.by_row = quads <= kSmHeld * kSmThreads && (P.n_vocab <= 16384 || P.n_rows >= 96);
    P.slices = P.by_row ? 1 : std::max(1, std::min((quads + kSmThreads - 1) / kSmThreads, kSmTarget / std::max(1, P.n_rows)));
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
    if (P.by_row) return launch(sample_row_kernel, all, block, 0, st, nullptr, P);
    hipError_t e;
    if ((e = launch(sample_max_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    if ((e = launch(sample_bins_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    return launch(sample_pick_kernel, all, block, 0, st, nullptr, P);
}

}  // namespace lstk
