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
// (x_max - x) / T of the last bin's lower edge: e^-31 * 2^44 = 0.6, so everything beyond rounds to zero or one step
constexpr float kSmRange = 31.0f;

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
    float temperature, top;
    float step; // bins per unit of x
    float min_p;
};
__device__ __forceinline__ double weight_of(const Row &r, float x) {
    return x == r.top ? 1.0 : exp(((double) x - (double) r.top) / (double) r.temperature);
}
// A value's weight as a whole number; 0 for one that min-p drops. The values that min-p keeps are a run from the top, so
// the first top_k of them are those of the first top_k values that it keeps.
__device__ __forceinline__ u64 mass_of(const Row &r, float x) {
    const double w = weight_of(r, x);
    return w >= (double) r.min_p ? (u64) __double2ll_rn(w * kUnit) : 0;
}
__device__ __forceinline__ int bin_of(const Row &r, float x) {
    const float d = r.top - x;
    return d == 0.0f ? 0 : (int) fminf(d * r.step, (float) (kSampleBins - 1));
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
    r.temperature = P.temperature ? P.temperature[b] : 1.0f;
    r.top = of_key((uint32_t) (best >> 32));
    r.step = (float) kSampleBins / (kSmRange * r.temperature);
    const float p = P.min_p ? P.min_p[b] : 0.0f;
    r.min_p = p > 0.0f ? fminf(p, 1.0f) : 0.0f;
    return r;
}
__device__ __forceinline__ bool greedy(const SampleParams &P, int b) { return P.temperature && !(P.temperature[b] > 0.0f); }

// Largest value of each slice, and cleared histograms for the next launch.
__global__ __launch_bounds__(kSmThreads) void sample_max_kernel(SampleParams P) {
    __shared__ u64 s_best[kSmThreads / kWave];
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    const float *x = P.logits + (int64_t) b * P.ld;
    const int end = min(P.n_vocab, (s + 1) * P.slice);
    u64 best = 0;
    for (int i = s * P.slice + tid; i < end; i += kSmThreads) {
        const float v = value_of(x[i]);
        if (v > -INFINITY) {
            const u64 p = place_of(v, i);
            best = p > best ? p : best;
        }
    }
    for (int i = s * kSmThreads + tid; i < kSampleBins; i += P.slices * kSmThreads) {
        P.mass[(int64_t) b * kSampleBins + i] = 0;
        P.count[(int64_t) b * kSampleBins + i] = 0;
    }
    if (s == 0 && tid == 0) P.n_list[b] = 0;
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
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    if (greedy(P, b)) return;
    const u64 best = best_of(P, b);
    if (best == 0) return;
    const Row r = row_of(P, b, best);
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        s_mass[i] = 0;
        s_count[i] = 0;
    }
    __syncthreads();
    const float *x = P.logits + (int64_t) b * P.ld;
    const int end = min(P.n_vocab, (s + 1) * P.slice);
    for (int i = s * P.slice + tid; i < end; i += kSmThreads) {
        const float v = value_of(x[i]);
        if (!(v > -INFINITY)) continue;
        const u64 m = mass_of(r, v);
        if (m == 0) continue;
        const int bin = bin_of(r, v);
        atomicAdd(&s_mass[bin], m);
        atomicAdd(&s_count[bin], 1u);
    }
    __syncthreads();
    for (int i = tid; i < kSampleBins; i += kSmThreads) {
        if (s_count[i] == 0) continue;
        atomicAdd(&P.mass[(int64_t) b * kSampleBins + i], s_mass[i]);
        atomicAdd(&P.count[(int64_t) b * kSampleBins + i], s_count[i]);
    }
}

// Inclusive running sums of a row's histogram in LDS.
struct Sums {
    u64 mass[kSampleBins];
    uint32_t count[kSampleBins];
    u64 wave_mass[kSmThreads / kWave];
    uint32_t wave_count[kSmThreads / kWave];
};
__device__ __forceinline__ void sums_of(const SampleParams &P, int b, Sums &S) {
    constexpr int per = kSampleBins / kSmThreads;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    u64 m[per];
    uint32_t c[per];
    u64 ms = 0;
    uint32_t cs = 0;
    for (int i = 0; i < per; i++) {
        ms += P.mass[(int64_t) b * kSampleBins + tid * per + i];
        cs += P.count[(int64_t) b * kSampleBins + tid * per + i];
        m[i] = ms;
        c[i] = cs;
    }
    u64 im = ms;
    uint32_t ic = cs;
    for (int d = 1; d < kWave; d *= 2) {
        const u64 om = __shfl_up(im, d, kWave);
        const uint32_t oc = __shfl_up(ic, d, kWave);
        if (lane >= d) {
            im += om;
            ic += oc;
        }
    }
    if (lane == kWave - 1) {
        S.wave_mass[wv] = im;
        S.wave_count[wv] = ic;
    }
    __syncthreads();
    u64 bm = im - ms;
    uint32_t bc = ic - cs;
    for (int w = 0; w < wv; w++) {
        bm += S.wave_mass[w];
        bc += S.wave_count[w];
    }
    for (int i = 0; i < per; i++) {
        S.mass[tid * per + i] = bm + m[i];
        S.count[tid * per + i] = bc + c[i];
    }
    __syncthreads();
}
// The first bin whose running sum reaches `target` (the last bin if none does).
template <typename T>
__device__ __forceinline__ int bin_reaching(const T *sums, T target) {
    int lo = 0, hi = kSampleBins - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] >= target) hi = mid;
        else lo = mid + 1;
    }
    return lo;
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
__device__ __forceinline__ uint32_t top_k_of(const SampleParams &P, int b) {
    const int k = P.top_k ? P.top_k[b] : 0;
    return k > 0 ? (uint32_t) k : UINT_MAX;
}

// The bins where a cut may fall. The cut by rank: bin `cut`, inside it where `part` is set (else at its end). What stays, M,
// lies between the sums before and after that bin, so the run that top-p keeps ends in bins [p_lo, p_hi] (where top-p cuts at
// all), and the draw in [d_lo, d_hi].
struct Cuts {
    uint32_t k; // values that stay by rank
    bool part, by_p;
    int cut, p_lo, p_hi, d_lo, d_hi;
    __device__ __forceinline__ bool holds(int bin) const {
        return (bin >= d_lo && bin <= d_hi) || (part && bin == cut) || (by_p && bin >= p_lo && bin <= p_hi);
    }
};
__device__ __forceinline__ Cuts cuts_of(const SampleParams &P, int b, const Sums &S) {
    Cuts c;
    c.k = min(top_k_of(P, b), S.count[kSampleBins - 1]);
    c.cut = bin_reaching(S.count, c.k);
    c.part = S.count[c.cut] != c.k;
    // the largest value is in bin 0 and stays, so no sum here is 0
    const u64 m_hi = S.mass[c.cut], m_lo = !c.part ? m_hi : c.cut > 0 ? S.mass[c.cut - 1] : 1;
    u64 s_lo = m_lo, s_hi = m_hi;
    const float p = P.top_p ? P.top_p[b] : 1.0f;
    c.by_p = p < 1.0f;
    c.p_lo = c.p_hi = 0;
    if (c.by_p) {
        c.p_lo = bin_reaching(S.mass, top_p_target(P, b, m_lo));
        c.p_hi = bin_reaching(S.mass, top_p_target(P, b, m_hi));
        s_lo = c.p_lo > 0 ? S.mass[c.p_lo - 1] : 1;
        s_hi = S.mass[c.p_hi] < m_hi ? S.mass[c.p_hi] : m_hi;
    }
    c.d_lo = bin_reaching(S.mass, draw_target(P, b, s_lo));
    c.d_hi = bin_reaching(S.mass, draw_target(P, b, s_hi));
    return c;
}

// Gathers the indices of the values in the bins where a cut may fall.
__global__ __launch_bounds__(kSmThreads) void sample_collect_kernel(SampleParams P) {
    __shared__ Sums S;
    const int b = blockIdx.x / P.slices, s = blockIdx.x % P.slices, tid = threadIdx.x;
    if (greedy(P, b)) return;
    const u64 best = best_of(P, b);
    if (best == 0) return;
    const Row r = row_of(P, b, best);
    sums_of(P, b, S);
    const Cuts c = cuts_of(P, b, S);
    const float *x = P.logits + (int64_t) b * P.ld;
    const int end = min(P.n_vocab, (s + 1) * P.slice);
    for (int i = s * P.slice + tid; i < end; i += kSmThreads) {
        const float v = value_of(x[i]);
        if (v > -INFINITY && c.holds(bin_of(r, v)) && mass_of(r, v) > 0) P.list[(int64_t) b * P.n_vocab + atomicAdd(&P.n_list[b], 1u)] = i;
    }
}

// One work-group per row finds the cuts among the gathered values and draws.
struct Digits {
    u64 mass[256];
    uint32_t count[256];
    u64 place, mass_before;
    uint32_t count_before;
};
struct Reached {
    u64 place;       // of the value at which the running sum reaches the target
    u64 mass_before; // running sum before it
};
// The value of bin `bin` at which the running sum of weights (by_mass) or of values reaches `target`; `mass0` and `count0`
// are the sums of the bins before. Found a byte of the place at a time, from the highest: histogram of the byte over the
// values that share the bytes so far, then the byte in which the sum gets there.
__device__ __forceinline__ Reached reach(const SampleParams &P, int b, const Row &r, Digits &D, int bin, bool by_mass, u64 target, u64 mass0,
                         uint32_t count0) {
    const int tid = threadIdx.x;
    const uint32_t n = P.n_list[b];
    const float *x = P.logits + (int64_t) b * P.ld;
    u64 prefix = 0, mask = 0;
    if (tid == 0) {
        D.place = 0;
        D.mass_before = mass0;
        D.count_before = count0;
    }
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        prefix = D.place;
        for (int i = tid; i < 256; i += kSmThreads) {
            D.mass[i] = 0;
            D.count[i] = 0;
        }
        __syncthreads();
        for (uint32_t i = tid; i < n; i += kSmThreads) {
            const uint32_t at = P.list[(int64_t) b * P.n_vocab + i];
            const float v = value_of(x[at]);
            const u64 p = place_of(v, at);
            if (bin_of(r, v) != bin || (p & mask) != prefix) continue;
            const int digit = (int) (p >> shift & 255);
            atomicAdd(&D.mass[digit], mass_of(r, v));
            atomicAdd(&D.count[digit], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            u64 m = D.mass_before;
            uint32_t c = D.count_before;
            int digit = 255, last = 255;
            for (; digit >= 0; digit--) {
                if (D.count[digit] == 0) continue;
                last = digit;
                if (by_mass ? m + D.mass[digit] >= target : c + D.count[digit] >= target) break;
                m += D.mass[digit];
                c += D.count[digit];
            }
            if (digit < 0) { // the sums hold the target, so this is not reached
                digit = last;
                m -= D.mass[digit];
                c -= D.count[digit];
            }
            D.mass_before = m;
            D.count_before = c;
            D.place = prefix | (u64) digit << shift;
        }
        mask |= (u64) 255 << shift;
    }
    __syncthreads();
    const Reached out{D.place, D.mass_before};
    __syncthreads();
    return out;
}

__global__ __launch_bounds__(kSmThreads) void sample_pick_kernel(SampleParams P) {
    __shared__ Sums S;
    __shared__ Digits D;
    const int b = blockIdx.x, tid = threadIdx.x;
    const u64 best = best_of(P, b);
    if (best == 0 || greedy(P, b)) {
        if (tid == 0) {
            P.tokens[b] = best == 0 ? -1 : (int32_t) ~(uint32_t) best;
            if (P.probs) P.probs[b] = best == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    const Row r = row_of(P, b, best);
    sums_of(P, b, S);
    const Cuts c = cuts_of(P, b, S);
    auto mass_at = [&](u64 place) { return mass_of(r, of_key((uint32_t) (place >> 32))); };
    auto before = [&](int bin) { return bin > 0 ? S.mass[bin - 1] : 0; };
    u64 M = S.mass[c.cut];
    if (c.part) {
        const Reached at = reach(P, b, r, D, c.cut, false, c.k, before(c.cut), c.cut > 0 ? S.count[c.cut - 1] : 0);
        M = at.mass_before + mass_at(at.place);
    }
    u64 total = M;
    if (c.by_p) {
        const u64 target = top_p_target(P, b, M);
        const int bin = bin_reaching(S.mass, target);
        const Reached at = reach(P, b, r, D, bin, true, target, before(bin), 0);
        total = at.mass_before + mass_at(at.place);
    }
    const u64 target = draw_target(P, b, total);
    const int bin = bin_reaching(S.mass, target);
    const Reached at = reach(P, b, r, D, bin, true, target, before(bin), 0);
    if (tid == 0) {
        P.tokens[b] = (int32_t) ~(uint32_t) at.place;
        if (P.probs) P.probs[b] = (float) (weight_of(r, of_key((uint32_t) (at.place >> 32))) * kUnit / (double) total);
    }
}

}  // namespace

size_t sample_plan(SampleParams &P, void *work) {
    // slices of at least 4096 values, as many as bring the launches to 512 work-groups
    P.slices = std::max(1, std::min((P.n_vocab + 4095) / 4096, 512 / std::max(1, P.n_rows)));
    P.slice = (P.n_vocab + P.slices - 1) / P.slices;
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
    take(P.list, rows * P.n_vocab);
    return off;
}

hipError_t launch_sample(const SampleParams &P, hipStream_t st) {
    if (P.n_rows <= 0) return hipSuccess;
    const dim3 all((unsigned) (P.n_rows * P.slices)), block(kSmThreads);
    hipError_t e;
    if ((e = launch(sample_max_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    if ((e = launch(sample_bins_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    if ((e = launch(sample_collect_kernel, all, block, 0, st, nullptr, P)) != hipSuccess) return e;
    return launch(sample_pick_kernel, dim3(P.n_rows), block, 0, st, nullptr, P);
}

}  // namespace lstk
