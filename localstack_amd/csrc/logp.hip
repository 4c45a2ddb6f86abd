// logp.hip - log probabilities of a given token per row of logits, the row's entropy and its largest values.
//
//   m = max x,  l = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   log p(i) = x_i - m - ln l,  entropy = ln l - t / l
//
// l is held as k + r, k values at the maximum and the sum r of the others, and ln l as log1p(k - 1 + r): beside a nearly certain token the
// others' share may be far below the last bit of 1, and is what the token's log probability and the entropy consist of.
//
// Bound by HBM where there are many rows: 1000 rows of 151936 values (608 MB) 97 us on MI355X, 6.3 TB/s, and 5 us for the join; 64 rows
// with 20 values each 15 and 6 us, one row with 5 values 5.8 and 4.7 us, bound by waits.
//
// A row is read once: a work-group holds a slice of it in registers (kLpThreads * HELD quads), so the maximum is known before the
// sums are taken, and the largest values can be looked for afterwards. The n-th largest of the threads' own maxima is a bound
// that the n largest values of the slice reach and few others do; those are gathered in LDS and put in order by counting. A row of
// several slices is joined by a second launch, a work-group a row.
#include <cfloat>
#include <type_traits>

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

typedef unsigned long long u64;

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / kWave;
constexpr int kLpHeld = 16, kLpFew = 4; // quads of a thread
constexpr int kLpSlices = 64;           // of a row: a lane each in the join
constexpr int kLpList = 1024;
constexpr int kLpTarget = 4096;         // work-groups of a launch
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kFar = -1000.0f;        // e^kFar is 0: x - m of -inf, so that 0 times it stays 0

__device__ __forceinline__ float counted(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); } // NaN: -inf
__device__ __forceinline__ unsigned key_of(float x) { // order-preserving
    const unsigned u = __float_as_uint(x + 0.0f);     // -0 and 0 are equal values
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u64 place_of(float x, unsigned i) { return (u64) key_of(x) << 32 | (unsigned) ~i; } // larger is earlier; 0: none

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ unsigned dpp_u(unsigned v) {
    return (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
    v = max(v, dpp_u<0xB1>(v));
    v = max(v, dpp_u<0x4E>(v));
    v = max(v, dpp_u<0x141>(v));
    v = max(v, dpp_u<0x140>(v));
    v = max(v, dpp_u<kDppRowBcast15, 0xA>(v));
    v = max(v, dpp_u<kDppRowBcast31, 0x8>(v));
    return (unsigned) __builtin_amdgcn_readlane((int) v, 63);
}
__device__ __forceinline__ u64 wave_place_max(u64 p) {
    const unsigned hi = wave_umax((unsigned) (p >> 32)), lo = wave_umax((unsigned) (p >> 32) == hi ? (unsigned) p : 0u);
    return (u64) hi << 32 | lo;
}
// wave_max gives rows that a DPP step leaves out a 0; here the maxima may be below it
__device__ __forceinline__ float wave_top(float v) { return of_key(wave_umax(key_of(v))); }

__device__ __forceinline__ double log_sum(double k, double r) { return log1p(k - 1.0 + r); } // ln(k + r), k >= 1
// A row's answers from its sums (m: its largest value, of which there are k).
__device__ __forceinline__ void answer(const LogpParams &P, int row, float m, double k, double r, double t, double &lse) {
    lse = m > -INFINITY ? log_sum(k, r) : 0.0;
    const float *x = P.logits + (int64_t) row * P.ld;
    const int token = P.tokens[row];
    float v = -INFINITY;
    if (token >= 0 && token < P.n_vocab) v = counted(x[token]);
    P.logp[row] = v > -INFINITY ? (float) ((double) v - (double) m - lse) : -INFINITY;
    if (P.entropy) P.entropy[row] = m > -INFINITY ? (float) (lse - t / (k + r)) : 0.0f;
}
__device__ __forceinline__ void alternative(const LogpParams &P, int row, int r, u64 place, float m, double lse) { // place 0: none
    const int64_t at = (int64_t) row * P.n_top + r;
    P.top_ids[at] = place == 0 ? -1 : (int32_t) ~(unsigned) place;
    P.top_logp[at] = place == 0 ? -INFINITY : (float) ((double) of_key((unsigned) (place >> 32)) - (double) m - lse);
}

template <int HELD>
__global__ __launch_bounds__(kLpThreads) void logp_slice_kernel(LogpParams P) {
    __shared__ float s_max[kLpThreads], s_k[kLpWaves], s_r[kLpWaves], s_t[kLpWaves];
    __shared__ unsigned s_bound, s_n;
    __shared__ u64 s_list[kLpList], s_best[kLogpMaxTop], s_place[kLpWaves];
    const int row = blockIdx.x / P.slices, slice = blockIdx.x % P.slices, tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    const float *x = P.logits + (int64_t) row * P.ld;
    // quads by the memory's alignment: value i of the row is place i + off of them
    const int off = (int) (reinterpret_cast<uintptr_t>(x) / 4 % 4), quads = (P.n_vocab + off + 3) / 4;
    const int q0 = slice * P.slice, q1 = min(quads, q0 + P.slice);
    float v[HELD][4];
    auto index = [&](int h, int e) { return 4 * (q0 + h * kLpThreads + tid) + e - off; };
#pragma unroll
    for (int h = 0; h < HELD; h++) {
        const int i = index(h, 0);
        if (q0 + h * kLpThreads + tid < q1 && i >= 0 && i + 4 <= P.n_vocab) {
            const float4 f = *reinterpret_cast<const float4 *>(x + i);
            v[h][0] = f.x;
            v[h][1] = f.y;
            v[h][2] = f.z;
            v[h][3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[h][e] = q0 + h * kLpThreads + tid < q1 && i + e >= 0 && i + e < P.n_vocab ? x[i + e] : -INFINITY;
        }
    }
    float most = -INFINITY;
#pragma unroll
    for (int h = 0; h < HELD; h++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[h][e] = counted(v[h][e]);
            most = fmaxf(most, v[h][e]);
        }
    s_max[tid] = most;
    if (tid == 0) s_n = 0;
    const float wave_most = wave_top(most);
    if (lane == 0) s_r[wv] = wave_most;
    __syncthreads();
    float m = s_r[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) m = fmaxf(m, s_r[w]);
    __syncthreads();
    float k = 0.0f, r = 0.0f, t = 0.0f;
    if (m > -INFINITY) {
#pragma unroll
        for (int h = 0; h < HELD; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = fmaxf(v[h][e] - m, kFar), w = d < 0.0f ? __builtin_amdgcn_exp2f(d * kLog2e) : 0.0f;
                r += w;
                t = fmaf(d, w, t);
            }
        if (most == m) { // few threads have any
#pragma unroll
            for (int h = 0; h < HELD; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) k += v[h][e] == m ? 1.0f : 0.0f;
        }
    }
    k = wave_sum_tree(k);
    r = wave_sum_tree(r);
    t = wave_sum_tree(t);
    if (lane == 0) {
        s_k[wv] = k;
        s_r[wv] = r;
        s_t[wv] = t;
    }
    if (P.n_top > 0 && wv == 0) {
        // the n-th largest of the threads' maxima, bit by bit; its upper 18 bits (2^-9 of it) let few more values through
        unsigned key[kLpWaves], bound = 0;
#pragma unroll
        for (int w = 0; w < kLpWaves; w++) key[w] = key_of(s_max[w * kWave + lane]);
        for (int bit = 31; bit >= 14; bit--) {
            const unsigned c = bound | 1u << bit;
            int n = 0;
#pragma unroll
            for (int w = 0; w < kLpWaves; w++) n += __popcll(__ballot(key[w] >= c));
            if (n >= P.n_top) bound = c;
        }
        if (lane == 0) s_bound = bound;
    }
    __syncthreads();
    double K = 0.0, R = 0.0, T = 0.0;
#pragma unroll
    for (int w = 0; w < kLpWaves; w++) {
        K += s_k[w];
        R += s_r[w];
        T += s_t[w];
    }
    const int64_t part = (int64_t) row * P.slices + slice;
    double lse = 0.0;
    if (tid == 0) {
        if (P.slices > 1) *reinterpret_cast<float4 *>(P.sums + 4 * part) = make_float4(m, (float) K, (float) R, (float) T);
        else answer(P, row, m, K, R, T, lse);
    }
    if (P.n_top == 0) return;
    const float bound = s_bound > key_of(-INFINITY) ? of_key(s_bound) : -INFINITY; // (keys below are those of NaN)
#pragma unroll
    for (int h = 0; h < HELD; h++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (v[h][e] >= bound && v[h][e] > -INFINITY) {
                const unsigned at = atomicAdd(&s_n, 1u);
                if (at < (unsigned) kLpList) s_list[at] = place_of(v[h][e], (unsigned) index(h, e));
            }
    if (tid < P.n_top) s_best[tid] = 0;
    __syncthreads();
    const int n = (int) s_n;
    if (n <= kLpList) {
        for (int i = tid; i < n; i += kLpThreads) {
            const u64 mine = s_list[i];
            int before = 0;
            for (int j = 0; j < n; j++) before += s_list[j] > mine;
            if (before < P.n_top) s_best[before] = mine;
        }
    } else {
        // many values alike: one after the other
        u64 last = ~0ull;
        for (int r = 0; r < P.n_top; r++) {
            u64 top = 0;
#pragma unroll
            for (int h = 0; h < HELD; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u64 p = place_of(v[h][e], (unsigned) index(h, e));
                    if (v[h][e] > -INFINITY && p < last && p > top) top = p;
                }
            top = wave_place_max(top);
            if (lane == 0) s_place[wv] = top;
            __syncthreads();
            last = 0;
#pragma unroll
            for (int w = 0; w < kLpWaves; w++) last = max(last, s_place[w]);
            if (tid == 0) s_best[r] = last;
            __syncthreads();
        }
    }
    __syncthreads();
    if (tid >= P.n_top) return;
    if (P.slices > 1) P.best[part * P.n_top + tid] = s_best[tid];
    else alternative(P, row, tid, s_best[tid], m, m > -INFINITY ? log_sum(K, R) : 0.0);
}

__global__ __launch_bounds__(kLpThreads) void logp_join_kernel(LogpParams P) {
    __shared__ u64 s_best[kLpSlices * kLogpMaxTop], s_left[kLpSlices * kLogpMaxTop], s_at[kLpSlices], s_bound;
    __shared__ double s_lse;
    __shared__ float s_m;
    __shared__ int s_n;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), n = P.n_top;
    // the slices' lists are on their way while the sums are joined
    constexpr int kEach = kLpSlices * kLogpMaxTop / kLpThreads;
    u64 list[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i++)
        if (tid + i * kLpThreads < P.slices * n) list[i] = P.best[(int64_t) row * P.slices * n + tid + i * kLpThreads];
    if (tid < kWave) {
        float4 s = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        if (lane < P.slices) s = *reinterpret_cast<const float4 *>(P.sums + 4 * ((int64_t) row * P.slices + lane));
        const float m = wave_top(s.x);
        double k = 0.0, r = 0.0, t = 0.0, lse;
        if (s.x == m) {
            k = s.y;
            r = s.z;
            t = s.w;
        } else if (s.x > -INFINITY) {
            const double d = (double) s.x - (double) m, w = exp(d);
            r = w * ((double) s.y + (double) s.z);
            t = w * s.w + d * r;
        }
        k = wave_sum_d(k);
        r = wave_sum_d(r);
        t = wave_sum_d(t);
        if (lane == 0) {
            answer(P, row, m, k, r, t, lse);
            s_lse = lse;
            s_m = m;
            s_n = 0;
        }
    }
    if (n == 0) return;
#pragma unroll
    for (int i = 0; i < kEach; i++)
        if (tid + i * kLpThreads < P.slices * n) s_best[tid + i * kLpThreads] = list[i];
    __syncthreads();
    // Element j of every slice's list, in order: the one that has q before it is no more than (q + 1) (j + 1) >= n_top values, so none
    // below it is among the n_top largest. The few that are left are put in order by counting.
    const int j = (n - 1) / P.slices, q = (n + j) / (j + 1) - 1;
    const u64 at = tid < P.slices ? s_best[tid * n + j] : 0;
    if (tid < kLpSlices) s_at[tid] = at;
    __syncthreads();
    if (tid < P.slices) {
        int before = 0;
        for (int i = 0; i < P.slices; i++) before += s_at[i] > at || (s_at[i] == at && i < tid);
        if (before == q) s_bound = at;
    }
    __syncthreads();
    const u64 bound = max(s_bound, (u64) 1);
    for (int i = tid; i < P.slices * n; i += kLpThreads)
        if (s_best[i] >= bound) s_left[atomicAdd(&s_n, 1)] = s_best[i]; // (in any order: they are counted)
    __syncthreads();
    const int left = s_n;
    for (int i = tid; i < left; i += kLpThreads) {
        const u64 place = s_left[i];
        int r = 0;
        for (int k = 0; k < left; k++) r += s_left[k] > place;
        if (r < n) alternative(P, row, r, place, s_m, s_lse);
    }
    for (int r = left + tid; r < n; r += kLpThreads) alternative(P, row, r, 0, s_m, s_lse);
}

}  // namespace

size_t logp_plan(LogpParams &P, void *work) {
    const int quads = (P.n_vocab + 6) / 4; // a row out of line has one more
    const int least = (quads + kLpHeld * kLpThreads - 1) / (kLpHeld * kLpThreads);
    const int want = std::min(kLpTarget / std::max(1, P.n_rows), (quads + kLpFew * kLpThreads - 1) / (kLpFew * kLpThreads));
    P.slices = std::min(kLpSlices, std::max({1, least, want}));
    P.slice = (quads + P.slices - 1) / P.slices;
    if (P.slices == 1) return 0;
    const size_t parts = (size_t) P.n_rows * P.slices;
    P.sums = static_cast<float *>(work);
    P.best = reinterpret_cast<unsigned long long *>(static_cast<uint8_t *>(work) + parts * 16);
    return parts * (16 + 8 * (size_t) P.n_top);
}

hipError_t launch_logp(const LogpParams &P, hipStream_t st) {
    if (P.n_rows <= 0) return hipSuccess;
    const dim3 all((unsigned) (P.n_rows * P.slices)), block(kLpThreads);
    const hipError_t e = P.slice <= kLpFew * kLpThreads ? launch(logp_slice_kernel<kLpFew>, all, block, 0, st, nullptr, P)
                                                        : launch(logp_slice_kernel<kLpHeld>, all, block, 0, st, nullptr, P);
    if (e != hipSuccess || P.slices == 1) return e;
    return launch(logp_join_kernel, dim3((unsigned) P.n_rows), block, 0, st, nullptr, P);
}

}  // namespace lstk
