// paged_parts.h - what the kernels of attention over pages share (paged_attn.hip, paged_attn_q8.hip): the pages of a sequence, the
// equal shares of the list of pages, the partial results of a prefix that come in, and what leaves a work-group.
#pragma once

#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kPaWaves = 4;
constexpr int kPaCus = 256; // of MI355X
constexpr int kPaPerCu = 2, kPaPerCuQ8 = 3; // work-groups of equal shares per CU
constexpr int kPaLeast = 4; // pages of a share
constexpr int kPaRound = 4;  // rounds of the wavefronts up to which a share is made a whole number of them
constexpr float kLowest = -3.0e38f; // a running maximum that any score replaces
// The running maximum m that is kept lies 15 below the largest score, so that weights reach 2^15 and fp16 holds those down to
// 2^-29 of the largest as normal numbers. Scores so large that the difference would be rounded by more than 2^-4 stay as they
// are (a weight of 2^16 would be an infinity).
constexpr float kBelow = 15.0f, kExactTo = 0x1p20f;
__device__ __forceinline__ float maximum_kept(float top) { return fabsf(top) < kExactTo ? top - kBelow : top; }

// The pages of a sequence that hold visible cells: [0, ps) and [pw, pw + count - ps).
struct Span {
    int n, lo, sink; // cells; first cell of the window; sink cells
    int ps, pw, count;
};
// Pages of n cells; n may be the largest 32-bit number.
__device__ __forceinline__ int pages_of(int n) { return n / kPageCells + (n % kPageCells != 0); }
// Pages that a sequence has in the list: one at least, so that one without any is written (zeros) like the others.
__device__ __forceinline__ int listed(const Span &s) { return max(1, s.count); }
__device__ __forceinline__ Span span_of(const PagedAttnParams &P, int len) {
    Span s;
    s.n = max(0, min(len, P.max_len));
    s.lo = P.window > 0 && s.n > P.window ? s.n - P.window : 0;
    s.sink = min(P.n_sink, s.lo);
    s.pw = s.lo / kPageCells;
    s.ps = min(pages_of(s.sink), s.pw);
    s.count = s.ps + pages_of(s.n) - s.pw;
    return s;
}

// The cells of a page that are visible, bit i for cell i0 + i.
__device__ __forceinline__ unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ unsigned visible_cells(const Span &s, int i0) {
    return bits_below(s.n - i0) & (~bits_below(s.lo - i0) | bits_below(s.sink - i0));
}

// K and V are read once a call, with the non-temporal hint: 128 sequences (1.2 GB) 225 us without it, 205 with it on one of the
// two, 200 on both; two of 100000 cells 89, 82 and 79.
__device__ __forceinline__ uint4 read_once(const char *p) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ half8v halves(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_bit_cast(half8v, make_uint4(a, b, c, d));
}
__device__ __forceinline__ float4v mfma(const half8v &a, const half8v &b, const float4v &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float across_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// A value that all lanes have alike, kept in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((int) v), hi = __builtin_amdgcn_readfirstlane((int) (v >> 32));
    return (int64_t) ((uint64_t) hi << 32 | lo);
}

// The share of a work-group in the list: `left` pages from page j of task `task` of sequence b on. The sequences' lengths and
// first table entries stay in LDS where they fit, so that the way to the first page is one wait for them and not three.
constexpr int kPaKept = kPaWaves * kWave;
struct Share {
    int b, task, j;
    int64_t left, each, total; // each: pages of a full share; total: of the list
};
struct Kept {
    int len[kPaKept], first[kPaKept];
};
__device__ __forceinline__ Share share_of(const PagedAttnParams &P, int tasks, Kept &K) {
    __shared__ int64_t s_sum[kPaWaves], s_before;
    __shared__ int s_b;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid / kWave;
    int64_t sum = 0;
    int mine = 0; // pages of sequence tid, and of the last one of every kPaKept
    for (int b = tid; b < P.n_seq; b += kPaKept) {
        const int len = P.len[b];
        if (P.n_seq <= kPaKept) {
            K.len[tid] = len;
            K.first[tid] = P.first[b];
        }
        mine = listed(span_of(P, len));
        sum += mine;
    }
    for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d, kWave);
    if (lane == 0) s_sum[wv] = sum;
    __syncthreads();
    Share s;
    s.total = 0;
    for (int w = 0; w < kPaWaves; w++) s.total += s_sum[w];
    s.total = uniform(s.total * tasks);
    // Small shares are whole rounds of the wavefronts, so that few sequences have fewer parts to join. Us a call so and without, with
    // room for 131072 cells: one sequence of 5000 cells 14.1 and 15.9, four of 200 to 3000 at 64 heads on 4 13.8 and 15.8; but 24
    // of 100 to 1500 18.4 and 16.8, 24 of 45 to 500 at 16 on 2 of 256 17.1 and 14.5; larger calls differ by 2% or less. Over the 8-bit
    // cache, whose work-groups are three a CU: 14.1 and 16.9, 14.0 and 16.1, 17.2 and 17.2, 18.6 and 16.4; 24 of 100 to 4100 with no
    // spare room 23.5 and 22.2 (9 pages a share become 12, and a third of the work-groups have none); larger calls differ by 1%.
    s.each = (s.total + gridDim.x - 1) / gridDim.x;
    if (s.each <= kPaRound * kPaWaves) s.each = (s.each + kPaWaves - 1) / kPaWaves * kPaWaves;
    const int64_t lo = s.each * blockIdx.x;
    s.each = uniform(s.each);
    s.left = uniform(min(s.each, s.total - lo));
    if (s.left <= 0) return s;
    // the sequence that page `lo` of the list is of
    int64_t before = 0; // of the sequences so far
    for (int b0 = 0; b0 < P.n_seq; b0 += kPaKept) {
        const int b = b0 + tid;
        if (P.n_seq > kPaKept) mine = b < P.n_seq ? listed(span_of(P, P.len[b])) : 0;
        int64_t upto = mine;
        for (int d = 1; d < kWave; d *= 2) {
            const int64_t o = __shfl_up(upto, d, kWave);
            if (lane >= d) upto += o;
        }
        __syncthreads();
        if (lane == kWave - 1) s_sum[wv] = upto;
        __syncthreads();
        upto += before;
        for (int i = 0; i < wv; i++) upto += s_sum[i];
        if ((upto - mine) * tasks <= lo && lo < upto * tasks) {
            s_b = b;
            s_before = upto - mine;
        }
        for (int i = 0; i < kPaWaves; i++) before += s_sum[i];
        if (lo < before * tasks) break;
    }
    __syncthreads();
    s.b = __builtin_amdgcn_readfirstlane(s_b);
    const int64_t into = lo - s_before * tasks;
    const int count = listed(span_of(P, P.n_seq <= kPaKept ? K.len[s.b] : P.len[s.b]));
    s.task = __builtin_amdgcn_readfirstlane((int) (into / count));
    s.j = __builtin_amdgcn_readfirstlane((int) (into - (int64_t) s.task * count));
    return s;
}

// What parts of a prefix left (P.pre) for four dims of a head, kPreAhead parts at a time. Up to kPreMost parts are joined where a task
// is done, more of them (or where a task is done in parts) by the launch that joins parts: it has more threads for a head.
constexpr int kPreAhead = 4, kPreMost = 8;
__host__ __device__ inline bool joins_at_once(const PagedAttnParams &P) { return P.n_wg == 0 && P.n_pre > 0 && P.n_pre <= kPreMost; }
template <int HD>
struct PrefixParts {
    float2 ml[kPreAhead];
    float4v o[kPreAhead];
    __device__ __forceinline__ void ask(const PagedAttnParams &P, int64_t head, int d, int c0) {
#pragma unroll
        for (int i = 0; i < kPreAhead; i++) {
            const float *p = P.pre + ((int64_t) min(c0 + i, P.n_pre - 1) * P.n_seq * P.n_head + head) * (HD + 4);
            ml[i] = *reinterpret_cast<const float2 *>(p);
            o[i] = *reinterpret_cast<const float4v *>(p + 4 + d);
        }
    }
    // Joined to sums l and a at maximum m.
    __device__ __forceinline__ void join(const PagedAttnParams &P, int c0, float &m, float &l, float4v &a) const {
        float top = m;
#pragma unroll
        for (int i = 0; i < kPreAhead; i++) top = fmaxf(top, ml[i].x);
        const float f = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f;
        a *= f;
#pragma unroll
        for (int i = 0; i < kPreAhead; i++) {
            const float e = c0 + i < P.n_pre ? __builtin_amdgcn_exp2f(ml[i].x - m) : 0.0f;
            if (c0 + i < P.n_pre) { // (a part that is there twice may hold NaN)
                l = fmaf(ml[i].y, e, l);
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] = fmaf(o[i][j], e, a[j]);
            }
        }
    }
};

// What a work-group's wavefronts have of a part of a task, in LDS at one maximum, goes to `out` if it is the whole task, otherwise to
// `part`. A part that continues one of the work-group before goes to the first of the work-group's two places, one that begins a
// task to the second; a whole task whose prefix is joined later goes behind the prefix's parts. With PRE the parts of a prefix are
// joined to the task before; `ahead` holds the first of them for the thread's first place.
template <int HD, bool SPLIT, bool PRE>
__device__ __forceinline__ void write_part(const PagedAttnParams &P, int b, int g, int rb, bool begins, bool whole, const float (*s_m)[16],
                                           const float (*s_l)[16], const float (*s_o)[16][HD + 4], PrefixParts<HD> &ahead) {
    const int grp = P.n_head / P.n_kv, rows = min(grp, 16);
    const int64_t place = 2 * (int64_t) blockIdx.x + (begins ? 1 : 0);
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += kPaWaves * kWave) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        if (rb * 16 + r >= grp) continue;
        const int64_t head = (int64_t) b * P.n_head + g * grp + rb * 16 + r;
        float4v a = *reinterpret_cast<const float4v *>(&s_o[0][r][d]);
        float l = s_l[0][r];
#pragma unroll
        for (int w = 1; w < kPaWaves; w++) {
            a += *reinterpret_cast<const float4v *>(&s_o[w][r][d]);
            l += s_l[w][r];
        }
        float m = s_m[0][r];
#pragma unroll
        for (int w = 1; w < kPaWaves; w++) m = fmaxf(m, s_m[w][r]);
        if constexpr (PRE) {
            for (int c0 = 0; c0 < P.n_pre; c0 += kPreAhead) {
                if (c0 > 0 || i != (int) threadIdx.x) ahead.ask(P, head, d, c0);
                ahead.join(P, c0, m, l, a);
            }
        }
        const bool behind = !PRE && whole && P.n_pre > 0;
        if ((!SPLIT || whole) && !behind) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l; // no visible cell: zeros
            ushort4 h;
            h.x = __half_as_ushort(__float2half_rn(a.x * inv));
            h.y = __half_as_ushort(__float2half_rn(a.y * inv));
            h.z = __half_as_ushort(__float2half_rn(a.z * inv));
            h.w = __half_as_ushort(__float2half_rn(a.w * inv));
            *reinterpret_cast<ushort4 *>(P.out + head * HD + d) = h;
        } else {
            float *dst = behind ? P.pre + ((int64_t) P.n_pre * P.n_seq * P.n_head + head) * (HD + 4) : P.part + (place * rows + r) * (HD + 4);
            *reinterpret_cast<float4v *>(dst + 4 + d) = a;
            if (d == 0) {
                dst[0] = m;
                dst[1] = l;
            }
        }
    }
}
// The first parts of a prefix for a thread's first place in write_part, asked for before the wavefronts meet.
template <int HD>
__device__ __forceinline__ void ask_first(const PagedAttnParams &P, int b, int g, int rb, PrefixParts<HD> &ahead) {
    const int grp = P.n_head / P.n_kv, r = threadIdx.x / (HD / 4);
    if (rb * 16 + r < grp) ahead.ask(P, (int64_t) b * P.n_head + g * grp + rb * 16 + r, 4 * (threadIdx.x % (HD / 4)), 0);
}

}  // namespace
}  // namespace lstk
