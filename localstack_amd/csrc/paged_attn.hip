// paged_attn.hip - attention of one new token per sequence over the paged fp16 cache (forward.h's cell layouts).
//
//   out[b][h] = sum_i p_i v_i / sum_i p_i,  p_i = 2^(s_i - m),  s_i = scale log2(e) q.k_i  over the visible cells i of b
//
// with the running maximum m and sum of a softmax taken in one pass. The work is a list of pages, task after task, a task being
// a (sequence, block of 16 query heads, KV head). Every work-group takes an equal share of that list (paged_attn_plan says how
// many work-groups), so a long sequence beside short ones costs no more than its pages; where a task does not end with the
// share, its parts meet in paged_attn_join_kernel. Short calls give each task a work-group and need no second launch. The
// wavefronts of a work-group take a task's pages in turn, each with its own m, sum and output, and join them in LDS.
//
// Bound by HBM: a visible cell is 4 HD bytes a KV head and 4 HD flops a query head. Measured on MI355X, 128 sequences of 1000 to
// 8192 cells at 32 heads on 4 of 128 (1.21 GB): 196 us, 6.2 TB/s, where a reading sum over 2 GiB reaches 6.2; two of 100000 cells
// at 64 on 4 (410 MB) 75 us. Short calls are bound by the way to the first page (length, first table entry, block number, K:
// four waits on memory, 4.4 us in all) and, split, by the second launch (4 to 6 us).
//
// A page (32 cells) costs a wavefront 2 HD / 32 16 x 16 x 32 fp16 matrix instructions for S^T = K Q^T and twice as many for
// O^T += V^T P^T (P as a sum of two fp16 parts, like the attention of steps of one sequence: 0.2% of the time of 128 sequences,
// 4% of 64 short ones'), every operand as the cache holds it: a lane's 16-byte load of K is 4 dims of two neighbouring cells, so one
// load feeds the tile of the even and that of the odd cells, and the two results leave a lane with 8 consecutive cells of one
// query head, which is its share of the second product's operand P. Nothing goes through LDS between the products. V
// likewise: 4 cells of two neighbouring dims.
#include "batch.h"
#include "device.h"

namespace lstk {
namespace {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kPaWaves = 4;
constexpr int kPaCus = 256; // of MI355X
constexpr int kPaPerCu = 2; // work-groups of equal shares per CU
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
    // of 100 to 1500 18.4 and 16.8, 24 of 45 to 500 at 16 on 2 of 256 17.1 and 14.5; larger calls differ by 2% or less.
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

// SPLIT: equal shares of the list; otherwise a task each.
template <int HD, bool SPLIT>
__global__ __launch_bounds__(kPaWaves *kWave, HD == 64 ? 4 : HD == 128 ? 3 : 2) void paged_attn_kernel(PagedAttnParams P) {
    constexpr int NK = HD / 16, NM = HD / 32; // 16-byte K loads of a lane per page; matrix steps over the dims
    __shared__ float s_m[kPaWaves][16], s_l[kPaWaves][16];
    __shared__ __align__(16) float s_o[kPaWaves][16][HD + 4];
    __shared__ uint4 s_q[NM][kWave];
    const int tasks = P.n_kv * P.n_rowblk;
    __shared__ Kept K;
    Share share;
    if constexpr (SPLIT) {
        share = share_of(P, tasks, K);
        if (share.left <= 0) return;
    } else {
        share.b = blockIdx.x / tasks;
        share.task = blockIdx.x % tasks;
        share.j = 0;
    }
    const int tid = threadIdx.x, lane = tid & (kWave - 1), col = lane & 15, g4 = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int grp = P.n_head / P.n_kv, rows = min(grp, 16);
    for (;;) {
        const int b = share.b, g = share.task % P.n_kv, rb = share.task / P.n_kv, row = rb * 16 + col;
        const bool kept = SPLIT && P.n_seq <= kPaKept;
        const Span sp = span_of(P, kept ? __builtin_amdgcn_readfirstlane(K.len[b]) : P.len[b]);
        const int count = listed(sp), j0 = share.j, j1 = SPLIT ? (int) min((int64_t) count, j0 + share.left) : count;

        // the operand Q^T: head `col`, dims 16 i + 4 g4 .. + 3 of steps i = 2 m, 2 m + 1. Kept in LDS: in registers its 16 (head
        // size 128) would leave two wavefronts to a SIMD instead of three, which calls with a work-group per task can fill
        for (int m = wv; m < NM; m += kPaWaves) {
            const uint16_t *src = P.q + ((int64_t) b * P.n_head + g * grp + min(row, grp - 1)) * HD + 4 * g4 + 32 * m;
            uint2 u = *reinterpret_cast<const uint2 *>(src), w = *reinterpret_cast<const uint2 *>(src + 16);
            if (row >= grp) u = w = make_uint2(0, 0);
            s_q[m][lane] = make_uint4(u.x, u.y, w.x, w.y);
        }
        float m_run = kLowest, l_run = 0.0f; // of head `col`; the sum of this lane's cells only
        float4v o[2 * NM];                   // o[2 t + e]: dims 32 t + 8 g4 + 2 i + e, i = 0 .. 3
#pragma unroll
        for (int t = 0; t < 2 * NM; t++) o[t] = float4v{0, 0, 0, 0};

        // The wavefront's pages are the part's pages wv, wv + 4, ..; lane l looks up the l-th of the next 64. A page that is out of
        // range reads page 0 and shows nothing.
        const int begin = j0 + wv, end = min(j1, sp.count);
        const int n_page = end > begin ? (end - begin + kPaWaves - 1) / kPaWaves : 0;
        const int64_t first = kept ? __builtin_amdgcn_readfirstlane(K.first[b]) : P.first[b];
        auto page_of = [&](int i) {
            const int j = begin + i * kPaWaves;
            return j < sp.ps ? j : sp.pw + (j - sp.ps);
        };
        auto look_up = [&](int i) {
            const int64_t at = first + page_of(i);
            const int id = i < n_page && at >= 0 && at < P.n_table ? P.blocks[at] : -1;
            return id >= 0 && id < P.kv_size / kPageCells ? id : -1;
        };
        const int seq = P.cell_seq ? P.seq[b] : 0;
        // addresses as a scalar base and a lane's 32-bit offset (kv_size <= 2^27)
        const char *const k_head = reinterpret_cast<const char *>(P.kc) + (int64_t) (g * (HD / 4)) * P.kv_size * 8;
        const char *const v_head = reinterpret_cast<const char *>(P.vc) + (int64_t) g * P.kv_size * (HD * 2);
        const unsigned k_lane = (unsigned) (g4 * (int) P.kv_size + 2 * col) * 8u, v_lane = (unsigned) (2 * g4 * HD * 8 + 16 * col);
        uint4 k[NK];
        int owner = 0;
        auto load_k = [&](int id) {
            const int64_t cell0 = (int64_t) max(id, 0) * kPageCells;
#pragma unroll
            for (int i = 0; i < NK; i++) k[i] = read_once(k_head + (cell0 + (int64_t) i * 4 * P.kv_size) * 8 + k_lane);
            if (P.cell_seq) owner = P.cell_seq[cell0 + (lane & (kPageCells - 1))];
        };
        int ids = look_up(lane), id = __builtin_amdgcn_readlane(ids, 0);
        if (n_page > 0) load_k(id);
        __syncthreads();
        for (int it = 0; it < n_page; it++) {
            const int64_t cell0 = (int64_t) max(id, 0) * kPageCells;
            uint4 v[NK];
#pragma unroll
            for (int t = 0; t < NM; t++) {
                v[2 * t] = read_once(v_head + cell0 * (HD * 2) + 256 * t + v_lane);
                v[2 * t + 1] = read_once(v_head + cell0 * (HD * 2) + HD * 8 + 256 * t + v_lane);
            }
            unsigned see = id >= 0 ? visible_cells(sp, page_of(it) * kPageCells) : 0u;
            if (P.cell_seq) see &= (unsigned) __ballot(owner == seq);
            float4v se{0, 0, 0, 0}, so{0, 0, 0, 0}; // cells 8 g4 + 2 i and + 1
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const half8v q = __builtin_bit_cast(half8v, s_q[m][lane]);
                se = mfma(halves(k[2 * m].x, k[2 * m].y, k[2 * m + 1].x, k[2 * m + 1].y), q, se);
                so = mfma(halves(k[2 * m].z, k[2 * m].w, k[2 * m + 1].z, k[2 * m + 1].w), q, so);
            }
            // the next page's K is on its way while this one's scores and V are worked on
            __builtin_amdgcn_sched_barrier(0);
            if ((it + 1) % kWave == 0) ids = look_up(it + 1 + lane);
            id = __builtin_amdgcn_readlane(ids, (it + 1) % kWave);
            if (it + 1 < n_page) load_k(id);
            __builtin_amdgcn_sched_barrier(0);
            float s[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[2 * i] = se[i] * P.scale;
                s[2 * i + 1] = so[i] * P.scale;
            }
            if (see != ~0u) {
                // the scores of cells that are not visible leave the sum, and what the cache holds there (it may be inf or NaN)
                // leaves the product
                const unsigned mine = see >> (8 * g4);
                unsigned keep[4];
#pragma unroll
                for (int e = 0; e < 8; e++) s[e] = mine >> e & 1u ? s[e] : -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    keep[e] = (mine >> (2 * e) & 1u ? 0xffffu : 0u) | (mine >> (2 * e + 1) & 1u ? 0xffff0000u : 0u);
#pragma unroll
                for (int t = 0; t < NK; t++) {
                    const unsigned k0 = keep[2 * (t & 1)], k1 = keep[2 * (t & 1) + 1];
                    v[t] = make_uint4(v[t].x & k0, v[t].y & k1, v[t].z & k0, v[t].w & k1);
                }
            }
            float top = s[0];
#pragma unroll
            for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
            top = fmaxf(m_run, maximum_kept(across_groups_max(top)));
            const float f = __builtin_amdgcn_exp2f(m_run - top);
            m_run = top;
            l_run *= f;
#pragma unroll
            for (int t = 0; t < 2 * NM; t++) o[t] *= f;
            // p = hi + lo in fp16 for the matrix products, to 2^-22 of each weight, or to 2^-40 of the largest where lo leaves
            // fp16's normal numbers; the sum takes p itself
            half8v hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = __builtin_amdgcn_exp2f(s[e] - m_run);
                hi[e] = (_Float16) p;
                lo[e] = (_Float16) (p - (float) hi[e]);
                l_run += p;
            }
            __builtin_amdgcn_sched_barrier(0); // (registers: without it four spill at head size 128)
#pragma unroll
            for (int t = 0; t < NM; t++) {
                o[2 * t] = mfma(halves(v[2 * t].x, v[2 * t].y, v[2 * t + 1].x, v[2 * t + 1].y), lo, o[2 * t]);
                o[2 * t + 1] = mfma(halves(v[2 * t].z, v[2 * t].w, v[2 * t + 1].z, v[2 * t + 1].w), lo, o[2 * t + 1]);
            }
#pragma unroll
            for (int t = 0; t < NM; t++) {
                o[2 * t] = mfma(halves(v[2 * t].x, v[2 * t].y, v[2 * t + 1].x, v[2 * t + 1].y), hi, o[2 * t]);
                o[2 * t + 1] = mfma(halves(v[2 * t].z, v[2 * t].w, v[2 * t + 1].z, v[2 * t + 1].w), hi, o[2 * t + 1]);
            }
        }

        // the wavefronts' shares at one maximum
        l_run = across_groups_sum(l_run);
        if (g4 == 0) s_m[wv][col] = m_run;
        __syncthreads();
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < kPaWaves; w++) top = fmaxf(top, s_m[w][col]);
        // a NaN among the scores is in l and o already; the maxima never hold one (fmaxf)
        const float f = __builtin_amdgcn_exp2f(m_run - top);
        if (g4 == 0) s_l[wv][col] = l_run * f;
#pragma unroll
        for (int t = 0; t < NM; t++) {
            float *dst = &s_o[wv][col][32 * t + 8 * g4];
            *reinterpret_cast<float4 *>(dst) = make_float4(o[2 * t][0] * f, o[2 * t + 1][0] * f, o[2 * t][1] * f, o[2 * t + 1][1] * f);
            *reinterpret_cast<float4 *>(dst + 4) = make_float4(o[2 * t][2] * f, o[2 * t + 1][2] * f, o[2 * t][3] * f, o[2 * t + 1][3] * f);
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == count;
        // a part that continues one of the work-group before goes to the first of the work-group's two places, one that begins a
        // task to the second
        const int64_t place = 2 * (int64_t) blockIdx.x + (j0 == 0 ? 1 : 0);
        for (int i = tid; i < 16 * (HD / 4); i += kPaWaves * kWave) {
            const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
            if (rb * 16 + r >= grp) continue;
            float4 a = *reinterpret_cast<const float4 *>(&s_o[0][r][d]);
            float l = s_l[0][r];
#pragma unroll
            for (int w = 1; w < kPaWaves; w++) {
                const float4 e = *reinterpret_cast<const float4 *>(&s_o[w][r][d]);
                a.x += e.x;
                a.y += e.y;
                a.z += e.z;
                a.w += e.w;
                l += s_l[w][r];
            }
            if (whole) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l; // no visible cell: zeros
                ushort4 h;
                h.x = __half_as_ushort(__float2half_rn(a.x * inv));
                h.y = __half_as_ushort(__float2half_rn(a.y * inv));
                h.z = __half_as_ushort(__float2half_rn(a.z * inv));
                h.w = __half_as_ushort(__float2half_rn(a.w * inv));
                *reinterpret_cast<ushort4 *>(P.out + ((int64_t) b * P.n_head + g * grp + rb * 16 + r) * HD + d) = h;
            } else {
                float *dst = P.part + (place * rows + r) * (HD + 4);
                *reinterpret_cast<float4 *>(dst + 4 + d) = a;
                if (d == 0) {
                    float m = s_m[0][r];
#pragma unroll
                    for (int w = 1; w < kPaWaves; w++) m = fmaxf(m, s_m[w][r]);
                    dst[0] = m;
                    dst[1] = l;
                }
            }
        }
        if constexpr (!SPLIT) return;
        // where this part begins a task: how many other work-groups have the rest (the last is the one whose share holds the
        // task's last page)
        if (tid == 0 && j0 == 0) {
            const int64_t last = min(share.each * (blockIdx.x + 1), share.total) - share.left + count - 1;
            P.split[(int64_t) b * tasks + share.task] = {(int) blockIdx.x, whole ? 0 : (int) (last / share.each) - (int) blockIdx.x};
        }
        share.left -= j1 - j0;
        if (share.left == 0) return;
        share.j = 0;
        if (++share.task == tasks) {
            share.task = 0;
            share.b++;
        }
        __syncthreads(); // s_m, s_l and s_o are written again
    }
}

// The parts of a task that lie in several shares: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A work-group takes NR of
// the task's heads; a thread four dims of a head, of every (kBlock / (NR HD / 4))-th part.
template <int HD, int NR>
__global__ __launch_bounds__(kBlock) void paged_attn_join_kernel(PagedAttnParams P) {
    constexpr int NQ = HD / 4, NC = kBlock / NQ / NR, kAhead = 4;
    __shared__ __align__(16) float4 s_o[NR][NC][NQ];
    __shared__ float s_l[NR][NC];
    const int tasks = P.n_kv * P.n_rowblk, b = blockIdx.x / tasks, task = blockIdx.x % tasks;
    const PagedAttnSplit d = P.split[blockIdx.x];
    if (d.more == 0) return;
    const int tid = threadIdx.x, dq = tid % NQ, rl = tid / NQ % NR, cl = tid / (NQ * NR);
    const int grp = P.n_head / P.n_kv, g = task % P.n_kv, rb = task / P.n_kv;
    const int n = d.more + 1, rows = min(grp, 16);
    const float *rest = P.part + 2 * (int64_t) d.wg * rows * (HD + 4), *first = rest + (int64_t) rows * (HD + 4);
    const int r = blockIdx.y * NR + rl;
    auto part = [&](int c) { return (c == 0 ? first : rest + (int64_t) c * 2 * rows * (HD + 4)) + min(r, rows - 1) * (HD + 4); };
    float m = kLowest, l = 0.0f;
    float4 a = make_float4(0, 0, 0, 0);
    for (int c0 = cl; c0 < n; c0 += kAhead * NC) {
        float2 ml[kAhead];
        float4 o[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float *p = part(min(c0 + i * NC, n - 1));
            ml[i] = *reinterpret_cast<const float2 *>(p);
            o[i] = *reinterpret_cast<const float4 *>(p + 4 + 4 * dq);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kAhead; i++) top = fmaxf(top, ml[i].x);
        const float f0 = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f0;
        a.x *= f0;
        a.y *= f0;
        a.z *= f0;
        a.w *= f0;
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (c0 + i * NC >= n) break;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
            l = fmaf(ml[i].y, f, l);
            a.x = fmaf(o[i].x, f, a.x);
            a.y = fmaf(o[i].y, f, a.y);
            a.z = fmaf(o[i].z, f, a.z);
            a.w = fmaf(o[i].w, f, a.w);
        }
    }
    // the threads of the same dims at one maximum
    __syncthreads();
    s_l[rl][cl] = m;
    __syncthreads();
    float top = kLowest;
#pragma unroll
    for (int i = 0; i < NC; i++) top = fmaxf(top, s_l[rl][i]);
    const float f = __builtin_amdgcn_exp2f(m - top);
    __syncthreads();
    s_o[rl][cl][dq] = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
    s_l[rl][cl] = l * f;
    __syncthreads();
    if (cl == 0 && rb * 16 + r < grp) {
        a = s_o[rl][0][dq];
        l = s_l[rl][0];
#pragma unroll
        for (int i = 1; i < NC; i++) {
            const float4 e = s_o[rl][i][dq];
            a.x += e.x;
            a.y += e.y;
            a.z += e.z;
            a.w += e.w;
            l += s_l[rl][i];
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        ushort4 h;
        h.x = __half_as_ushort(__float2half_rn(a.x * inv));
        h.y = __half_as_ushort(__float2half_rn(a.y * inv));
        h.z = __half_as_ushort(__float2half_rn(a.z * inv));
        h.w = __half_as_ushort(__float2half_rn(a.w * inv));
        *reinterpret_cast<ushort4 *>(P.out + ((int64_t) b * P.n_head + g * grp + rb * 16 + r) * HD + 4 * dq) = h;
    }
}

template <int HD>
hipError_t launch_paged_attn_hd(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    const dim3 block(kPaWaves * kWave);
    if (P.n_wg > 0) return launch(paged_attn_kernel<HD, true>, dim3(P.n_wg), block, 0, st, tm, P);
    return launch(paged_attn_kernel<HD, false>, dim3((unsigned) P.n_seq * P.n_kv * P.n_rowblk), block, 0, st, tm, P);
}

template <int HD>
hipError_t launch_paged_attn_join_hd(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    // a task of many parts takes a work-group per head, so that more threads share its parts (two sequences of 100000 tokens at
    // 64 heads in 96 parts a task: 9 us, 20 with four heads to a work-group; in 64 parts, as now, 6)
    const unsigned tasks = (unsigned) P.n_seq * P.n_kv * P.n_rowblk, rows = std::min(16, P.n_head / P.n_kv);
    if ((int64_t) tasks * 4 <= P.n_wg) return launch(paged_attn_join_kernel<HD, 1>, dim3(tasks, rows), dim3(kBlock), 0, st, tm, P);
    return launch(paged_attn_join_kernel<HD, 4>, dim3(tasks, (rows + 3) / 4), dim3(kBlock), 0, st, tm, P);
}

}  // namespace

// Entries of P.split, one per task, rounded up to 16 bytes.
static size_t split_entries(const PagedAttnParams &P) { return ((size_t) P.n_seq * P.n_kv * P.n_rowblk + 1) / 2 * 2; }

size_t paged_attn_plan(PagedAttnParams &P) {
    const int grp = P.n_head / P.n_kv;
    P.n_rowblk = (grp + 15) / 16;
    // the most pages a sequence can show: all, or the window's (cut at both ends) and the sinks'
    const int64_t all = ((int64_t) P.max_len + kPageCells - 1) / kPageCells;
    int64_t pages = all;
    if (P.window > 0) pages = std::min<int64_t>(all, (int64_t) P.window / kPageCells + 2 + ((int64_t) P.n_sink + kPageCells - 1) / kPageCells);
    const int64_t tasks = (int64_t) P.n_seq * P.n_kv * P.n_rowblk;
    P.n_wg = 0;
    // A work-group per task, in one launch, for sequences of up to 16 pages, and of up to 64 where there is a task for every CU:
    // the equal shares cost some 10 us more (their way to the first page and the second launch). Us a call at 32 heads on 4:
    // 64 sequences of 100 to 500 cells 12 and 22, 64 of 100 to 1000 18 and 26, one of 1000 15 and 14.
    if (pages <= 16 || (pages <= 64 && tasks >= kPaCus) || tasks == 0) return 0;
    // equal shares, of kPaLeast pages or more, for two work-groups a CU: all of them are there at once
    P.n_wg = (int) std::max<int64_t>(1, std::min<int64_t>(kPaCus * kPaPerCu, tasks * pages / kPaLeast));
    return split_entries(P) * sizeof(PagedAttnSplit) + (size_t) P.n_wg * 2 * std::min(grp, 16) * (P.hd + 4) * sizeof(float);
}

hipError_t launch_paged_attn(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    switch (P.hd) {
    case 64: return launch_paged_attn_hd<64>(P, st, tm);
    case 128: return launch_paged_attn_hd<128>(P, st, tm);
    case 256: return launch_paged_attn_hd<256>(P, st, tm);
    default: return hipErrorInvalidValue;
    }
}

hipError_t launch_paged_attn_join(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    if (P.n_wg <= 1) return hipSuccess;
    switch (P.hd) {
    case 64: return launch_paged_attn_join_hd<64>(P, st, tm);
    case 128: return launch_paged_attn_join_hd<128>(P, st, tm);
    case 256: return launch_paged_attn_join_hd<256>(P, st, tm);
    default: return hipErrorInvalidValue;
    }
}

void paged_attn_work(PagedAttnParams &P, void *work) {
    P.split = static_cast<PagedAttnSplit *>(work);
    P.part = reinterpret_cast<float *>(P.split + split_entries(P));
}

}  // namespace lstk
