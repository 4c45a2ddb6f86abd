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
#include "paged_parts.h"

namespace lstk {
namespace {

// SPLIT: equal shares of the list; otherwise a task each. PRE: the parts of a prefix are joined to a task (otherwise a
// later launch does it).
template <int HD, bool SPLIT, bool PRE>
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
    const int grp = P.n_head / P.n_kv;
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

        PrefixParts<HD> ahead;
        if constexpr (PRE) ask_first(P, b, g, rb, ahead);
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
        write_part<HD, SPLIT, PRE>(P, b, g, rb, j0 == 0, whole, s_m, s_l, s_o, ahead);
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

// The parts of a task that lie in several shares, and those of a prefix: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A work-group takes NR of
// the task's heads; a thread four dims of a head, of every (kBlock / (NR HD / 4))-th part.
template <int HD, int NR>
__global__ __launch_bounds__(kBlock) void paged_attn_join_kernel(PagedAttnParams P) {
    constexpr int NQ = HD / 4, NC = kBlock / NQ / NR, kAhead = 4;
    __shared__ __align__(16) float4 s_o[NR][NC][NQ];
    __shared__ float s_l[NR][NC];
    const int tasks = P.n_kv * P.n_rowblk, b = blockIdx.x / tasks, task = blockIdx.x % tasks;
    const PagedAttnSplit d = P.n_wg > 0 ? P.split[blockIdx.x] : PagedAttnSplit{0, 0};
    if (d.more == 0 && P.n_pre == 0) return;
    const int tid = threadIdx.x, dq = tid % NQ, rl = tid / NQ % NR, cl = tid / (NQ * NR);
    const int grp = P.n_head / P.n_kv, g = task % P.n_kv, rb = task / P.n_kv;
    const int own = d.more == 0 ? 0 : d.more + 1, n = own + P.n_pre + (d.more == 0), rows = min(grp, 16); // (a whole task: behind the prefix's)
    const float *rest = P.part + 2 * (int64_t) d.wg * rows * (HD + 4), *first = rest + (int64_t) rows * (HD + 4);
    const int r = blockIdx.y * NR + rl;
    const float *pre = P.pre + ((int64_t) b * P.n_head + g * grp + min(rb * 16 + r, grp - 1)) * (HD + 4);
    auto part = [&](int c) {
        if (c >= own) return pre + (int64_t) (c - own) * P.n_seq * P.n_head * (HD + 4);
        return (c == 0 ? first : rest + (int64_t) c * 2 * rows * (HD + 4)) + min(r, rows - 1) * (HD + 4);
    };
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
    const dim3 block(kPaWaves * kWave), all(P.n_wg > 0 ? P.n_wg : (unsigned) P.n_seq * P.n_kv * P.n_rowblk);
    if (P.n_wg > 0) return launch(paged_attn_kernel<HD, true, false>, all, block, 0, st, tm, P);
    return joins_at_once(P) ? launch(paged_attn_kernel<HD, false, true>, all, block, 0, st, tm, P)
                            : launch(paged_attn_kernel<HD, false, false>, all, block, 0, st, tm, P);
}

template <int HD>
hipError_t launch_paged_attn_join_hd(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    // a task of many parts takes a work-group per head, so that more threads share its parts (two sequences of 100000 tokens at
    // 64 heads in 96 parts a task: 9 us, 20 with four heads to a work-group; in 64 parts, as now, 6)
    const unsigned tasks = (unsigned) P.n_seq * P.n_kv * P.n_rowblk, rows = std::min(16, P.n_head / P.n_kv);
    if ((int64_t) tasks * 4 <= P.n_wg + P.n_pre * (int64_t) tasks / 8) return launch(paged_attn_join_kernel<HD, 1>, dim3(tasks, rows), dim3(kBlock), 0, st, tm, P);
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
    // equal shares, of kPaLeast pages or more, for two work-groups a CU (three where they take half the bytes and registers allow it):
    // all of them are there at once
    const int per_cu = P.in_q8 && P.hd < 256 ? kPaPerCuQ8 : kPaPerCu;
    P.n_wg = (int) std::max<int64_t>(1, std::min<int64_t>(kPaCus * per_cu, tasks * pages / kPaLeast));
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
    if (P.n_pre > 0 ? joins_at_once(P) : P.n_wg <= 1) return hipSuccess;
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
