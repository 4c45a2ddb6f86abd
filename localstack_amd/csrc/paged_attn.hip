// paged_attn.hip - attention of one new token per sequence over the paged fp16 cache (forward.h's cell layouts).
//
//   out[b][h] = sum_i p_i v_i / sum_i p_i,  p_i = 2^(s_i - m),  s_i = scale log2(e) q.k_i  over the visible cells i of b
//
// with the running maximum m and sum of a softmax taken in one pass. A work-group takes a chunk of the pages of one
// (sequence, KV head, block of 16 query heads); its wavefronts take the pages in turn, each with its own m, sum and output,
// and join them in LDS. Chunks of a sequence meet in paged_attn_join_kernel.
//
// A page (32 cells) costs a wavefront 2 HD / 32 16 x 16 x 32 fp16 matrix instructions for S^T = K Q^T and as many for
// O^T += V^T P^T, every operand as the cache holds it: a lane's 16-byte load of K is 4 dims of two neighbouring cells, so one
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
constexpr float kLowest = -3.0e38f; // a running maximum that any score replaces

// The pages of a sequence that hold visible cells: [0, ps) and [pw, pw + count - ps).
struct Span {
    int n, lo, sink; // cells; first cell of the window; sink cells
    int ps, pw, count;
};
__device__ __forceinline__ Span span_of(const PagedAttnParams &P, int b) {
    Span s;
    s.n = max(0, min(P.len[b], P.max_len));
    s.lo = P.window > 0 && s.n > P.window ? s.n - P.window : 0;
    s.sink = min(P.n_sink, s.lo);
    s.pw = s.lo / kPageCells;
    s.ps = min((s.sink + kPageCells - 1) / kPageCells, s.pw);
    s.count = s.ps + (s.n + kPageCells - 1) / kPageCells - s.pw;
    return s;
}

// The cells of a page that are visible, bit i for cell i0 + i.
__device__ __forceinline__ unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ unsigned visible_cells(const Span &s, int i0) {
    return bits_below(s.n - i0) & (~bits_below(s.lo - i0) | bits_below(s.sink - i0));
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

template <int HD>
__global__ __launch_bounds__(kPaWaves *kWave) void paged_attn_kernel(PagedAttnParams P) {
    constexpr int NK = HD / 16, NM = HD / 32; // 16-byte K loads of a lane per page; matrix steps over the dims
    __shared__ float s_m[kPaWaves][16], s_l[kPaWaves][16];
    __shared__ __align__(16) float s_o[kPaWaves][16][HD + 4];
    const int b = blockIdx.x / P.n_chunk, c = blockIdx.x % P.n_chunk;
    const int g = blockIdx.y % P.n_kv, rb = blockIdx.y / P.n_kv;
    const Span sp = span_of(P, b);
    const int n_chunk = (sp.count + P.chunk - 1) / P.chunk; // of this sequence
    if (c >= n_chunk && c > 0) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), col = lane & 15, g4 = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int grp = P.n_head / P.n_kv, row = rb * 16 + col;

    half8v q[NM]; // the operand Q^T: head `col`, dims 16 i + 4 g4 .. + 3 of steps i = 2 m, 2 m + 1
    {
        const uint16_t *src = P.q + ((int64_t) b * P.n_head + g * grp + min(row, grp - 1)) * HD + 4 * g4;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            uint2 a = *reinterpret_cast<const uint2 *>(src + 32 * m), e = *reinterpret_cast<const uint2 *>(src + 32 * m + 16);
            if (row >= grp) a = e = make_uint2(0, 0);
            q[m] = halves(a.x, a.y, e.x, e.y);
        }
    }
    float m_run = kLowest, l_run = 0.0f; // of head `col`; the sum of this lane's cells only
    float4v o[2 * NM];                   // o[2 t + e]: dims 32 t + 8 g4 + 2 i + e, i = 0 .. 3
#pragma unroll
    for (int t = 0; t < 2 * NM; t++) o[t] = float4v{0, 0, 0, 0};

    // The wavefront's pages are the chunk's pages wv, wv + 4, ..; lane l looks up the l-th of the next 64. A page that is out of
    // range reads page 0 and shows nothing.
    const int begin = c * P.chunk + wv, end = min((c + 1) * P.chunk, sp.count);
    const int n_page = end > begin ? (end - begin + kPaWaves - 1) / kPaWaves : 0;
    const int64_t first = P.first[b];
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
    const uint16_t *const k_lane = P.kc + ((int64_t) (g * (HD / 4) + g4) * P.kv_size + 2 * col) * 4;
    const uint16_t *const v_lane = P.vc + ((int64_t) g * P.kv_size / 4 + 2 * g4) * HD * 4 + 8 * col;
    uint4 k[NK];
    int owner = 0;
    auto load_k = [&](int id) {
        const int64_t cell0 = (int64_t) max(id, 0) * kPageCells;
#pragma unroll
        for (int i = 0; i < NK; i++) k[i] = *reinterpret_cast<const uint4 *>(k_lane + cell0 * 4 + (int64_t) i * 16 * P.kv_size);
        if (P.cell_seq) owner = P.cell_seq[cell0 + (lane & (kPageCells - 1))];
    };
    int ids = look_up(lane), id = __builtin_amdgcn_readlane(ids, 0);
    if (n_page > 0) load_k(id);
    for (int it = 0; it < n_page; it++) {
        const int64_t cell0 = (int64_t) max(id, 0) * kPageCells;
        uint4 v[NK];
#pragma unroll
        for (int t = 0; t < NM; t++) {
            v[2 * t] = *reinterpret_cast<const uint4 *>(v_lane + cell0 * HD + 128 * t);
            v[2 * t + 1] = *reinterpret_cast<const uint4 *>(v_lane + cell0 * HD + HD * 4 + 128 * t);
        }
        unsigned see = id >= 0 ? visible_cells(sp, page_of(it) * kPageCells) : 0u;
        if (P.cell_seq) see &= (unsigned) __ballot(owner == seq);
        float4v se{0, 0, 0, 0}, so{0, 0, 0, 0}; // cells 8 g4 + 2 i and + 1
#pragma unroll
        for (int m = 0; m < NM; m++) {
            se = mfma(halves(k[2 * m].x, k[2 * m].y, k[2 * m + 1].x, k[2 * m + 1].y), q[m], se);
            so = mfma(halves(k[2 * m].z, k[2 * m].w, k[2 * m + 1].z, k[2 * m + 1].w), q[m], so);
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
        top = fmaxf(m_run, across_groups_max(top));
        const float f = __builtin_amdgcn_exp2f(m_run - top);
        m_run = top;
        l_run *= f;
#pragma unroll
        for (int t = 0; t < 2 * NM; t++) o[t] *= f;
        // p rounded to fp16 for the matrix product (half a step, 2^-11 of each weight), and summed as rounded, so that the
        // weights used add up to the sum divided by
        half8v p;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = (_Float16) __builtin_amdgcn_exp2f(s[e] - m_run);
            l_run += (float) p[e];
        }
#pragma unroll
        for (int t = 0; t < NM; t++) {
            o[2 * t] = mfma(halves(v[2 * t].x, v[2 * t].y, v[2 * t + 1].x, v[2 * t + 1].y), p, o[2 * t]);
            o[2 * t + 1] = mfma(halves(v[2 * t].z, v[2 * t].w, v[2 * t + 1].z, v[2 * t + 1].w), p, o[2 * t + 1]);
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
        const int64_t head = (int64_t) b * P.n_head + g * grp + rb * 16 + r;
        if (n_chunk <= 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l; // no visible cell: zeros
            ushort4 h;
            h.x = __half_as_ushort(__float2half_rn(a.x * inv));
            h.y = __half_as_ushort(__float2half_rn(a.y * inv));
            h.z = __half_as_ushort(__float2half_rn(a.z * inv));
            h.w = __half_as_ushort(__float2half_rn(a.w * inv));
            *reinterpret_cast<ushort4 *>(P.out + head * HD + d) = h;
        } else {
            float *dst = P.part + (head * P.n_chunk + c) * (HD + 4);
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
}

// The chunks of one (sequence, head): out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c. A thread takes four dims of every
// (kBlock / (HD / 4))-th chunk; those of the same dims meet in LDS.
template <int HD>
__global__ __launch_bounds__(kBlock) void paged_attn_join_kernel(PagedAttnParams P) {
    constexpr int NQ = HD / 4, NC = kBlock / NQ, kAhead = 4;
    __shared__ __align__(16) float4 s_o[NC][NQ];
    __shared__ float s_m[kBlock / kWave], s_l[NC];
    const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, dq = tid % NQ, cl = tid / NQ;
    const Span sp = span_of(P, b);
    const int n = (sp.count + P.chunk - 1) / P.chunk;
    if (n <= 1) return; // written by the first launch
    const float *src = P.part + ((int64_t) b * P.n_head + h) * P.n_chunk * (HD + 4);
    float m = kLowest;
    for (int c = tid; c < n; c += kBlock) m = fmaxf(m, src[(int64_t) c * (HD + 4)]);
    m = wave_max(m);
    if (tid % kWave == 0) s_m[tid / kWave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float l = 0.0f;
    float4 a = make_float4(0, 0, 0, 0);
    for (int c0 = cl; c0 < n; c0 += kAhead * NC) {
        float2 ml[kAhead];
        float4 o[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float *p = src + (int64_t) min(c0 + i * NC, n - 1) * (HD + 4);
            ml[i] = *reinterpret_cast<const float2 *>(p);
            o[i] = *reinterpret_cast<const float4 *>(p + 4 + 4 * dq);
        }
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
    s_o[cl][dq] = a;
    if (dq == 0) s_l[cl] = l;
    __syncthreads();
    if (tid >= HD) return;
    float sum = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        sum += reinterpret_cast<const float *>(s_o[i])[tid];
        l += s_l[i];
    }
    P.out[((int64_t) b * P.n_head + h) * HD + tid] = __half_as_ushort(__float2half_rn(l == 0.0f ? 0.0f : sum / l));
}

template <int HD>
hipError_t launch_paged_attn_hd(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    const dim3 grid((unsigned) (P.n_seq * P.n_chunk), P.n_kv * P.n_rowblk);
    return launch(paged_attn_kernel<HD>, grid, dim3(kPaWaves * kWave), 0, st, tm, P);
}

}  // namespace

size_t paged_attn_plan(PagedAttnParams &P) {
    const int grp = P.n_head / P.n_kv;
    P.n_rowblk = (grp + 15) / 16;
    // the most pages a sequence can show: all, or the window's (cut at both ends) and the sinks'
    const int64_t all = ((int64_t) P.max_len + kPageCells - 1) / kPageCells;
    int64_t pages = all;
    if (P.window > 0) pages = std::min<int64_t>(all, (int64_t) P.window / kPageCells + 2 + ((int64_t) P.n_sink + kPageCells - 1) / kPageCells);
    // chunks of 32 pages, up to 4096 work-groups in all
    const int64_t one = std::max<int64_t>(1, (int64_t) P.n_seq * P.n_kv * P.n_rowblk);
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>((pages + 31) / 32, 4096 / one));
    P.chunk = (int) std::max<int64_t>(1, (pages + most - 1) / most);
    P.n_chunk = (int) std::max<int64_t>(1, (pages + P.chunk - 1) / P.chunk);
    // room for `most` chunks: more pages never take less, so a workspace for longer sequences serves shorter ones
    return most == 1 ? 0 : (size_t) P.n_seq * P.n_head * most * (P.hd + 4) * sizeof(float);
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
    if (P.n_chunk == 1) return hipSuccess;
    const dim3 grid(P.n_seq, P.n_head);
    switch (P.hd) {
    case 64: return launch(paged_attn_join_kernel<64>, grid, dim3(kBlock), 0, st, tm, P);
    case 128: return launch(paged_attn_join_kernel<128>, grid, dim3(kBlock), 0, st, tm, P);
    case 256: return launch(paged_attn_join_kernel<256>, grid, dim3(kBlock), 0, st, tm, P);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lstk
