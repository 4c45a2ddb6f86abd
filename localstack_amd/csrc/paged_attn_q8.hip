// paged_attn_q8.hip - attention of one new token per sequence over the quantised cache of cache_q8.h (values d q, blocks of 32 dims).
//
//   s_i = scale log2(e) sum_m d_im (q_m . k_im)      k_im: the 32 whole numbers of block m of cell i
//   o_m = sum_i (p_i d'_im) v_im,  p_i = 2^(s_i - r),  out = o / sum_i p_i
//
// List of pages, shares, parts and joins are those of attention over the fp16 cache (paged_parts.h, paged_attn_join_kernel). The
// products take the whole numbers, which fp16 holds exactly, so the scales come after the first product (one fma a score and block)
// and before the second one, in its weights; the result is that of the values d q in fp32.
//
// Bound by HBM: a visible cell is 2.125 HD bytes a KV head, half of the fp16 cache's and a bit. Measured on MI355X, 128 sequences of
// 1000 to 8192 cells at 32 heads on 4 of 128 (642 MB): 112 us, 5.7 TB/s, where a reading sum reaches 6.2; 24 of 100 to 4100 21 us and 4
// for the join. A page costs a wavefront some 410 vector instructions (160 of them make fp16 of 128 bytes a lane, 32 scale scores, 80
// make the weights' two parts), about half of the time that HBM takes, so there are three work-groups a CU where the fp16 cache's
// kernel has two (115 us, 117 with two, in the version that this was tried on). A page's scales go by way of LDS, 4 bytes a lane of
// each load: asked for by every lane that uses them they took 32 registers (145 us; 117 by way of LDS).
#include "cache_q8.h"
#include "paged_parts.h"

namespace lstk {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

// Eight signed bytes as fp16, by the well-known way of writing a small whole number into the mantissa: the byte with its sign bit
// flipped, under the exponent of 1024, is 1152 more than the number.
__device__ __forceinline__ half8v wide(unsigned a, unsigned b) {
    const half2v less = {(_Float16) 1152.0f, (_Float16) 1152.0f};
    unsigned r[4];
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    r[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(half2v, r[i]) - less);
    return halves(r[0], r[1], r[2], r[3]);
}
// Half e of eight.
__device__ __forceinline__ float half_of(const uint4 &u, int e) {
    const unsigned w = e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
    return (float) __builtin_bit_cast(half2v, w)[e & 1];
}
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { // of two pairs of halves that are not negative
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a), __builtin_bit_cast(ushort2v, b)));
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ unsigned dpp_bits(unsigned v) {
    return (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, ROWS, 0xF, false);
}
// The largest of the wavefront's halves, numbers that are not negative, as bits.
__device__ __forceinline__ unsigned most_of(unsigned v) {
    v = larger(v, dpp_bits<0xB1>(v));
    v = larger(v, dpp_bits<0x4E>(v));
    v = larger(v, dpp_bits<0x141>(v));
    v = larger(v, dpp_bits<0x140>(v));
    v = larger(v, dpp_bits<kDppRowBcast15, 0xA>(v));
    v = larger(v, dpp_bits<kDppRowBcast31, 0x8>(v));
    v = (unsigned) __builtin_amdgcn_readlane((int) v, 63);
    return max(v & 0xffffu, v >> 16);
}
// A page's scales, HD numbers of fp16: a lane's share of them on the way to LDS.
template <int HD>
struct ScaleShare {
    static constexpr int kLanes = HD == 64 ? 32 : 64, kWords = HD == 256 ? 2 : 1;
    unsigned w[kWords];
    __device__ __forceinline__ void load(const char *p, int lane) {
        if constexpr (kWords == 2) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p + 8 * lane);
            w[0] = u.x;
            w[1] = u.y;
        } else {
            w[0] = *reinterpret_cast<const unsigned *>(p + 4 * (lane % kLanes));
        }
    }
    // Of cells that are not visible: 0.
    __device__ __forceinline__ void hide(unsigned see, int lane) {
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const unsigned two = see >> ((2 * kWords * lane + 2 * i) % kPageCells);
            w[i] &= (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
        }
    }
    __device__ __forceinline__ unsigned most() const { return most_of(larger(w[0], w[kWords - 1])); }
    __device__ __forceinline__ void store(uint4 *dst, int lane) const {
        unsigned *p = reinterpret_cast<unsigned *>(dst) + kWords * (lane % kLanes);
        if constexpr (kWords == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else *p = w[0];
    }
};
// Between a wavefront's writes to LDS and its own reads of them.
__device__ __forceinline__ void lds_settled() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int HD, bool SPLIT, bool PRE>
__global__ __launch_bounds__(kPaWaves *kWave, HD == 256 ? 2 : 3) void paged_attn_q8_kernel(PagedAttnParams P) {
    constexpr int NM = HD / kQ8Dims;
    __shared__ float s_m[kPaWaves][16], s_l[kPaWaves][16];
    __shared__ __align__(16) float s_o[kPaWaves][16][HD + 4];
    __shared__ uint4 s_q[NM][kWave];
    __shared__ uint4 s_d[2][kPaWaves][NM * 4]; // a page's scales of K and of V, of each wavefront
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

        // the operand Q^T: head `col`, dims 32 m + 8 g4 .. + 7
        for (int m = wv; m < NM; m += kPaWaves) {
            const uint4 u = *reinterpret_cast<const uint4 *>(P.q + ((int64_t) b * P.n_head + g * grp + min(row, grp - 1)) * HD + 32 * m + 8 * g4);
            s_q[m][lane] = row < grp ? u : make_uint4(0, 0, 0, 0);
        }
        float minus = -1.0f; // kept from the compiler: w - hi is one instruction as an fma of fp16 numbers, four as a difference
        asm("" : "+v"(minus));
        float m_run = kLowest, l_run = 0.0f; // of head `col`; the sum of this lane's cells only
        float4v o[2 * NM];                   // o[2 m + t]: dims 32 m + 16 t + 4 g4 + 0 .. 3
#pragma unroll
        for (int t = 0; t < 2 * NM; t++) o[t] = float4v{0, 0, 0, 0};

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
        auto record = [&](int id) { return reinterpret_cast<const char *>(P.q8) + ((int64_t) max(id, 0) * P.n_kv + g) * q8_record(HD); };
        uint4 k[NM];
        ScaleShare<HD> kd;
        int owner = 0;
        auto load_k = [&](int id) {
            const char *rec = record(id);
#pragma unroll
            for (int m = 0; m < NM; m++) k[m] = read_once(rec + 1024 * m + 16 * lane);
            kd.load(rec + q8_k_scale(HD, 0, 0), lane);
            if (P.cell_seq) owner = P.cell_seq[(int64_t) max(id, 0) * kPageCells + (lane & (kPageCells - 1))];
        };
        int ids = look_up(lane), id = __builtin_amdgcn_readlane(ids, 0);
        if (n_page > 0) load_k(id);
        __syncthreads();
        for (int it = 0; it < n_page; it++) {
            const char *rec = record(id);
            uint4 v[NM];
            ScaleShare<HD> vd;
            kd.store(s_d[0][wv], lane);
            vd.load(rec + q8_v_scale(HD, 0, 0), lane);
#pragma unroll
            for (int m = 0; m < NM; m++) v[m] = read_once(rec + q8_v(HD, m, 0, 0) + 16 * lane);
            unsigned see = id >= 0 ? visible_cells(sp, page_of(it) * kPageCells) : 0u;
            if (P.cell_seq) see &= (unsigned) __ballot(owner == seq);
            lds_settled();
            float s[8]; // cells 8 g4 + 0 .. 7
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const half8v q = __builtin_bit_cast(half8v, s_q[m][lane]);
                const uint4 d8 = s_d[0][wv][4 * m + g4];
                const float4v none{0, 0, 0, 0};
                const float4v s0 = mfma(wide(k[m].x, k[m].y), q, none), s1 = mfma(wide(k[m].z, k[m].w), q, none);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = e < 4 ? s0[e] : s1[e - 4], d = half_of(d8, e);
                    s[e] = fmaf(x, d, m == 0 ? 0.0f : s[e]); // (an fma takes d as fp16, a product does not)
                }
            }
            // the next page's K is on its way while this one's scores and V are worked on
            __builtin_amdgcn_sched_barrier(0);
            if ((it + 1) % kWave == 0) ids = look_up(it + 1 + lane);
            id = __builtin_amdgcn_readlane(ids, (it + 1) % kWave);
            if (it + 1 < n_page) load_k(id);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] *= P.scale;
            if (see != ~0u) {
                // the scores of cells that are not visible leave the sum, and their scales (what is there may be inf or NaN) the product
                const unsigned mine = see >> (8 * g4);
#pragma unroll
                for (int e = 0; e < 8; e++) s[e] = mine >> e & 1u ? s[e] : -INFINITY;
                vd.hide(see, lane);
            }
            // The reference r of the weights takes the scales of V in: p d' has to stay below 2^16 as an fp16 operand whatever the
            // scales are, and as far up as it can, so that small weights keep their bits. 2^above is more than any scale of the page.
            // Among scores whose neighbours lie far apart a sum with `above` may be rounded up by a whole step, and the weights be
            // lost; there they are 1 at most, which a scale may multiply as it is.
            const int above = (int) (vd.most() >> 10) - 14;
            vd.store(s_d[1][wv], lane);
            float top = s[0];
#pragma unroll
            for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
            top = across_groups_max(top);
            top = fmaxf(m_run, fabsf(top) < kExactTo ? top + ((float) above - kBelow) : top + (float) min(above, 0));
            if (__any(top > m_run)) {
                const float f = __builtin_amdgcn_exp2f(m_run - top);
                m_run = top;
                l_run *= f;
#pragma unroll
                for (int t = 0; t < 2 * NM; t++) o[t] *= f;
            }
            lds_settled();
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = __builtin_amdgcn_exp2f(s[e] - m_run);
                l_run += p[e];
            }
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const uint4 d8 = s_d[1][wv][4 * m + g4];
                // p d' = hi + lo in fp16, as in attention over the fp16 cache
                half8v hi, lo;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float w = fmaf(p[e], half_of(d8, e), 0.0f);
                    hi[e] = (_Float16) w;
                    lo[e] = (_Float16) fmaf((float) hi[e], minus, w);
                }
                const half8v v0 = wide(v[m].x, v[m].y), v1 = wide(v[m].z, v[m].w);
                o[2 * m] = mfma(v0, lo, o[2 * m]);
                o[2 * m + 1] = mfma(v1, lo, o[2 * m + 1]);
                o[2 * m] = mfma(v0, hi, o[2 * m]);
                o[2 * m + 1] = mfma(v1, hi, o[2 * m + 1]);
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
        const float f = __builtin_amdgcn_exp2f(m_run - top);
        if (g4 == 0) s_l[wv][col] = l_run * f;
#pragma unroll
        for (int t = 0; t < 2 * NM; t++)
            *reinterpret_cast<float4 *>(&s_o[wv][col][16 * t + 4 * g4]) = make_float4(o[t][0] * f, o[t][1] * f, o[t][2] * f, o[t][3] * f);
        __syncthreads();
        const bool whole = j0 == 0 && j1 == count;
        write_part<HD, SPLIT, PRE>(P, b, g, rb, j0 == 0, whole, s_m, s_l, s_o, ahead);
        if constexpr (!SPLIT) return;
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

template <int HD>
hipError_t launch_paged_attn_q8_hd(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    const dim3 block(kPaWaves * kWave), all(P.n_wg > 0 ? P.n_wg : (unsigned) P.n_seq * P.n_kv * P.n_rowblk);
    if (P.n_wg > 0) return launch(paged_attn_q8_kernel<HD, true, false>, all, block, 0, st, tm, P);
    return joins_at_once(P) ? launch(paged_attn_q8_kernel<HD, false, true>, all, block, 0, st, tm, P)
                            : launch(paged_attn_q8_kernel<HD, false, false>, all, block, 0, st, tm, P);
}

}  // namespace

hipError_t launch_paged_attn_q8(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    switch (P.hd) {
    case 64: return launch_paged_attn_q8_hd<64>(P, st, tm);
    case 128: return launch_paged_attn_q8_hd<128>(P, st, tm);
    case 256: return launch_paged_attn_q8_hd<256>(P, st, tm);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lstk
