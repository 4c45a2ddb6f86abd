// prefix_attn.hip - attention of the query tokens of many sequences over the cells that all of them share (a prompt).
//
// For a KV head the queries of all sequences are the rows of one matrix product with the shared cells, so K and V are read once a
// row block and not once a sequence:
//   S^T = K Q^T,  p = 2^(s - m),  O^T += V^T P^T,  l += sum p       (m: a row's running reference, s in units of log 2)
// over a share of the prefix's pages; what a share leaves (m, l, O) goes to `part` and is joined where a sequence's own cells are
// done (write_part, paged_parts.h) or by the launch that joins parts.
//
// A page (32 cells) is the A operand of 32 x 32 x 16 fp16 matrix instructions, 32 query rows the B operand: HD / 16 of them for S^T,
// twice as many for O^T, whose P enters as two fp16 parts. Their results leave a lane with 16 cells of one row, 8 in a row of each half
// of the page, which is what it needs of the operand P: nothing is moved between the products. One part a
// weight took 101 us where two take 121 (the long prefix below), but is off by 2^-12 of the weight and not 2^-22, which values that nearly
// cancel bring out.
//
// Many rows: four wavefronts (128 rows) share a page in LDS, two such groups a work-group, two pages a turn; few rows (up to 64): each
// wavefront takes a page of its own from memory to registers. Measured on MI355X at 1024 rows a KV head, 4 KV heads of 128: 8000 cells 43
// us, 30001 121 us (520 TFLOP/s of the sums' flops; some 15 us of it are the way to the first page and 17 MB of parts). Of 217 k busy cycles
// there the vector units take 93 k, the matrix units 91 k and LDS (16 KB a wavefront and page, at 280 bytes a ns and CU) 78 k: the three
// hardly overlap, with two wavefronts a SIMD or three, in step or not. The work-groups of the same pages run on one XCD, whose L2 then has
// 86% of the reads.
#include <type_traits>

#include "device.h"
#include "paged_parts.h"

namespace lstk {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kPxRows = 32;   // query rows of a wavefront
constexpr int kPxTiles = 4;   // wavefronts that share a page
// Groups of such wavefronts, a page at a time each. Head size 256 has one, with all registers of a SIMD to each wavefront.
template <int HD>
constexpr int px_groups() { return HD == 256 ? 1 : 2; }
// The reference m lies kPxUnder below the row's largest score when it is set, and is set anew when a score lies more than kPxUnder +
// kPxSlack above it: weights stay below 2^16, the largest at 2^12 or more, so that half a step of fp16's subnormal numbers (2^-25) is
// 2^-37 of it or less.
constexpr float kPxUnder = 12.0f, kPxSlack = 3.9f;

__device__ __forceinline__ float16v mfma32(const half8v &a, const half8v &b, const float16v &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half8v pair(const uint2 &a, const uint2 &b) { return halves(a.x, a.y, b.x, b.y); }

template <int HD, bool SHARED>
constexpr int px_waves() { return SHARED ? kPxTiles * px_groups<HD>() : HD == 256 ? 4 : 8; }

template <int HD, bool SHARED>
__global__ __launch_bounds__((px_waves<HD, SHARED>()) * kWave, HD < 256 ? 2 : 1) void prefix_attn_kernel(PrefixAttnParams P) {
    constexpr int W = px_waves<HD, SHARED>(), G = SHARED ? px_groups<HD>() : W, NT = SHARED ? kPxTiles : 1; // page groups, row tiles
    constexpr int NS = HD / 16, ND = HD / 32;                                                        // steps over the dims; dim tiles
    constexpr int kBytes = HD * 64, kPages = SHARED && HD < 256 ? 2 : 1; // of K, and of V, of a page; pages of a turn
    // SHARED: [2 buffers][G][kPages][K | V]; then what W / 2 wavefronts have, [W / 2][HD / 4][32 rows] float4
    constexpr int kRoom = std::max(SHARED ? 2 * G * kPages * 2 * kBytes : 0, W / 2 * HD * kPxRows * 4);
    __shared__ __align__(16) char s_mem[kRoom];
    __shared__ float s_m[W][kPxRows], s_l[W][kPxRows];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), col = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(tid / kWave), tile = wv % NT, group = wv / NT;

    // work-groups of the same pages on the same XCD, one after the other
    const int xcd = blockIdx.x % 8, at = blockIdx.x / 8, pair_no = at / P.n_rowblk * 8 + xcd, rowblk = at % P.n_rowblk;
    if (pair_no >= P.n_chunk * P.n_kv) return;
    const int g = pair_no % P.n_kv, chunk = pair_no / P.n_kv, grp = P.n_head / P.n_kv, n_rows = P.n_seq * grp;
    const int row = (rowblk * NT + tile) * kPxRows + col, rc = min(row, n_rows - 1);
    const int64_t head = (int64_t) (rc / grp) * P.n_head + g * grp + rc % grp; // of all heads of all sequences

    // Q^T: row `col`, dims 16 i + 4 h + 0 .. 3 and 16 i + 8 + 4 h + 0 .. 3; with its sign turned where the scale is negative
    half8v q[NS];
    const unsigned turn = P.scale < 0.0f ? 0x80008000u : 0u;
    const float scale = fmaxf(fabsf(P.scale), 1e-38f); // (a zero would make NaN of the -inf of cells that are not visible)
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const uint16_t *src = P.q + head * HD + 16 * i + 4 * h;
        uint2 a = *reinterpret_cast<const uint2 *>(src), b = *reinterpret_cast<const uint2 *>(src + 8);
        q[i] = halves(a.x ^ turn, a.y ^ turn, b.x ^ turn, b.y ^ turn);
    }
    float minus = -1.0f; // kept from the compiler: p - hi is one instruction as an fma of fp16 numbers, three as a difference
    asm("" : "+v"(minus));
    float m_run = kLowest, l_run = 0.0f; // of row `col`; the sum of this lane's cells
    float16v o[ND];                      // o[t][i]: dim 32 t + 8 (i / 4) + 4 h + i % 4
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = 0.0f;

    const int len = max(0, min(P.len[0], P.max_len)), pages = pages_of(len), each = (pages + P.n_chunk - 1) / P.n_chunk;
    const int begin = min(pages, chunk * each), end = min(pages, begin + each);
    const int n_it = (end - begin + G * kPages - 1) / (G * kPages); // turns of kPages pages
    auto page_at = [&](int i) { return begin + i * G + group; };      // this group's page i
    auto look_up = [&](int i) {                                       // its number; -1: none
        const int j = page_at(i);
        const int id = j < end && j < P.n_table ? P.blocks[j] : -1;
        return id >= 0 && id < P.kv_size / kPageCells ? id : -1;
    };
    const char *const k_head = reinterpret_cast<const char *>(P.kc) + (int64_t) (g * (HD / 4)) * P.kv_size * 8;
    const char *const v_head = reinterpret_cast<const char *>(P.vc) + (int64_t) g * P.kv_size * (HD * 2);

    // NP pages: k_of(n, i): the lane's cell of page n, dims as q[i]; v_of(n, s, t): the lane's dim of tile t, cells 16 s + 4 h + 0 .. 3
    // and 16 s + 8 + 4 h + 0 .. 3, zeros where a cell is not visible.
    auto work = [&](auto np, const unsigned *see, auto &&k_of, auto &&between, auto &&v_of) {
        constexpr int NP = decltype(np)::value;
        float16v s[NP];
#pragma unroll
        for (int n = 0; n < NP; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[n][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int n = 0; n < NP; n++) s[n] = mfma32(k_of(n, i), q[i], s[n]);
        between();
#pragma unroll
        for (int n = 0; n < NP; n++)
            if (see[n] != ~0u) {
                const unsigned mine = see[n] >> (4 * h); // cell of s[i]: bit 8 (i / 4) + i % 4
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = mine >> (8 * (i / 4) + i % 4) & 1u ? s[n][i] : -INFINITY;
            }
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < NP; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[n][i]);
        top = fmaxf(top, __shfl_xor(top, 32, kWave)) * scale;
        // Scores so large that they are rounded by more than 2^-4 have the largest itself for a reference.
        const bool fine = fabsf(top) < kExactTo, raise = top > m_run && !(fine && top - m_run <= kPxUnder + kPxSlack);
        if (__any(raise)) {
            const float to = !raise ? m_run : fine ? top - kPxUnder : top, f = __builtin_amdgcn_exp2f(m_run - to);
            m_run = to;
            l_run *= f;
#pragma unroll
            for (int t = 0; t < ND; t++) o[t] *= f;
        }
        // (the fma's exact product may lie above the rounded one that the reference comes from)
        if (__any(!(fabsf(m_run) < kExactTo))) {
#pragma unroll
            for (int n = 0; n < NP; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = s[n][i] * scale - m_run;
        } else {
#pragma unroll
            for (int n = 0; n < NP; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = fmaf(s[n][i], scale, -m_run);
        }
        // p = hi + lo in fp16 for the products, as over a sequence's own cells: to 2^-22 of each weight, or to 2^-37 of the largest where
        // lo leaves fp16's normal numbers; the sum takes p itself.
#pragma unroll
        for (int n = 0; n < NP; n++) {
            half8v hi[2], lo[2];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(s[n][i]), p1 = __builtin_amdgcn_exp2f(s[n][i + 1]);
                const half2v h = __builtin_convertvector(float2v{p0, p1}, half2v);
                const half2v r = __builtin_convertvector(float2v{fmaf((float) h[0], minus, p0), fmaf((float) h[1], minus, p1)}, half2v);
                hi[i / 8][i % 8] = h[0];
                hi[i / 8][i % 8 + 1] = h[1];
                lo[i / 8][i % 8] = r[0];
                lo[i / 8][i % 8 + 1] = r[1];
                l_run += p0;
                l_run += p1;
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++)
#pragma unroll
                for (int t = 0; t < ND; t++) {
                    const half8v v = v_of(n, s2, t);
                    o[t] = mfma32(v, lo[s2], o[t]);
                    o[t] = mfma32(v, hi[s2], o[t]);
                }
        }
    };
    auto seen = [&](int id, int i) { return id < 0 ? 0u : bits_below(len - page_at(i) * kPageCells); };
    auto keep = [](unsigned see, int c) { return (see >> c & 1u ? 0xffffu : 0u) | (see >> (c + 1) & 1u ? 0xffff0000u : 0u); }; // cells c, c + 1

    if constexpr (SHARED) {
        // Pages go by way of registers to LDS as they lie in the cache: K [HD / 4][32 cells][4 dims], V [8][HD][4 cells]. The next
        // ones are on their way while these are worked on.
        constexpr int NP = kPages, NL = kBytes / 1024 / NT; // a wavefront's KiB of K, and of V, of a page
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        u32x4 kl[NP][NL], vl[NP][NL];
        int id[NP], next[NP];
        auto ask = [&](const int *id) {
#pragma unroll
            for (int n = 0; n < NP; n++) {
                const char *kp = k_head + (int64_t) max(id[n], 0) * (kPageCells * 8), *vp = v_head + (int64_t) max(id[n], 0) * (kPageCells * HD * 2);
#pragma unroll
                for (int c = 0; c < NL; c++) {
                    const int part = c * NT + tile; // 1 KiB: 4 quads of dims of K
                    kl[n][c] = *reinterpret_cast<const u32x4 *>(kp + (int64_t) (4 * part + lane / 16) * P.kv_size * 8 + lane % 16 * 16);
                    vl[n][c] = *reinterpret_cast<const u32x4 *>(vp + part * 1024 + lane * 16);
                }
            }
        };
        auto put = [&](const int *id, int it, int buffer) {
            char *dst = s_mem + (buffer * G + group) * NP * 2 * kBytes;
#pragma unroll
            for (int n = 0; n < NP; n++) {
                const unsigned see = seen(id[n], it * NP + n);
#pragma unroll
                for (int c = 0; c < NL; c++) {
                    const int part = c * NT + tile;
                    u32x4 v = vl[n][c];
                    if (see != ~0u) {
                        // what the cache holds in cells that are not visible (it may be inf or NaN) leaves the product
                        const int cell = (part * 1024 + lane * 16) / (HD * 8) * 4;
                        const unsigned k0 = keep(see, cell), k1 = keep(see, cell + 2);
                        v &= u32x4{k0, k1, k0, k1};
                    }
                    *reinterpret_cast<u32x4 *>(dst + n * 2 * kBytes + part * 1024 + lane * 16) = kl[n][c];
                    *reinterpret_cast<u32x4 *>(dst + n * 2 * kBytes + kBytes + part * 1024 + lane * 16) = v;
                }
            }
        };
        int ids = look_up(lane);
        auto ids_of = [&](int it, int *id) {
            if (it * NP % kWave == 0 && it > 0) ids = look_up(it * NP + lane);
#pragma unroll
            for (int n = 0; n < NP; n++) id[n] = __builtin_amdgcn_readlane(ids, (it * NP + n) % kWave);
        };
        ids_of(0, id);
        if (n_it > 0) {
            ask(id);
            put(id, 0, 0);
        }
        for (int it = 0; it < n_it; it++) {
            __syncthreads(); // these pages are there, and nobody reads the ones before any more
            if (it + 1 < n_it) {
                ids_of(it + 1, next);
                ask(next);
            }
            unsigned see[NP], any = 0;
#pragma unroll
            for (int n = 0; n < NP; n++) any |= see[n] = seen(id[n], it * NP + n);
            const char *src = s_mem + ((it & 1) * G + group) * NP * 2 * kBytes;
            if (any != 0)
                work(std::integral_constant<int, NP>(), see, [&](int n, int i) {
                    const char *p = src + n * 2 * kBytes + (4 * i + h) * 256 + col * 8;
                    return pair(*reinterpret_cast<const uint2 *>(p), *reinterpret_cast<const uint2 *>(p + 512));
                }, [] {}, [&](int n, int s2, int t) {
                    const char *p = src + n * 2 * kBytes + kBytes + ((4 * s2 + h) * HD + 32 * t + col) * 8;
                    return pair(*reinterpret_cast<const uint2 *>(p), *reinterpret_cast<const uint2 *>(p + 2 * HD * 8));
                });
            if (it + 1 < n_it) put(next, it + 1, (it + 1) & 1);
#pragma unroll
            for (int n = 0; n < NP; n++) id[n] = next[n];
        }
        __syncthreads(); // the pages' room is written again
    } else {
        uint2 k[2 * NS];
        auto load_k = [&](int id) {
            const char *p = k_head + (int64_t) max(id, 0) * (kPageCells * 8) + col * 8;
#pragma unroll
            for (int i = 0; i < 2 * NS; i++) k[i] = *reinterpret_cast<const uint2 *>(p + (int64_t) (2 * i + h) * P.kv_size * 8);
        };
        int ids = look_up(lane), id = __builtin_amdgcn_readlane(ids, 0);
        if (n_it > 0) load_k(id);
        for (int it = 0; it < n_it; it++) {
            uint2 v[2 * ND][2];
            const char *p = v_head + (int64_t) max(id, 0) * (kPageCells * HD * 2) + (h * HD + col) * 8;
#pragma unroll
            for (int i = 0; i < 2 * ND; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) v[i][e] = *reinterpret_cast<const uint2 *>(p + ((4 * (i & 1) + 2 * e) * HD + 32 * (i / 2)) * 8);
            const unsigned see = seen(id, it);
            if ((it + 1) % kWave == 0) ids = look_up(it + 1 + lane);
            id = __builtin_amdgcn_readlane(ids, (it + 1) % kWave);
            work(std::integral_constant<int, 1>(), &see, [&](int, int i) { return pair(k[2 * i], k[2 * i + 1]); }, [&] {
                // the next page's K is on its way while this one's scores and V are worked on
                __builtin_amdgcn_sched_barrier(0);
                if (it + 1 < n_it) load_k(id);
                __builtin_amdgcn_sched_barrier(0);
                if (see != ~0u) {
#pragma unroll
                    for (int i = 0; i < 2 * ND; i++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int c = 16 * (i & 1) + 8 * e + 4 * h;
                            v[i][e] = make_uint2(v[i][e].x & keep(see, c), v[i][e].y & keep(see, c + 2));
                        }
                }
            }, [&](int, int s2, int t) { return pair(v[2 * t + s2][0], v[2 * t + s2][1]); });
        }
    }
    l_run += __shfl_xor(l_run, 32, kWave);

    // the groups' shares, in halves
    float4 *const s_o = reinterpret_cast<float4 *>(s_mem);
#pragma unroll
    for (int n = G / 2; n >= 1; n /= 2) {
        if (group >= n && group < 2 * n) {
            if (h == 0) {
                s_m[wv][col] = m_run;
                s_l[wv][col] = l_run;
            }
            float4 *dst = s_o + (int64_t) ((group - n) * NT + tile) * (HD / 4) * kPxRows;
#pragma unroll
            for (int t = 0; t < ND; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    dst[(8 * t + 2 * i + h) * kPxRows + col] = make_float4(o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
        }
        __syncthreads();
        if (group < n) {
            const int other = (group + n) * NT + tile;
            const float m2 = s_m[other][col], top = fmaxf(m_run, m2), f = __builtin_amdgcn_exp2f(m_run - top), e = __builtin_amdgcn_exp2f(m2 - top);
            m_run = top;
            l_run = l_run * f + s_l[other][col] * e;
            const float4 *src = s_o + (int64_t) (group * NT + tile) * (HD / 4) * kPxRows;
#pragma unroll
            for (int t = 0; t < ND; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 x = src[(8 * t + 2 * i + h) * kPxRows + col];
                    o[t][4 * i] = o[t][4 * i] * f + x.x * e;
                    o[t][4 * i + 1] = o[t][4 * i + 1] * f + x.y * e;
                    o[t][4 * i + 2] = o[t][4 * i + 2] * f + x.z * e;
                    o[t][4 * i + 3] = o[t][4 * i + 3] * f + x.w * e;
                }
        }
        __syncthreads();
    }
    if (group != 0 || row >= n_rows) return;
    float *dst = P.part + ((int64_t) chunk * P.n_seq * P.n_head + head) * (HD + 4);
    if (h == 0) *reinterpret_cast<float2 *>(dst) = make_float2(m_run, l_run);
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<float4 *>(dst + 4 + 32 * t + 8 * i + 4 * h) = make_float4(o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
}

template <int HD, bool SHARED>
hipError_t launch_prefix(const PrefixAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    const unsigned pairs = ((unsigned) P.n_chunk * P.n_kv + 7) / 8 * 8;
    return launch(prefix_attn_kernel<HD, SHARED>, dim3(pairs * P.n_rowblk), dim3(px_waves<HD, SHARED>() * kWave), 0, st, tm, P);
}

template <int HD>
hipError_t launch_prefix_hd(const PrefixAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    return P.shared ? launch_prefix<HD, true>(P, st, tm) : launch_prefix<HD, false>(P, st, tm);
}

}  // namespace

size_t prefix_attn_plan(PrefixAttnParams &P) {
    const int64_t rows = (int64_t) P.n_seq * (P.n_head / P.n_kv), pages = ((int64_t) P.max_len + kPageCells - 1) / kPageCells;
    P.n_chunk = P.n_rowblk = 0;
    if (pages == 0 || rows == 0) return 0;
    P.shared = rows > 2 * kPxRows;
    const int tile = P.shared ? kPxRows * kPxTiles : kPxRows, groups = !P.shared ? (P.hd == 256 ? 4 : 8) : P.hd == 256 ? 1 : 2;
    P.n_rowblk = (int) ((rows + tile - 1) / tile);
    // a work-group a CU, with two turns of its groups at least where they share pages, and a page for each wavefront where not
    const int64_t most = std::max<int64_t>(1, kPaCus / ((int64_t) P.n_rowblk * P.n_kv));
    P.n_chunk = (int) std::max<int64_t>(1, std::min(most, pages / (P.shared ? 4 * groups : groups)));
    return (size_t) (P.n_chunk + 1) * P.n_seq * P.n_head * (P.hd + 4) * sizeof(float);
}

hipError_t launch_prefix_attn(const PrefixAttnParams &P, hipStream_t st, const LaunchTiming *tm) {
    if (P.n_chunk == 0) return hipSuccess;
    switch (P.hd) {
    case 64: return launch_prefix_hd<64>(P, st, tm);
    case 128: return launch_prefix_hd<128>(P, st, tm);
    case 256: return launch_prefix_hd<256>(P, st, tm);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lstk
