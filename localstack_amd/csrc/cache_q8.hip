// cache_q8.hip - rows of K and V quantised as they are written to a cache (cache_q8.h), and read back.
//
//   d = min { fp16 numbers >= max |x| / 127 },  q = x / d to the nearest whole number, halves to the even one;  back: d q
//
// over 32 dims of a row. d is no less than a 127th of the largest, so |q| <= 127 without a clamp, and no value is off by more than
// d / 2. The 32-bit quotient only guesses q; the remainder x - q d is exact in one fma and settles it.
//
// Bound by memory, and by the launch for the rows of a decode step. A work-group takes kCrRows rows of a KV head: the whole numbers
// meet in LDS, because a row of V is single bytes 16 apart in its record. Where 8 rows fill an octet of cells, as the rows of a
// prompt do, a thread turns 4 dims of the 8 rows over in registers and moves 8 bytes a dim; the work-groups' rows are shifted so
// that the first row's octet (and with it those of the rows behind it in a prompt) begins with a work-group's rows.
// Measured on MI355X, 20000 rows of 4 heads of 128 in fp16 (63 MB in and out): store 21 us (36 with single bytes and rows where they
// lie), load 18 us; 10 us would be HBM's. A work-group is a chain of waits (the first cell, the rows, LDS), and there are 1.2 rounds
// of them.
#include "cache_q8.h"
#include "device.h"

namespace lstk {
namespace {

constexpr int kCrRows = 32;
constexpr float kMostMost = 65504.0f * 127.0f; // of a block that a finite d can hold

// Per-row cells and where 8 rows in a row fill an octet of cells: 1 at its first row, 2 at the others, 0 elsewhere.
struct Cells {
    int cell[kCrRows], octet[kCrRows]; // cell: -1 outside the cache
};
__device__ __forceinline__ void look_up_cells(const CacheRowsParams &P, Cells &C, int row0) {
    const int i = threadIdx.x;
    if (i < kCrRows) {
        const int c = row0 + i >= 0 && row0 + i < P.n ? P.cells[row0 + i] : -1;
        C.cell[i] = c >= 0 && c < P.n_cells ? c : -1;
    }
    __syncthreads();
    if (i < kCrRows) {
        const int c = C.cell[i], first = i - (c & 7);
        bool full = c >= 0 && first >= 0 && first + 8 <= kCrRows;
        for (int k = 0; k < 8 && full; k++) full = C.cell[first + k] == c - (c & 7) + k;
        C.octet[i] = full ? (first == i ? 1 : 2) : 0;
    }
    __syncthreads();
}
// The first of a work-group's rows; may be below 0.
__device__ __forceinline__ int first_row(const CacheRowsParams &P) { return (int) (blockIdx.x / P.n_kv) * kCrRows - (P.cells[0] & 7); }
// Four 4-byte words as the rows of a 4 x 4 matrix of bytes, turned over.
__device__ __forceinline__ void turn_over(unsigned (&w)[4]) {
    const unsigned a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u),
                   c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}
__device__ __forceinline__ uint8_t *record_of(const CacheRowsParams &P, int cell, int g) {
    return P.cache + ((int64_t) (cell / kPageCells) * P.n_kv + g) * q8_record(P.hd);
}

// 16 bytes of a row, as 32-bit values: N = 4 or 8 dims.
template <typename T>
constexpr int kDims = 16 / (int) sizeof(T);
template <typename T>
__device__ __forceinline__ void values_of(const uint4 &u, float (&x)[kDims<T>]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = h2f(w[i]);
            x[2 * i + 1] = h2f(w[i] >> 16);
        }
    }
}
template <typename T>
__device__ __forceinline__ void put_values(T *p, const float (&x)[kDims<T>]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
        else w[i] = (unsigned) __half_as_ushort(__float2half_rn(x[2 * i])) | (unsigned) __half_as_ushort(__float2half_rn(x[2 * i + 1])) << 16;
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// x / d to the nearest whole numbers, halves to the even one; |x| <= 127 d.
template <int N>
__device__ __forceinline__ void whole_of(const float (&x)[N], float d, float inv, int (&q)[N]) {
    float r[N], far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        r[i] = rintf(x[i] * inv);                       // within one of it, and it unless the remainder is nearly d / 2
        far = fmaxf(far, fabsf(fmaf(-r[i], d, x[i])));
    }
    if (far >= 0.4999f * d) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float rest = fmaf(-r[i], d, x[i]), half = 0.5f * d; // exact: a whole number of bits of x or of d, below 2 d
            const bool odd = ((int) r[i] & 1) != 0;
            if (rest > half || (rest == half && odd)) r[i] += 1.0f;
            else if (rest < -half || (rest == -half && odd)) r[i] -= 1.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = (int) r[i];
}

template <int HD, typename T>
__global__ __launch_bounds__(kBlock) void cache_store_kernel(CacheRowsParams P) {
    constexpr int NM = HD / kQ8Dims, N = kDims<T>, NL = kQ8Dims / N; // lanes of a block of 32 dims
    __shared__ Cells C;
    __shared__ uint32_t s_q[2][kCrRows][HD / 4 + 1]; // (+ 1: columns of V are read)
    __shared__ uint16_t s_d[2][kCrRows][NM];
    const int g = blockIdx.x % P.n_kv, row0 = first_row(P), tid = threadIdx.x;
    // all of a thread's values are on their way while the cells are looked up
    constexpr int kTurns = 2 * kCrRows * NM * NL / kBlock;
    uint4 raw[kTurns];
#pragma unroll
    for (int t = 0; t < kTurns; t++) {
        const int i = tid + t * kBlock, lane = i % NL, m = i / NL % NM, r = i / (NL * NM) % kCrRows, kind = i / (NL * NM * kCrRows);
        const int row = min(max(row0 + r, 0), P.n - 1);
        raw[t] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(kind ? P.v : P.k) + row * (kind ? P.ld_v : P.ld_k) + g * HD + 32 * m + N * lane);
    }
    look_up_cells(P, C, row0);
#pragma unroll
    for (int t = 0; t < kTurns; t++) {
        const int i = tid + t * kBlock, lane = i % NL, m = i / NL % NM, r = i / (NL * NM) % kCrRows, kind = i / (NL * NM * kCrRows);
        float x[N];
        values_of<T>(raw[t], x);
        // the largest magnitude by its bits, so that infinities and NaN are larger than any number
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < N; j++) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
        for (int d = 1; d < NL; d *= 2) most = max(most, (unsigned) __shfl_xor((int) most, d, kWave));
        unsigned bits = 0x7e00u; // NaN, for a block that holds one, an infinity or more than d can
        int q[N] = {};
        if (most <= __float_as_uint(kMostMost)) {
            const float a = __uint_as_float(most);
            bits = __half_as_ushort(__float2half_rn(a / 127.0f));
            if (h2f(bits) * 127.0f < a) bits++; // (19 bits: exact)
            const float d = h2f(bits);
            whole_of(x, d, d == 0.0f ? 0.0f : 1.0f / d, q);
        }
#pragma unroll
        for (int j = 0; j < N / 4; j++)
            s_q[kind][r][8 * m + lane * (N / 4) + j] = (q[4 * j] & 0xff) | (q[4 * j + 1] & 0xff) << 8 | (q[4 * j + 2] & 0xff) << 16 | (unsigned) q[4 * j + 3] << 24;
        if (lane == 0) s_d[kind][r][m] = (uint16_t) bits;
    }
    __syncthreads();
    // K: 8 dims of a row
    for (int i = tid; i < kCrRows * (HD / 8); i += kBlock) {
        const int r = i % kCrRows, p = i / kCrRows, cell = C.cell[r];
        if (cell < 0) continue;
        *reinterpret_cast<uint2 *>(record_of(P, cell, g) + q8_k(p / 4, cell % kPageCells, p % 4 * 8)) =
            make_uint2(s_q[0][r][2 * p], s_q[0][r][2 * p + 1]);
    }
    // V: 4 dims of a row, or of 8 rows
    for (int i = tid; i < kCrRows * (HD / 4); i += kBlock) {
        const int p = i % (HD / 4), r = i / (HD / 4), cell = C.cell[r];
        if (cell < 0 || C.octet[r] == 2) continue;
        uint8_t *dst = record_of(P, cell, g) + q8_v(HD, p / 8, cell % kPageCells, p % 8 * 4); // the dims behind it 16 apart
        if (C.octet[r] == 0) {
            const uint32_t w = s_q[1][r][p];
#pragma unroll
            for (int j = 0; j < 4; j++) dst[16 * j] = (uint8_t) (w >> (8 * j));
            continue;
        }
        unsigned lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            lo[k] = s_q[1][r + k][p];
            hi[k] = s_q[1][r + 4 + k][p];
        }
        turn_over(lo);
        turn_over(hi);
#pragma unroll
        for (int j = 0; j < 4; j++) *reinterpret_cast<uint2 *>(dst + 16 * j) = make_uint2(lo[j], hi[j]);
    }
    for (int i = tid; i < 2 * kCrRows * NM; i += kBlock) {
        const int r = i % kCrRows, m = i / kCrRows % NM, kind = i / (kCrRows * NM), cell = C.cell[r];
        if (cell < 0) continue;
        const int at = kind ? q8_v_scale(HD, m, cell % kPageCells) : q8_k_scale(HD, m, cell % kPageCells);
        *reinterpret_cast<uint16_t *>(record_of(P, cell, g) + at) = s_d[kind][r][m];
    }
}

template <int HD, typename T>
__global__ __launch_bounds__(kBlock) void cache_load_kernel(CacheRowsParams P) {
    constexpr int NM = HD / kQ8Dims, N = kDims<T>, NL = kQ8Dims / N;
    __shared__ Cells C;
    __shared__ uint32_t s_q[2][kCrRows][HD / 4 + 1];
    __shared__ uint16_t s_d[2][kCrRows][NM];
    const int g = blockIdx.x % P.n_kv, row0 = first_row(P), tid = threadIdx.x;
    look_up_cells(P, C, row0);
    constexpr int kTurns = kCrRows * (HD / 8) / kBlock;
    uint2 raw[kTurns];
#pragma unroll
    for (int t = 0; t < kTurns; t++) {
        const int i = tid + t * kBlock, r = i % kCrRows, p = i / kCrRows, cell = C.cell[r];
        raw[t] = make_uint2(0, 0);
        if (cell >= 0) raw[t] = *reinterpret_cast<const uint2 *>(record_of(P, cell, g) + q8_k(p / 4, cell % kPageCells, p % 4 * 8));
    }
    for (int i = tid; i < kCrRows * (HD / 4); i += kBlock) {
        const int p = i % (HD / 4), r = i / (HD / 4), cell = C.cell[r];
        if (C.octet[r] == 2) continue;
        if (cell < 0) {
            s_q[1][r][p] = 0;
            continue;
        }
        const uint8_t *src = record_of(P, cell, g) + q8_v(HD, p / 8, cell % kPageCells, p % 8 * 4);
        if (C.octet[r] == 0) {
            s_q[1][r][p] = (unsigned) src[0] | (unsigned) src[16] << 8 | (unsigned) src[32] << 16 | (unsigned) src[48] << 24;
            continue;
        }
        unsigned lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint2 u = *reinterpret_cast<const uint2 *>(src + 16 * j);
            lo[j] = u.x;
            hi[j] = u.y;
        }
        turn_over(lo);
        turn_over(hi);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            s_q[1][r + k][p] = lo[k];
            s_q[1][r + 4 + k][p] = hi[k];
        }
    }
    for (int i = tid; i < 2 * kCrRows * NM; i += kBlock) {
        const int r = i % kCrRows, m = i / kCrRows % NM, kind = i / (kCrRows * NM), cell = C.cell[r];
        const int at = kind ? q8_v_scale(HD, m, cell % kPageCells) : q8_k_scale(HD, m, cell % kPageCells);
        s_d[kind][r][m] = cell < 0 ? 0 : *reinterpret_cast<const uint16_t *>(record_of(P, cell, g) + at);
    }
#pragma unroll
    for (int t = 0; t < kTurns; t++) {
        const int i = tid + t * kBlock, r = i % kCrRows, p = i / kCrRows;
        s_q[0][r][2 * p] = raw[t].x;
        s_q[0][r][2 * p + 1] = raw[t].y;
    }
    __syncthreads();
    for (int i = tid; i < 2 * kCrRows * NM * NL; i += kBlock) {
        const int lane = i % NL, m = i / NL % NM, r = i / (NL * NM) % kCrRows, kind = i / (NL * NM * kCrRows), row = row0 + r;
        if (row < 0 || row >= P.n) continue;
        const float d = h2f(s_d[kind][r][m]);
        float x[N];
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = (float) (int8_t) (s_q[kind][r][8 * m + lane * (N / 4) + j / 4] >> (8 * (j % 4))) * d;
        put_values(static_cast<T *>(const_cast<void *>(kind ? P.v : P.k)) + row * (kind ? P.ld_v : P.ld_k) + g * HD + 32 * m + N * lane, x);
    }
}

template <int HD>
hipError_t launch_store_hd(const CacheRowsParams &P, dim3 grid, hipStream_t st) {
    return P.f32 ? launch(cache_store_kernel<HD, float>, grid, dim3(kBlock), 0, st, nullptr, P)
                 : launch(cache_store_kernel<HD, uint16_t>, grid, dim3(kBlock), 0, st, nullptr, P);
}
template <int HD>
hipError_t launch_load_hd(const CacheRowsParams &P, dim3 grid, hipStream_t st) {
    return P.f32 ? launch(cache_load_kernel<HD, float>, grid, dim3(kBlock), 0, st, nullptr, P)
                 : launch(cache_load_kernel<HD, uint16_t>, grid, dim3(kBlock), 0, st, nullptr, P);
}
dim3 rows_grid(const CacheRowsParams &P) { return dim3((unsigned) ((int64_t) ((P.n + 7 + kCrRows - 1) / kCrRows) * P.n_kv)); }

}  // namespace

hipError_t launch_cache_store(const CacheRowsParams &P, hipStream_t st) {
    switch (P.hd) {
    case 64: return launch_store_hd<64>(P, rows_grid(P), st);
    case 128: return launch_store_hd<128>(P, rows_grid(P), st);
    case 256: return launch_store_hd<256>(P, rows_grid(P), st);
    default: return hipErrorInvalidValue;
    }
}

hipError_t launch_cache_load(const CacheRowsParams &P, hipStream_t st) {
    switch (P.hd) {
    case 64: return launch_load_hd<64>(P, rows_grid(P), st);
    case 128: return launch_load_hd<128>(P, rows_grid(P), st);
    case 256: return launch_load_hd<256>(P, rows_grid(P), st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lstk
