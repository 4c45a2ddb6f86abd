// cache_q8.hip - rows of K and V quantised as they are written to a cache (cache_q8.h), and read back.
//
//   d = min { fp16 numbers >= max |x| / 127 },  q = x / d to the nearest whole number, halves to the even one;  back: d q
//
// over 32 dims of a row. d is no less than a 127th of the largest, so |q| <= 127 without a clamp, and no value is off by more than
// d / 2. The 32-bit quotient only guesses q; the remainder x - q d is exact in one fma and settles it.
//
// Bound by memory, and by the launch for the rows of a decode step. A work-group takes kCrRows rows of a KV head: the whole numbers
// meet in LDS, because a row of V is single bytes 16 apart in its record: where the work-group's rows fill an octet of cells, as
// the rows of a prompt do, they leave as 8 bytes at a time.
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
__device__ __forceinline__ void look_up_cells(const CacheRowsParams &P, Cells &C, int row0, int n) {
    const int i = threadIdx.x;
    if (i < kCrRows) {
        const int c = i < n ? P.cells[row0 + i] : -1;
        C.cell[i] = c >= 0 && c < P.n_cells ? c : -1;
    }
    __syncthreads();
    if (i < kCrRows) {
        const int c = C.cell[i], first = i - (c & 7);
        bool full = c >= 0 && first >= 0 && first + 8 <= n;
        for (int k = 0; k < 8 && full; k++) full = C.cell[first + k] == c - (c & 7) + k;
        C.octet[i] = full ? (first == i ? 1 : 2) : 0;
    }
    __syncthreads();
}
__device__ __forceinline__ uint8_t *record_of(const CacheRowsParams &P, int cell, int g) {
    return P.cache + ((int64_t) (cell / kPageCells) * P.n_kv + g) * q8_record(P.hd);
}

// Four neighbouring dims of a row, as 32-bit values.
template <typename T>
__device__ __forceinline__ float4 four(const T *p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4 *>(p);
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        return make_float4(h2f(u.x), h2f(u.x >> 16), h2f(u.y), h2f(u.y >> 16));
    }
}
template <typename T>
__device__ __forceinline__ void put_four(T *p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = v;
    } else {
        ushort4 h;
        h.x = __half_as_ushort(__float2half_rn(v.x));
        h.y = __half_as_ushort(__float2half_rn(v.y));
        h.z = __half_as_ushort(__float2half_rn(v.z));
        h.w = __half_as_ushort(__float2half_rn(v.w));
        *reinterpret_cast<ushort4 *>(p) = h;
    }
}

// x / d to the nearest whole number, halves to the even one; |x| <= 127 d.
__device__ __forceinline__ int whole_of(float x, float d, float inv) {
    float q = rintf(x * inv);                              // within one of it
    const float rest = fmaf(-q, d, x), half = 0.5f * d;    // exact: a whole number of bits of x or of d, below 2 d
    const bool odd = ((int) q & 1) != 0;
    if (rest > half || (rest == half && odd)) q += 1.0f;
    else if (rest < -half || (rest == -half && odd)) q -= 1.0f;
    return (int) q;
}

template <int HD, typename T>
__global__ __launch_bounds__(kBlock) void cache_store_kernel(CacheRowsParams P) {
    constexpr int NM = HD / kQ8Dims;
    __shared__ Cells C;
    __shared__ uint32_t s_q[2][kCrRows][HD / 4 + 1]; // (+ 1: columns of V are read)
    __shared__ uint16_t s_d[2][kCrRows][NM];
    const int g = blockIdx.x % P.n_kv, row0 = blockIdx.x / P.n_kv * kCrRows, n = min(kCrRows, P.n - row0), tid = threadIdx.x;
    look_up_cells(P, C, row0, n);
    // 8 lanes a block of 32 dims
    for (int i = tid; i < n * NM * 2 * 8; i += kBlock) {
        const int lane = i & 7, m = i / 8 % NM, r = i / (8 * NM) % n, kind = i / (8 * NM * n);
        const T *src = static_cast<const T *>(kind ? P.v : P.k) + (row0 + r) * (kind ? P.ld_v : P.ld_k) + g * HD + 32 * m + 4 * lane;
        const float4 x = four(src);
        // the largest magnitude by its bits, so that infinities and NaN are larger than any number
        unsigned most = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
                            max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
        for (int d = 1; d < 8; d *= 2) most = max(most, (unsigned) __shfl_xor((int) most, d, kWave));
        unsigned bits = 0x7e00u; // NaN, for a block that holds one, an infinity or more than d can
        uint32_t q = 0;
        if (most <= __float_as_uint(kMostMost)) {
            const float a = __uint_as_float(most);
            bits = __half_as_ushort(__float2half_rn(a / 127.0f));
            if (h2f(bits) * 127.0f < a) bits++; // (19 bits: exact)
            const float d = h2f(bits), inv = d == 0.0f ? 0.0f : 1.0f / d;
            q = ((unsigned) whole_of(x.x, d, inv) & 0xffu) | ((unsigned) whole_of(x.y, d, inv) & 0xffu) << 8 |
                ((unsigned) whole_of(x.z, d, inv) & 0xffu) << 16 | (unsigned) whole_of(x.w, d, inv) << 24;
        }
        s_q[kind][r][8 * m + lane] = q;
        if (lane == 0) s_d[kind][r][m] = (uint16_t) bits;
    }
    __syncthreads();
    // K: 8 dims of a row
    for (int i = tid; i < n * (HD / 8); i += kBlock) {
        const int r = i % n, p = i / n, cell = C.cell[r];
        if (cell < 0) continue;
        *reinterpret_cast<uint2 *>(record_of(P, cell, g) + q8_k(p / 4, cell % kPageCells, p % 4 * 8)) =
            make_uint2(s_q[0][r][2 * p], s_q[0][r][2 * p + 1]);
    }
    // V: a dim of a row, or of 8 rows; lanes take neighbouring dims
    for (int i = tid; i < n * HD; i += kBlock) {
        const int r = i / HD, d = i % HD, cell = C.cell[r];
        if (cell < 0 || C.octet[r] == 2) continue;
        uint8_t *dst = record_of(P, cell, g) + q8_v(HD, d / 32, cell % kPageCells, d % 32);
        auto byte = [&](int row) { return s_q[1][row][d / 4] >> (8 * (d & 3)) & 0xffu; };
        if (C.octet[r] == 0) {
            *dst = (uint8_t) byte(r);
            continue;
        }
        unsigned lo = 0, hi = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            lo |= byte(r + k) << (8 * k);
            hi |= byte(r + 4 + k) << (8 * k);
        }
        *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
    }
    for (int i = tid; i < n * NM * 2; i += kBlock) {
        const int r = i % n, m = i / n % NM, kind = i / (n * NM), cell = C.cell[r];
        if (cell < 0) continue;
        const int at = kind ? q8_v_scale(HD, m, cell % kPageCells) : q8_k_scale(HD, m, cell % kPageCells);
        *reinterpret_cast<uint16_t *>(record_of(P, cell, g) + at) = s_d[kind][r][m];
    }
}

template <int HD, typename T>
__global__ __launch_bounds__(kBlock) void cache_load_kernel(CacheRowsParams P) {
    constexpr int NM = HD / kQ8Dims;
    __shared__ Cells C;
    __shared__ uint32_t s_q[2][kCrRows][HD / 4 + 1];
    __shared__ uint16_t s_d[2][kCrRows][NM];
    const int g = blockIdx.x % P.n_kv, row0 = blockIdx.x / P.n_kv * kCrRows, n = min(kCrRows, P.n - row0), tid = threadIdx.x;
    look_up_cells(P, C, row0, n);
    for (int i = tid; i < n * (HD / 8); i += kBlock) {
        const int r = i % n, p = i / n, cell = C.cell[r];
        uint2 u = make_uint2(0, 0);
        if (cell >= 0) u = *reinterpret_cast<const uint2 *>(record_of(P, cell, g) + q8_k(p / 4, cell % kPageCells, p % 4 * 8));
        s_q[0][r][2 * p] = u.x;
        s_q[0][r][2 * p + 1] = u.y;
    }
    for (int i = tid; i < n * HD; i += kBlock) {
        const int r = i / HD, d = i % HD, cell = C.cell[r];
        if (C.octet[r] == 2) continue;
        auto put = [&](int row, unsigned b) { reinterpret_cast<uint8_t *>(&s_q[1][row][0])[d] = (uint8_t) b; };
        if (cell < 0) {
            put(r, 0);
            continue;
        }
        const uint8_t *src = record_of(P, cell, g) + q8_v(HD, d / 32, cell % kPageCells, d % 32);
        if (C.octet[r] == 0) {
            put(r, *src);
            continue;
        }
        const uint2 u = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            put(r + k, u.x >> (8 * k));
            put(r + 4 + k, u.y >> (8 * k));
        }
    }
    for (int i = tid; i < n * NM * 2; i += kBlock) {
        const int r = i % n, m = i / n % NM, kind = i / (n * NM), cell = C.cell[r];
        const int at = kind ? q8_v_scale(HD, m, cell % kPageCells) : q8_k_scale(HD, m, cell % kPageCells);
        s_d[kind][r][m] = cell < 0 ? 0 : *reinterpret_cast<const uint16_t *>(record_of(P, cell, g) + at);
    }
    __syncthreads();
    for (int i = tid; i < n * NM * 2 * 8; i += kBlock) {
        const int lane = i & 7, m = i / 8 % NM, r = i / (8 * NM) % n, kind = i / (8 * NM * n);
        const uint32_t q = s_q[kind][r][8 * m + lane];
        const float d = h2f(s_d[kind][r][m]);
        auto value = [&](int k) { return (float) (int8_t) (q >> (8 * k)) * d; };
        T *dst = static_cast<T *>(const_cast<void *>(kind ? P.v : P.k)) + (row0 + r) * (kind ? P.ld_v : P.ld_k) + g * HD + 32 * m + 4 * lane;
        put_four(dst, make_float4(value(0), value(1), value(2), value(3)));
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
dim3 rows_grid(const CacheRowsParams &P) { return dim3((unsigned) ((int64_t) ((P.n + kCrRows - 1) / kCrRows) * P.n_kv)); }

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
