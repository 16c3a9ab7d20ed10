// Device helpers of the operators that work on rows of features: units of
// eight elements per lane, their loads and stores for every element type, and
// float8 blocks with a power-of-two scale.
//
// A unit is eight consecutive elements, so the sixteen lanes of a DPP row
// hold one block of 128 and its maximum needs four lane rotations.
#pragma once

#include <type_traits>

#include "mdx_internal.h"

namespace mdx::rows {

constexpr int kUnit = 8;             // elements per lane
constexpr int kScaleBlock = 128;     // elements per scale along the contraction
constexpr int kLeastScale = 10;      // 2^-117 with the bias of 127: 2^-9 of it is the smallest normal float32
constexpr int kNoScale = 255;        // NaN: the block holds an infinity or a NaN

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Eight elements at an address that is aligned to one: the device's global
// loads and stores of 16 bytes take any address.
template <typename T> struct Wide {
    static constexpr int kPart = 16 / int(sizeof(T));
    typedef T part __attribute__((ext_vector_type(kPart), aligned(sizeof(T))));
};

template <typename T> __device__ __forceinline__ void load_wide(const T* p, float (&v)[kUnit]) {
    constexpr int kPart = Wide<T>::kPart;
#pragma unroll
    for (int h = 0; h < kUnit / kPart; ++h) {
        const typename Wide<T>::part a = reinterpret_cast<const typename Wide<T>::part*>(p)[h];
#pragma unroll
        for (int i = 0; i < kPart; ++i) v[h * kPart + i] = static_cast<float>(a[i]);
    }
}

// Past: past the L2, for results that it cannot hold.
template <typename T, bool Past = false> __device__ __forceinline__ void store_wide(T* p, const float (&v)[kUnit]) {
    constexpr int kPart = Wide<T>::kPart;
#pragma unroll
    for (int h = 0; h < kUnit / kPart; ++h) {
        typename Wide<T>::part a;
#pragma unroll
        for (int i = 0; i < kPart; ++i) a[i] = static_cast<T>(v[h * kPart + i]);
        if constexpr (Past) __builtin_nontemporal_store(a, reinterpret_cast<typename Wide<T>::part*>(p) + h);
        else reinterpret_cast<typename Wide<T>::part*>(p)[h] = a;
    }
}

// Elements col..col+7 of a row; zeros from `width` on.
template <typename T, typename I>
__device__ __forceinline__ void load_unit(const T* row, I col, I width, float (&v)[kUnit]) {
    if (col + kUnit <= width) {
        load_wide(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = col + i < width ? static_cast<float>(row[col + i]) : 0.0f;
    }
}

// The same for rows whose lanes wait for each other: the end of a row, n < 8
// elements, in accesses of four, two and one that are under way together,
// where up to seven conditional ones follow each other (gradients of 20,000 x
// 7,380 bfloat16 with a residual's 276 us, 330 with those).  The norm itself gains nothing by it
// (65,536 x 3,696 bfloat16 165 us, 157 without).
template <typename T> __device__ __forceinline__ void load_unit_together(const T* row, int col, int width, float (&v)[kUnit]) {
    if (col + kUnit <= width) {
        load_wide(row + col, v);
        return;
    }
    constexpr int kHalf = int(sizeof(T)) / 2; // words of two elements
    typedef uint32_t four __attribute__((ext_vector_type(2 * kHalf), aligned(sizeof(T))));
    typedef uint32_t pair __attribute__((ext_vector_type(kHalf), aligned(sizeof(T))));
    typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> one;
    const int n = max(width - col, 0);
    const T* p = row + col;
    four a = {};
    pair b = {};
    uint32_t c = 0;
    if (n & 4) a = *reinterpret_cast<const four*>(p);
    if (n & 2) b = *reinterpret_cast<const pair*>(p + (n & 4));
    if (n & 1) c = *reinterpret_cast<const one*>(p + (n & 6));
    uint32_t words[4 * kHalf];
#pragma unroll
    for (int i = 0; i < 2 * kHalf; ++i) { // what follows the four, then all
        const uint32_t first = a[i], two = i < kHalf ? uint32_t(b[i < kHalf ? i : 0]) : i == kHalf ? c : 0u;
        const uint32_t next = n & 2 ? two : i == 0 ? c : 0u;
        words[i] = n & 4 ? first : next;
        words[2 * kHalf + i] = n & 4 ? next : 0u;
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(words[i]);
        else v[i] = static_cast<float>(__builtin_bit_cast(T, uint16_t(words[i / 2] >> (16 * (i % 2)))));
    }
}

template <bool Past = false, typename T, typename I>
__device__ __forceinline__ void store_unit(T* row, I col, I width, const float (&v)[kUnit]) {
    if (col + kUnit <= width) {
        store_wide<T, Past>(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
            if (col + i < width) row[col + i] = static_cast<T>(v[i]);
    }
}

// ---------------------------------------------------------- float8 blocks

__device__ __forceinline__ uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Largest of the sixteen lanes of a DPP row, in all of them.  Sizes are
// compared as integers: an infinity or a NaN is larger than every number.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x128, 0xf, 0xf, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x124, 0xf, 0xf, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x122, 0xf, 0xf, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x121, 0xf, 0xf, false)));
    return x;
}

// Largest of lanes i, i + 16, i + 32 and i + 48 of a wavefront, in all of
// them: the instructions swap rows of sixteen lanes, or halves, of two copies.
__device__ __forceinline__ uint32_t across_max(uint32_t x) {
    const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(uint32_t(rows[0]), uint32_t(rows[1]));
    const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(uint32_t(halves[0]), uint32_t(halves[1]));
}

__device__ __forceinline__ uint32_t unit_max(const float (&v)[kUnit]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) m = max(m, size_bits(v[i]));
    return m;
}

// The scale's byte for a block whose largest size has these bits: 127 plus
// the smallest e >= -117 with that size <= 448 * 2^e (448 = 1.75 * 2^8, the
// largest float8).  A power of two keeps every code's relative precision, is
// exact to multiply by, and is what the matrix cores apply by themselves.
__device__ __forceinline__ int scale_byte(uint32_t most) {
    if (most >= 0x7F800000u) return kNoScale;
    return max(int(most >> 23) - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0), kLeastScale);
}

// Factor that takes a block's values to codes (1 over its scale).
__device__ __forceinline__ float code_factor(int byte) {
    return byte == kNoScale ? 0.0f : __uint_as_float(uint32_t(254 - byte) << 23);
}

__device__ __forceinline__ float scale_value(int byte) { return __uint_as_float(uint32_t(byte) << 23); }

// Four codes, rounded to nearest even; zeros for a block without a scale (its
// NaN scale says what it holds).
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, int byte) {
    const float f = code_factor(byte);
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a * f, b * f, 0, false);
    const uint32_t w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c * f, d * f, low, true));
    return byte == kNoScale ? 0u : w;
}

__device__ __forceinline__ u2 unit_codes(const float (&v)[kUnit], int byte) {
    return u2{four_codes(v[0], v[1], v[2], v[3], byte), four_codes(v[4], v[5], v[6], v[7], byte)};
}

__device__ __forceinline__ void unit_values(u2 c, float (&v)[kUnit]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        v[4 * h + 0] = __builtin_amdgcn_cvt_f32_fp8(int(c[h]), 0);
        v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(int(c[h]), 1);
        v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(int(c[h]), 2);
        v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(int(c[h]), 3);
    }
}

// --------------------------------------------------------------- sums

// Sum over Lanes neighbouring lanes (a power of two), in all of them; the same
// order in each.  Over more than a wavefront `part` holds one float per
// wavefront of the workgroup, is free again after the caller's next barrier,
// and all lanes of the workgroup have to be here.
template <int Lanes> __device__ __forceinline__ float group_sum(float x, float* part) {
#pragma unroll
    for (int d = 1; d < (Lanes < kWave ? Lanes : kWave); d *= 2) x += __shfl_xor(x, d, kWave);
    if constexpr (Lanes > kWave) {
        constexpr int kWaves = Lanes / kWave;
        const int wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0) part[wave] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += part[wave / kWaves * kWaves + w];
    }
    return x;
}

inline bool aligned16(const void* p, int64_t pitch_bytes) {
    return (reinterpret_cast<uintptr_t>(p) % 16) == 0 && pitch_bytes % 16 == 0;
}

}  // namespace mdx::rows
