// One AdamW step over many tensors in few launches.
//
// Every element is read and written once (28 bytes with float32 states and
// gradients, 14 with 8-bit states and 16-bit gradients), so the step is bound
// by HBM, or by the launch where the tensors are small.  The tensors' pointers
// travel in the kernel's arguments: nothing is copied to the device ahead of
// the launch, nothing is kept from step to step, and 48 tensors take one
// launch.  40 tensors of 60.4 M elements with 8-bit states take 154 us (5.5
// TB/s), twelve of 0.56 M with 32-bit states 5.8 us.
#include "rows_device.h"

#include <algorithm>
#include <cmath>

#include "rows_internal.h"

namespace mdx {
namespace {

using namespace rows;

typedef uint32_t u2_any __attribute__((ext_vector_type(2), aligned(1))); // eight codes at any address

constexpr int kTensors = 48;            // per launch: 48 * 68 bytes of arguments and the numbers, under the 4 KB of a launch
constexpr int kChunk = 256 * kUnit;    // elements per workgroup: with two or four units a lane, 5 and 20 % slower
static_assert(kChunk == kAdamwChunk, "the size that the entry point refuses follows from it");

struct AdamwTable {
    float* params[kTensors];
    const void* grads[kTensors];
    void* first[kTensors];
    void* second[kTensors];
    uint8_t* first_scales[kTensors];
    uint8_t* second_scales[kTensors];
    int64_t n[kTensors];
    int64_t end[kTensors]; // chunks up to and with this tensor's
    int32_t place[kTensors];
    int32_t count;
    float keep;      // 1 - lr * weight_decay
    float rate;      // lr / (1 - beta1^step)
    float root;      // 1 / sqrt(1 - beta2^step)
    float eps, beta1, beta2, rest1, rest2;
    uint32_t seed;
    // in device memory, where given: read when the kernel runs, so that a replayed graph goes on with what stands there
    const int64_t* step_at;
    const int64_t* seed_at;
    double lr, log1, log2; // of the betas
};
static_assert(sizeof(AdamwTable) <= 4096, "a launch takes 4 KB of arguments");

__device__ __forceinline__ uint32_t mixed(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// A size in [0, 448] to one of its two neighbours among the float8 values, up
// with the probability of its distance from the lower one: 16 random bits are
// added below the three bits of the fraction and the rest is cut off.  Under
// 2^-6, where the values are evenly spaced, the same with 2^-6 added.
__device__ __forceinline__ float rounded(float size, uint32_t bits) {
    const bool small = size < 0x1p-6f;
    const float lifted = small ? size + 0x1p-6f : size;
    const float cut = __uint_as_float((__float_as_uint(lifted) + (bits << 4)) & 0xFFF00000u);
    return small ? cut - 0x1p-6f : cut;
}

template <bool Root>
__device__ __forceinline__ void store_codes(const float (&v)[kUnit], const uint32_t (&bits)[kUnit], uint8_t* codes,
                                            uint8_t* scale, int64_t left) {
    const int byte = scale_byte(row_max(unit_max(v)));
    const float f = code_factor(byte);
    float c[kUnit];
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        float size = rounded(fabsf(v[i]) * f, Root ? bits[i] >> 16 : bits[i] & 0xFFFFu);
        if (Root && v[i] > 0.0f) size = fmaxf(size, 0x1p-9f);
        c[i] = copysignf(size, v[i]);
    }
    const u2 w = unit_codes(c, byte == kNoScale ? kNoScale : 127);
    if (threadIdx.x % 16 == 0 && left > 0) *scale = uint8_t(byte);
    if (left >= kUnit) {
        *reinterpret_cast<u2_any*>(codes) = w;
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
            if (i < left) codes[i] = uint8_t(w[i / 4] >> (8 * (i % 4)));
    }
}

// Codes at..at+7 of a tensor of n; zeros from n on.
__device__ __forceinline__ u2 load_codes(const uint8_t* codes, int64_t at, int64_t n) {
    if (at + kUnit <= n) return *reinterpret_cast<const u2_any*>(codes + at);
    u2 c{0u, 0u};
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
        if (at + i < n) c[i / 4] |= uint32_t(codes[at + i]) << (8 * (i % 4));
    return c;
}

// Moving: step and seed, as far as they are given so, come from device memory (0.3 us more for twelve tensors, 158 us in
// place of 154 for 60.4 M elements with 8-bit states: the corrections are computed by every wavefront).
template <typename G, bool Codes, bool Moving> __global__ __launch_bounds__(256) void k_adamw(const AdamwTable a) {
    const int64_t chunk = blockIdx.x;
    uint32_t seed = a.seed;
    int64_t step = 1;
    if constexpr (Moving) {
        if (a.seed_at != nullptr) seed = uint32_t(*a.seed_at);
        if (a.step_at != nullptr) step = *a.step_at;
        if (step < 1) return; // there is no such step
    }
    // the tensor: each lane compares one entry, and the ballot counts those that end before this chunk
    const int lane = threadIdx.x % kWave;
    const int k = __popcll(__ballot(lane < a.count && chunk >= a.end[min(lane, kTensors - 1)]));
    const int64_t n = a.n[k];
    const int64_t begin = (chunk - (k == 0 ? 0 : a.end[k - 1])) * kChunk;
    float* params = a.params[k];
    const G* grads = static_cast<const G*>(a.grads[k]);
    const int64_t at = begin + threadIdx.x * kUnit;
    float rate = a.rate, root = a.root;
    // whole blocks of 128 go on together: their lanes find the maximum
    if (at / kScaleBlock * kScaleBlock >= n) return;
    float p[kUnit], g[kUnit], m[kUnit], v[kUnit], r[kUnit];
    load_unit(params, at, n, p);
    load_unit(grads, at, n, g);
    if constexpr (Codes) {
        const u2 codes_m = load_codes(static_cast<const uint8_t*>(a.first[k]), at, n);
        const u2 codes_v = load_codes(static_cast<const uint8_t*>(a.second[k]), at, n);
        const int byte_m = a.first_scales[k][at / kScaleBlock], byte_v = a.second_scales[k][at / kScaleBlock];
        const float scale_m = byte_m == kNoScale ? __builtin_nanf("") : scale_value(byte_m);
        const float scale_v = byte_v == kNoScale ? __builtin_nanf("") : scale_value(byte_v);
        unit_values(codes_m, m);
        unit_values(codes_v, v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            m[i] *= scale_m;
            v[i] *= scale_v;
            v[i] *= v[i];
        }
    } else {
        load_unit(static_cast<const float*>(a.first[k]), at, n, m);
        load_unit(static_cast<const float*>(a.second[k]), at, n, v);
    }
    if constexpr (Moving) {
        if (a.step_at != nullptr) { // 1 - beta^step; while the loads above are under way
            rate = float(a.lr / -expm1(double(step) * a.log1));
            root = float(1.0 / sqrt(-expm1(double(step) * a.log2)));
        }
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        m[i] = fmaf(a.beta1, m[i], a.rest1 * g[i]);
        v[i] = fmaf(a.beta2, v[i], a.rest2 * g[i] * g[i]);
        // the device's own root and reciprocal, good to one unit in the last place (a v below the normal numbers has
        // the root zero); correctly rounded ones take ten instructions each, and the 8-bit step is then bound by
        // them: 195 us in place of 161 for 60.4 M elements
        r[i] = __builtin_amdgcn_sqrtf(v[i]);
        p[i] = fmaf(p[i], a.keep, -(rate * m[i]) * __builtin_amdgcn_rcpf(fmaf(r[i], root, a.eps)));
    }
    store_unit(params, at, n, p);
    if constexpr (Codes) {
        // past the tensor's end lie zeros: g, m and v are
        const uint32_t high = uint32_t(uint64_t(at) >> 32);
        const uint32_t key = mixed(seed + 0x9E3779B9u * uint32_t(a.place[k] + 1) + 0x85EBCA6Bu * high);
        uint32_t bits[kUnit];
#pragma unroll
        for (int i = 0; i < kUnit; ++i) bits[i] = mixed(uint32_t(at + i) ^ key);
        store_codes<false>(m, bits, static_cast<uint8_t*>(a.first[k]) + at, a.first_scales[k] + at / kScaleBlock, n - at);
        store_codes<true>(r, bits, static_cast<uint8_t*>(a.second[k]) + at, a.second_scales[k] + at / kScaleBlock, n - at);
    } else {
        store_unit(static_cast<float*>(a.first[k]), at, n, m);
        store_unit(static_cast<float*>(a.second[k]), at, n, v);
    }
}

template <typename G> void launch_adamw(const AdamwTable& t, bool codes, hipStream_t s) {
    const dim3 grid(unsigned(t.end[t.count - 1]));
    if (t.step_at != nullptr || t.seed_at != nullptr) {
        if (codes) k_adamw<G, true, true><<<grid, 256, 0, s>>>(t);
        else k_adamw<G, false, true><<<grid, 256, 0, s>>>(t);
    } else {
        if (codes) k_adamw<G, true, false><<<grid, 256, 0, s>>>(t);
        else k_adamw<G, false, false><<<grid, 256, 0, s>>>(t);
    }
    MDX_HIP(hipGetLastError());
}

} // namespace

void adamw_step(const mdx_adamw_args& g, const int64_t* step_at, const int64_t* seed_at, hipStream_t s) {
    AdamwTable t{};
    const double step = double(g.step);
    t.keep = float(1.0 - g.lr * g.weight_decay);
    t.rate = float(g.lr / (1.0 - std::pow(g.beta1, step)));
    t.root = float(1.0 / std::sqrt(1.0 - std::pow(g.beta2, step)));
    t.eps = float(g.eps);
    t.beta1 = float(g.beta1);
    t.beta2 = float(g.beta2);
    t.rest1 = float(1.0 - g.beta1);
    t.rest2 = float(1.0 - g.beta2);
    t.seed = g.seed;
    t.step_at = step_at;
    t.seed_at = seed_at;
    t.lr = g.lr;
    t.log1 = std::log(g.beta1);
    t.log2 = std::log(g.beta2);
    constexpr int64_t kMostChunks = kAdamwMost / kChunk; // workgroups per launch
    auto flush = [&] {
        if (t.count == 0) return;
        const bool codes = g.bits == 8;
        if (g.grad_dtype == MDX_FLOAT32) launch_adamw<float>(t, codes, s);
        else if (g.grad_dtype == MDX_BFLOAT16) launch_adamw<__bf16>(t, codes, s);
        else launch_adamw<_Float16>(t, codes, s);
        t.count = 0;
    };
    for (int64_t i = 0; i < g.count; ++i) {
        const mdx_adamw_tensor& x = g.tensors[i];
        if (x.n == 0) continue;
        const int64_t chunks = (x.n + kChunk - 1) / kChunk;
        const int64_t before = t.count == 0 ? 0 : t.end[t.count - 1];
        if (t.count == kTensors || (t.count > 0 && before + chunks > kMostChunks)) flush();
        const int k = t.count++;
        t.params[k] = x.params;
        t.grads[k] = x.grads;
        t.first[k] = x.first;
        t.second[k] = x.second;
        t.first_scales[k] = x.first_scales;
        t.second_scales[k] = x.second_scales;
        t.n[k] = x.n;
        t.end[k] = (k == 0 ? 0 : t.end[k - 1]) + chunks;
        t.place[k] = int32_t(i);
    }
    flush();
}

} // namespace mdx
