// Root-mean-square norm of feature rows, with the residual's addition and a
// float8 output, and its gradients.
//
// values = t rstd gain with t = x + residual and rstd = (mean(t^2) + eps)^-1/2.
// A row is read once: its units stay in registers between the sum of squares
// and the products, so both directions move each byte once and are bound by
// HBM once there are rows enough to fill the device: 65,536 x 3,696 float32 to
// float8 takes 210 us (5.8 TB/s), the gradients of 65,536 x 1,024 bfloat16 with a
// residual's 100 us (5.35 TB/s).  One row of 3,696 takes 2.8 us on the device.
#include "rows_device.h"

#include <algorithm>
#include <cmath>

#include "rows_internal.h"

namespace mdx {
namespace {

using namespace rows;

struct NormView {
    int64_t rows, width;
    const void* x;
    int64_t x_pitch;
    const void* residual;
    int64_t residual_pitch;
    const float* gain;
    void* values;
    int64_t values_pitch;
    uint8_t* scales;
    int64_t scales_pitch;
    void* total;
    int64_t total_pitch;
    float* rstd;
    float eps;
};

// Units of one row: t = x + residual.  The total is rounded to the rows' type
// where it is stored; the norm goes on with the float32 sum.
template <typename T>
__device__ __forceinline__ void load_total(const NormView& a, int64_t row, int64_t col, float (&v)[kUnit]) {
    load_unit(static_cast<const T*>(a.x) + row * a.x_pitch, col, a.width, v);
    if (a.residual != nullptr) {
        float r[kUnit];
        load_unit(static_cast<const T*>(a.residual) + row * a.residual_pitch, col, a.width, r);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] += r[i];
    }
}

template <typename T, bool Codes, bool Past>
__device__ __forceinline__ void store_values(const NormView& a, int64_t row, int64_t col, float rstd,
                                             const float (&v)[kUnit]) {
    float g[kUnit], y[kUnit];
    load_unit(a.gain, col, a.width, g);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) y[i] = v[i] * rstd * g[i];
    if constexpr (Codes) {
        // all sixteen lanes of a block are here: units past the width are zeros
        const int byte = scale_byte(row_max(unit_max(y)));
        const u2 codes = unit_codes(y, byte);
        u2* to = reinterpret_cast<u2*>(static_cast<uint8_t*>(a.values) + row * a.values_pitch + col);
        if constexpr (Past) __builtin_nontemporal_store(codes, to);
        else *to = codes;
        if (threadIdx.x % 16 == 0) a.scales[row * a.scales_pitch + col / kScaleBlock] = uint8_t(byte);
    } else {
        store_unit<Past>(static_cast<T*>(a.values) + row * a.values_pitch, col, a.width, y);
    }
}

// Lanes neighbouring lanes take a row of at most Lanes * 8 * Units elements; a
// workgroup of 256 holds 256 / Lanes rows.  Units 0: a row of any width, read
// twice.
template <typename T, bool Codes, int Lanes, int Units, bool Past>
__global__ __launch_bounds__(Lanes > 256 ? Lanes : 256) void k_norm(const NormView a) {
    constexpr int kThreads = Lanes > 256 ? Lanes : 256;
    __shared__ float part[kThreads / kWave];
    const int lane = threadIdx.x % Lanes;
    const int64_t row = int64_t(blockIdx.x) * (kThreads / Lanes) + threadIdx.x / Lanes;
    const int64_t width = row < a.rows ? a.width : 0; // lanes without a row stay for the barrier
    // the blocks of 128 that a float8 output fills are taken whole
    const int64_t end = Codes ? (width + kScaleBlock - 1) / kScaleBlock * kScaleBlock : width;
    constexpr int kHeld = Units > 0 ? Units : 1;
    float v[kHeld][kUnit];
    float squares = 0.0f;
    if constexpr (Units > 0) {
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int64_t col = int64_t(lane + u * Lanes) * kUnit;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) v[u][i] = 0.0f;
            if (col < width) load_total<T>(a, row, col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int64_t col = int64_t(lane + u * Lanes) * kUnit;
            if (a.total != nullptr && col < width)
                store_unit<Past>(static_cast<T*>(a.total) + row * a.total_pitch, col, a.width, v[u]);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) s = fmaf(v[u][i], v[u][i], s);
            squares += s;
        }
    } else {
        for (int64_t col = int64_t(lane) * kUnit; col < width; col += Lanes * kUnit) {
            load_total<T>(a, row, col, v[0]);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) s = fmaf(v[0][i], v[0][i], s);
            squares += s;
        }
    }
    squares = group_sum<Lanes>(squares, part);
    const float rstd = 1.0f / sqrtf(squares / float(a.width) + a.eps);
    if (lane == 0 && row < a.rows && a.rstd != nullptr) a.rstd[row] = rstd;
    if constexpr (Units > 0) {
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int64_t col = int64_t(lane + u * Lanes) * kUnit;
            if (col < end) store_values<T, Codes, Past>(a, row, col, rstd, v[u]);
        }
    } else {
        for (int64_t col = int64_t(lane) * kUnit; col < end; col += Lanes * kUnit) {
            if (col < width) {
                // the same lane reads its units again before it writes them: the total may be x or the residual
                load_total<T>(a, row, col, v[0]);
                if (a.total != nullptr)
                    store_unit<Past>(static_cast<T*>(a.total) + row * a.total_pitch, col, a.width, v[0]);
            } else {
#pragma unroll
                for (int i = 0; i < kUnit; ++i) v[0][i] = 0.0f;
            }
            store_values<T, Codes, Past>(a, row, col, rstd, v[0]);
        }
    }
}

// Rows first..first+most-1, as far as there are such.
template <typename T, bool Codes> NormView rows_from(NormView a, int64_t first, int64_t most) {
    a.rows = std::min(a.rows - first, most);
    a.x = static_cast<const T*>(a.x) + first * a.x_pitch;
    if (a.residual != nullptr) a.residual = static_cast<const T*>(a.residual) + first * a.residual_pitch;
    if (a.total != nullptr) a.total = static_cast<T*>(a.total) + first * a.total_pitch;
    if (a.rstd != nullptr) a.rstd += first;
    if constexpr (Codes) {
        a.values = static_cast<uint8_t*>(a.values) + first * a.values_pitch;
        a.scales += first * a.scales_pitch;
    } else {
        a.values = static_cast<T*>(a.values) + first * a.values_pitch;
    }
    return a;
}

template <typename T, bool Codes, int Lanes, int Units> void launch_norm(const NormView& a, bool past, hipStream_t s) {
    constexpr int kThreads = Lanes > 256 ? Lanes : 256, kRows = kThreads / Lanes;
    in_runs((a.rows + kRows - 1) / kRows, kThreads, [&](int64_t first, int64_t count) {
        const NormView b = rows_from<T, Codes>(a, first * kRows, count * kRows);
        if (past) k_norm<T, Codes, Lanes, Units, true><<<dim3(unsigned(count)), kThreads, 0, s>>>(b);
        else k_norm<T, Codes, Lanes, Units, false><<<dim3(unsigned(count)), kThreads, 0, s>>>(b);
        MDX_HIP(hipGetLastError());
    });
}

template <typename T, bool Codes> void choose_norm(const NormView& a, bool past, hipStream_t s) {
    // lanes a row: few enough that most of them hold a unit and each has two to four in flight, the row's barrier
    // over two wavefronts at most where there are rows enough (65,536 x 3,696 float32 to float8: 303 us with one
    // wavefront a row, 234 with two, 243 with four); more lanes where rows are few
    const bool many = a.rows >= 1024;
    if (a.width <= 128) return launch_norm<T, Codes, 16, 1>(a, past, s);
    if (a.width <= 256) return launch_norm<T, Codes, 32, 1>(a, past, s);
    if (many && a.width <= 1024) return launch_norm<T, Codes, 64, 2>(a, past, s);
    if (many && a.width <= 2048) return launch_norm<T, Codes, 128, 2>(a, past, s);
    if (many && a.width <= 4096) return launch_norm<T, Codes, 128, 4>(a, past, s);
    if (a.width <= 4096) return launch_norm<T, Codes, 256, 2>(a, past, s);
    if (a.width <= 8192) return launch_norm<T, Codes, 256, 4>(a, past, s);
    if (a.width <= 32768) return launch_norm<T, Codes, 1024, 4>(a, past, s);
    return launch_norm<T, Codes, 1024, 0>(a, past, s);
}

struct BackView {
    int64_t rows, width;
    const void* grad;
    int64_t grad_pitch;
    const void* t;
    int64_t t_pitch;
    const void* grad_total;
    int64_t grad_total_pitch;
    const float* gain;
    const float* rstd;
    void* grad_x;
    int64_t grad_x_pitch;
    float* part; // [workgroups][width]: each workgroup's share of the gain's gradient
};

// Lanes neighbouring lanes take a row, a workgroup 256 / Lanes rows at a time,
// a grid apart, and keeps its share of the gain's gradient in registers: one
// partial row per workgroup, whatever the number of rows.
template <typename T, int Lanes, int Units>
__global__ __launch_bounds__(Lanes > 256 ? Lanes : 256, 4) void k_norm_back(const BackView a) {
    constexpr int kThreads = Lanes > 256 ? Lanes : 256;
    constexpr int kRows = kThreads / Lanes; // in hand per workgroup
    __shared__ float part[2][kThreads / kWave];
    const int lane = threadIdx.x % Lanes, mine = threadIdx.x / Lanes, width = int(a.width);
    float gain[Units][kUnit], sum[Units][kUnit];
#pragma unroll
    for (int u = 0; u < Units; ++u) {
        load_unit(a.gain, (lane + u * Lanes) * kUnit, width, gain[u]);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) sum[u][i] = 0.0f;
    }
    int turn = 0;
    for (int64_t base = int64_t(blockIdx.x) * kRows; base < a.rows; base += int64_t(gridDim.x) * kRows) {
        // lanes without a row stay for the barrier and load zeros: another row's elements would not cancel (an infinite
        // gradient times a u of zero is NaN), and its owner may already store grad_x over them
        // (one row a workgroup is always there; said as a constant, the kernels of 256 and more lanes spill: 20,000 x 7,380
        // bfloat16 without a residual's gradient 317 us, 215 so)
        const bool there = base + mine < a.rows;
        const int64_t row = there ? base + mine : a.rows - 1;
        const int here = kRows == 1 || there ? width : 0;
        float t[Units][kUnit], h[Units][kUnit];
        const float rstd = there ? a.rstd[row] : 0.0f;
        float along = 0.0f;
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int col = (lane + u * Lanes) * kUnit;
            load_unit_together(static_cast<const T*>(a.t) + row * a.t_pitch, col, here, t[u]);
            load_unit_together(static_cast<const T*>(a.grad) + row * a.grad_pitch, col, here, h[u]);
        }
#pragma unroll
        for (int u = 0; u < Units; ++u) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) {
                t[u][i] *= rstd;
                sum[u][i] = fmaf(h[u][i], t[u][i], sum[u][i]);
                h[u][i] *= gain[u][i];
                along = fmaf(h[u][i], t[u][i], along);
            }
        }
        along = group_sum<Lanes>(along, part[turn]) / float(width);
        turn ^= 1; // the next row's sums are written while this row's may still be read
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int col = (lane + u * Lanes) * kUnit;
            if (!there || col >= width) continue;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) h[u][i] = rstd * fmaf(-t[u][i], along, h[u][i]);
            if (a.grad_total != nullptr) {
                float r[kUnit];
                load_unit_together(static_cast<const T*>(a.grad_total) + row * a.grad_total_pitch, col, width, r);
#pragma unroll
                for (int i = 0; i < kUnit; ++i) h[u][i] += r[i];
            }
            store_unit(static_cast<T*>(a.grad_x) + row * a.grad_x_pitch, col, width, h[u]);
        }
    }
    float* out = a.part + int64_t(blockIdx.x) * a.width;
    if constexpr (kRows > 1) {
        // the shares of the rows side by side, added in their order
        __shared__ float shares[kRows][Lanes * kUnit];
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kUnit; ++i) shares[mine][i * Lanes + lane] = sum[u][i];
            __syncthreads();
            for (int e = threadIdx.x; e < Lanes * kUnit; e += kThreads) {
                const int col = (u * Lanes + e % Lanes) * kUnit + e / Lanes;
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kRows; ++w) s += shares[w][e];
                if (col < width) out[col] = s;
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < Units; ++u) {
            const int col = (lane + u * Lanes) * kUnit;
#pragma unroll
            for (int i = 0; i < kUnit; ++i)
                if (col + i < width) out[col + i] = sum[u][i];
        }
    }
}

// Rows too wide for registers: one workgroup per row, read twice.
template <typename T> __global__ __launch_bounds__(1024) void k_norm_back_long(const BackView a) {
    __shared__ float part[16];
    const int64_t row = blockIdx.x;
    const T* t = static_cast<const T*>(a.t) + row * a.t_pitch;
    const T* grad = static_cast<const T*>(a.grad) + row * a.grad_pitch;
    const float rstd = a.rstd[row];
    float along = 0.0f;
    float x[kUnit], h[kUnit], g[kUnit];
    for (int64_t col = int64_t(threadIdx.x) * kUnit; col < a.width; col += 1024 * kUnit) {
        load_unit(t, col, a.width, x);
        load_unit(grad, col, a.width, h);
        load_unit(a.gain, col, a.width, g);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kUnit; ++i) s = fmaf(h[i] * g[i], x[i] * rstd, s);
        along += s;
    }
    along = group_sum<1024>(along, part) / float(a.width);
    for (int64_t col = int64_t(threadIdx.x) * kUnit; col < a.width; col += 1024 * kUnit) {
        load_unit(t, col, a.width, x);
        load_unit(grad, col, a.width, h);
        load_unit(a.gain, col, a.width, g);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) h[i] = rstd * fmaf(-(x[i] * rstd), along, h[i] * g[i]);
        if (a.grad_total != nullptr) {
            load_unit(static_cast<const T*>(a.grad_total) + row * a.grad_total_pitch, col, a.width, g);
#pragma unroll
            for (int i = 0; i < kUnit; ++i) h[i] += g[i];
        }
        store_unit(static_cast<T*>(a.grad_x) + row * a.grad_x_pitch, col, a.width, h);
    }
}

// Their gain's gradient: a column strip of 2048 per workgroup, rows a grid's
// second dimension apart.  It runs first: grad_x may be grad itself.
template <typename T> __global__ __launch_bounds__(256) void k_norm_gain_long(const BackView a) {
    const int64_t col = (int64_t(blockIdx.x) * 256 + threadIdx.x) * kUnit;
    float sum[kUnit] = {};
    if (col >= a.width) return;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        float x[kUnit], h[kUnit];
        load_unit(static_cast<const T*>(a.t) + row * a.t_pitch, col, a.width, x);
        load_unit(static_cast<const T*>(a.grad) + row * a.grad_pitch, col, a.width, h);
        const float rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < kUnit; ++i) sum[i] = fmaf(h[i], x[i] * rstd, sum[i]);
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
        if (col + i < a.width) a.part[int64_t(blockIdx.y) * a.width + col + i] = sum[i];
}

// Sum of the workgroups' partial rows: Cols columns per workgroup, 1024 / Cols
// groups of rows side by side, joined pairwise.
template <int Cols>
__global__ __launch_bounds__(1024) void k_norm_gain(const float* part, int64_t parts, int64_t width, float* out,
                                                    int64_t first) {
    constexpr int kGroups = 1024 / Cols;
    __shared__ float sums[kGroups][Cols + 1];
    const int mine = threadIdx.x % Cols, group = threadIdx.x / Cols;
    const int64_t col = (first + int64_t(blockIdx.x)) * Cols + mine;
    float s = 0.0f;
    if (col < width) {
        int64_t p = group;
        for (; p + 7 * kGroups < parts; p += 8 * kGroups) { // eight loads under way
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = part[(p + e * kGroups) * width + col];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += x[e];
        }
        for (; p < parts; p += kGroups) s += part[p * width + col];
    }
    sums[group][mine] = s;
    __syncthreads();
    for (int half = kGroups / 2; half > 0; half /= 2) {
        if (group < half) sums[group][mine] += sums[group + half][mine];
        __syncthreads();
    }
    if (group == 0 && col < width) out[col] = sums[0][mine];
}

struct BackShape {
    int lanes, units;
    int64_t groups;
};

// Lanes per row, units per lane and workgroups: no more than there are rows
// for, and than the device holds at once, so that the partial rows are few
// (5,321 x 5,621 float32 without a residual's: 84 us, 107 with twice the workgroups).
BackShape back_shape(int64_t rows, int64_t width) {
    BackShape b{1024, 0, 1};
    // two units a lane: 128 registers, four wavefronts a SIMD.  One unit and twice the lanes is 5 % slower at 1,024 to
    // 4,096, four units and half the lanes 30 % at 7,380.
    if (width <= 128) b = {16, 1, 1};
    else if (width <= 256) b = {32, 1, 1};
    else if (width <= 512) b = {64, 1, 1};
    else if (width <= 1024) b = {64, 2, 1};
    else if (width <= 2048) b = {128, 2, 1};
    else if (width <= 4096) b = {256, 2, 1};
    else if (width <= 8192) b = {512, 2, 1};
    else if (width <= 16384) b = {1024, 2, 1};
    const int64_t in_hand = std::max(1, 256 / b.lanes);
    const int64_t most = 262144 / std::max(256, b.lanes); // that the device holds at once: four wavefronts a SIMD
    // a few rows: one workgroup, whose share is the gradient itself, and no second launch
    b.groups = rows <= 2 * in_hand && b.units > 0 ? 1 : std::min<int64_t>((rows + in_hand - 1) / in_hand, most);
    return b;
}

template <typename T, int Lanes, int Units> void launch_back(const BackView& a, int64_t groups, hipStream_t s) {
    k_norm_back<T, Lanes, Units><<<dim3(unsigned(groups)), Lanes > 256 ? Lanes : 256, 0, s>>>(a);
    MDX_HIP(hipGetLastError());
}

template <typename T> void choose_back(const BackView& a, const BackShape& b, hipStream_t s) {
    switch (b.lanes * 8 + b.units) {
        case 16 * 8 + 1: return launch_back<T, 16, 1>(a, b.groups, s);
        case 32 * 8 + 1: return launch_back<T, 32, 1>(a, b.groups, s);
        case 64 * 8 + 1: return launch_back<T, 64, 1>(a, b.groups, s);
        case 64 * 8 + 2: return launch_back<T, 64, 2>(a, b.groups, s);
        case 128 * 8 + 2: return launch_back<T, 128, 2>(a, b.groups, s);
        case 256 * 8 + 2: return launch_back<T, 256, 2>(a, b.groups, s);
        case 512 * 8 + 2: return launch_back<T, 512, 2>(a, b.groups, s);
        case 1024 * 8 + 2: return launch_back<T, 1024, 2>(a, b.groups, s);
        default: break;
    }
    const dim3 strips(unsigned((a.width + 2047) / 2048), unsigned(b.groups));
    k_norm_gain_long<T><<<strips, 256, 0, s>>>(a);
    MDX_HIP(hipGetLastError());
    in_runs(a.rows, 1024, [&](int64_t first, int64_t count) {
        BackView part = a;
        part.rows = count;
        part.grad = static_cast<const T*>(a.grad) + first * a.grad_pitch;
        part.t = static_cast<const T*>(a.t) + first * a.t_pitch;
        if (a.grad_total != nullptr) part.grad_total = static_cast<const T*>(a.grad_total) + first * a.grad_total_pitch;
        part.rstd = a.rstd + first;
        part.grad_x = static_cast<T*>(a.grad_x) + first * a.grad_x_pitch;
        k_norm_back_long<T><<<dim3(unsigned(count)), 1024, 0, s>>>(part);
        MDX_HIP(hipGetLastError());
    });
}

template <int Cols>
void launch_gain(const float* part, int64_t parts, int64_t width, float* out, hipStream_t s) {
    in_runs((width + Cols - 1) / Cols, 1024, [&](int64_t first, int64_t count) {
        k_norm_gain<Cols><<<dim3(unsigned(count)), 1024, 0, s>>>(part, parts, width, out, first);
        MDX_HIP(hipGetLastError());
    });
}

} // namespace

void rms_norm(const mdx_norm_args& g, hipStream_t s) {
    const bool codes = g.out_dtype == MDX_FLOAT8;
    // The eight L2s hold 32 MB: more results than that only push out what is being read (65,536 x 1,024 bfloat16 with a
    // residual 70 us, 86 through the L2; x 3,696 float32 225 and 231).  The gradients, the quantisation and the AdamW
    // step gain nothing by it.
    const int64_t size = g.dtype == MDX_FLOAT32 ? 4 : 2;
    const bool past = g.rows * g.width * ((codes ? 1 : size) + (g.total != nullptr ? size : 0)) > (int64_t(32) << 20);
    const NormView a{g.rows, g.width, g.x, g.x_pitch, g.residual, g.residual_pitch, g.gain, g.values, g.values_pitch,
               g.scales, g.scales_pitch, g.total, g.total_pitch, g.rstd, float(g.eps)};
    if (g.dtype == MDX_FLOAT32) codes ? choose_norm<float, true>(a, past, s) : choose_norm<float, false>(a, past, s);
    else if (g.dtype == MDX_BFLOAT16) codes ? choose_norm<__bf16, true>(a, past, s) : choose_norm<__bf16, false>(a, past, s);
    else codes ? choose_norm<_Float16, true>(a, past, s) : choose_norm<_Float16, false>(a, past, s);
}

int64_t rms_norm_backward_workspace(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const int64_t groups = back_shape(rows, width).groups;
    return groups == 1 ? 0 : groups * width * int64_t(sizeof(float));
}

void rms_norm_backward(const mdx_norm_backward_args& g, hipStream_t s) {
    const BackShape b = back_shape(g.rows, g.width);
    const BackView a{g.rows, g.width, g.grad, g.grad_pitch, g.t, g.t_pitch, g.grad_total, g.grad_total_pitch, g.gain,
                     g.rstd, g.grad_x, g.grad_x_pitch, b.groups == 1 ? g.grad_gain : static_cast<float*>(g.workspace)};
    if (g.rows > 0) {
        if (g.dtype == MDX_FLOAT32) choose_back<float>(a, b, s);
        else if (g.dtype == MDX_BFLOAT16) choose_back<__bf16>(a, b, s);
        else choose_back<_Float16>(a, b, s);
    }
    if (g.rows > 0 && b.groups == 1) return;
    // a sum over no rows is zero
    const int64_t parts = g.rows > 0 ? b.groups : 0;
    // few columns: more workgroups of fewer (50,225 x 176 bfloat16, both launches: 16.9 us, 17.7 with 32 columns each)
    if (g.width <= 512) launch_gain<8>(a.part, parts, g.width, g.grad_gain, s);
    else launch_gain<32>(a.part, parts, g.width, g.grad_gain, s);
}

} // namespace mdx
