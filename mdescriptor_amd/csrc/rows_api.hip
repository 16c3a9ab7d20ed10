// The extern "C" boundary of the operators on feature rows (declared in
// include/mdx_hip.h): arguments are checked against what the kernels assume,
// then the kernels are queued on the caller's stream.  Nothing is allocated
// and no call waits, so each may be captured into a graph.
#include "rows_device.h"

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "rows_internal.h"

namespace {

using mdx::Error;

void require(bool holds, const char* message) {
    if (!holds) throw Error(MDX_INVALID_ARGUMENT, message);
}

// The stream's device for the time of a call.
struct OnDevice {
    int previous = -1, device;
    explicit OnDevice(int d) : device(d) {
        MDX_HIP(hipGetDevice(&previous));
        if (previous != device) MDX_HIP(hipSetDevice(device));
    }
    ~OnDevice() {
        if (previous >= 0 && previous != device) (void)hipSetDevice(previous);
    }
};

constexpr int64_t kMostRows = int64_t(1) << 31; // with widths below 2^31 too, products of two sizes fit 64 bits
constexpr int64_t kMostWidth = int64_t(1) << 31;
constexpr int64_t kMostResults = int64_t(1) << 39; // of a product, so that its bytes do too

int64_t element_size(int32_t dtype) { return dtype == MDX_FLOAT32 ? 4 : dtype == MDX_FLOAT8 ? 1 : 2; }

bool in_range(int64_t rows, int64_t width) {
    return rows >= 0 && width >= 0 && rows < kMostRows && width < kMostWidth;
}

void check_shape(int64_t rows, int64_t width) {
    require(rows >= 0 && width >= 0, "rows and width must not be negative");
    require(rows < kMostRows && width < kMostWidth, "rows and width must be below 2^31");
}

void check_dtype(int32_t dtype) {
    require(dtype == MDX_FLOAT32 || dtype == MDX_BFLOAT16 || dtype == MDX_FLOAT16,
            "the element type must be float32, bfloat16 or float16");
}

void check_matrix(const void* p, int64_t pitch, int64_t width, int32_t dtype, const char* what) {
    if (p == nullptr) throw Error(MDX_INVALID_ARGUMENT, std::string(what) + " must not be null");
    if (pitch < width) throw Error(MDX_INVALID_ARGUMENT, std::string(what) + ": the pitch is below the width");
    if (reinterpret_cast<uintptr_t>(p) % size_t(element_size(dtype)) != 0)
        throw Error(MDX_INVALID_ARGUMENT, std::string(what) + " is not aligned to its elements");
}

void check_codes(const uint8_t* codes, int64_t pitch, int64_t width, const uint8_t* scales, int64_t scales_pitch) {
    require(codes != nullptr && scales != nullptr, "float8 output needs codes and scales");
    require(pitch % 128 == 0 && pitch >= width, "the pitch of written codes must be a multiple of 128");
    require(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "written codes must be 16-byte aligned");
    require(scales_pitch >= (width + 127) / 128, "the pitch of the scales is below their number");
}

// What a step writes may be read or written by its own lanes alone: workgroups run in any order.
void check_apart(const mdx_adamw_args& g) {
    typedef std::pair<uintptr_t, uintptr_t> Range; // bytes from and up to
    std::vector<Range> written;
    written.reserve(size_t(g.count) * 5);
    auto range = [](const void* p, int64_t bytes) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(p);
        return Range(from, from + uintptr_t(bytes));
    };
    const int64_t state = g.bits == 8 ? 1 : 4;
    for (int64_t i = 0; i < g.count; ++i) {
        const mdx_adamw_tensor& x = g.tensors[i];
        if (x.n == 0) continue;
        written.push_back(range(x.params, x.n * 4));
        written.push_back(range(x.first, x.n * state));
        written.push_back(range(x.second, x.n * state));
        if (g.bits == 32) continue;
        written.push_back(range(x.first_scales, (x.n + 127) / 128));
        written.push_back(range(x.second_scales, (x.n + 127) / 128));
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        require(written[i].first >= written[i - 1].second, "a tensor that the step writes is given twice, or overlaps another");
    const int64_t size = element_size(g.grad_dtype);
    for (int64_t i = 0; i < g.count; ++i) {
        const mdx_adamw_tensor& x = g.tensors[i];
        // in the very place of its own tensor each lane reads before it writes
        if (x.n == 0 || (size == 4 && (x.grads == x.params || (state == 4 && (x.grads == x.first || x.grads == x.second)))))
            continue;
        const Range r = range(x.grads, x.n * size);
        const auto after = std::lower_bound(written.begin(), written.end(), Range(r.second, 0)); // the first from its end on
        require(after == written.begin() || std::prev(after)->second <= r.first, "a gradient overlaps what the step writes");
    }
}

} // namespace

extern "C" {

int mdx_hip_rms_norm(int device, const mdx_norm_args* args, void* stream) {
    return mdx::guarded_call([&] {
        require(args != nullptr, "arguments must not be null");
        const mdx_norm_args& g = *args;
        check_shape(g.rows, g.width);
        check_dtype(g.dtype);
        require(g.out_dtype == g.dtype || g.out_dtype == MDX_FLOAT8, "values have the rows' type or float8");
        require(std::isfinite(g.eps) && g.eps > 0.0 && float(g.eps) > 0.0f, "eps must be positive and finite");
        if (g.rows == 0 || g.width == 0) return;
        check_matrix(g.x, g.x_pitch, g.width, g.dtype, "x");
        if (g.residual != nullptr) check_matrix(g.residual, g.residual_pitch, g.width, g.dtype, "residual");
        if (g.total != nullptr) check_matrix(g.total, g.total_pitch, g.width, g.dtype, "total");
        require(g.gain != nullptr, "gain must not be null");
        if (g.out_dtype == MDX_FLOAT8) check_codes(static_cast<uint8_t*>(g.values), g.values_pitch, g.width, g.scales,
                                                   g.scales_pitch);
        else check_matrix(g.values, g.values_pitch, g.width, g.dtype, "values");
        OnDevice on(device);
        mdx::rms_norm(g, static_cast<hipStream_t>(stream));
    });
}

int64_t mdx_hip_rms_norm_backward_workspace(int64_t rows, int64_t width) {
    return in_range(rows, width) ? mdx::rms_norm_backward_workspace(rows, width) : 0;
}

int mdx_hip_rms_norm_backward(int device, const mdx_norm_backward_args* args, void* stream) {
    return mdx::guarded_call([&] {
        require(args != nullptr, "arguments must not be null");
        const mdx_norm_backward_args& g = *args;
        check_shape(g.rows, g.width);
        check_dtype(g.dtype);
        if (g.width == 0) return;
        require(g.grad_gain != nullptr, "grad_gain must not be null");
        if (g.rows > 0) {
            check_matrix(g.grad, g.grad_pitch, g.width, g.dtype, "grad");
            check_matrix(g.t, g.t_pitch, g.width, g.dtype, "t");
            check_matrix(g.grad_x, g.grad_x_pitch, g.width, g.dtype, "grad_x");
            if (g.grad_total != nullptr)
                check_matrix(g.grad_total, g.grad_total_pitch, g.width, g.dtype, "grad_total");
            require(g.gain != nullptr && g.rstd != nullptr, "gain and rstd must not be null");
            const int64_t needed = mdx::rms_norm_backward_workspace(g.rows, g.width);
            require(needed == 0
                        || (g.workspace != nullptr && g.workspace_bytes >= needed
                            && reinterpret_cast<uintptr_t>(g.workspace) % 16 == 0),
                    "the workspace is smaller than mdx_hip_rms_norm_backward_workspace says, or not 16-byte aligned");
        }
        OnDevice on(device);
        mdx::rms_norm_backward(g, static_cast<hipStream_t>(stream));
    });
}

int mdx_hip_quantize_fp8(int device, const mdx_quantize_args* args, void* stream) {
    return mdx::guarded_call([&] {
        require(args != nullptr, "arguments must not be null");
        const mdx_quantize_args& g = *args;
        check_shape(g.rows, g.width);
        check_dtype(g.dtype);
        require(g.tile == 1 || g.tile == 128, "tile must be 1 or 128");
        if (g.rows == 0 || g.width == 0) return;
        check_matrix(g.x, g.x_pitch, g.width, g.dtype, "x");
        check_codes(g.codes, g.codes_pitch, g.transpose ? g.rows : g.width, g.scales, g.scales_pitch);
        OnDevice on(device);
        mdx::quantize_fp8(g, static_cast<hipStream_t>(stream));
    });
}

int64_t mdx_hip_matmul_fp8_workspace(const mdx_matmul_args* args) {
    if (args == nullptr || !in_range(args->m, args->n) || !in_range(args->k, 0)) return 0;
    return args->m * args->n < kMostResults ? mdx::matmul_fp8_workspace(*args) : 0;
}

int mdx_hip_matmul_fp8(int device, const mdx_matmul_args* args, void* stream) {
    return mdx::guarded_call([&] {
        require(args != nullptr, "arguments must not be null");
        const mdx_matmul_args& g = *args;
        check_shape(g.m, g.n);
        check_shape(g.k, 0);
        check_dtype(g.out_dtype);
        require(g.b_tile == 1 || g.b_tile == 128, "b_tile must be 1 or 128");
        require(g.m * g.n < kMostResults, "the result must have fewer than 2^39 elements");
        if (g.m == 0 || g.n == 0) return;
        check_matrix(g.out, g.out_pitch, g.n, g.out_dtype, "out");
        const int64_t blocks = (g.k + 127) / 128;
        if (g.k > 0) {
            check_matrix(g.a, g.a_pitch, g.k, MDX_FLOAT8, "a");
            check_matrix(g.b, g.b_pitch, g.k, MDX_FLOAT8, "b");
            check_matrix(g.a_scales, g.a_scales_pitch, blocks, MDX_FLOAT8, "a_scales");
            check_matrix(g.b_scales, g.b_scales_pitch, blocks, MDX_FLOAT8, "b_scales");
            auto packed = [](const uint8_t* codes, int64_t pitch, const uint8_t* scales, int64_t scales_pitch) {
                return mdx::rows::aligned16(codes, pitch) && scales_pitch % 4 == 0
                    && reinterpret_cast<uintptr_t>(scales) % 4 == 0;
            };
            require(!g.a_packed || packed(g.a, g.a_pitch, g.a_scales, g.a_scales_pitch),
                    "a's rows are not aligned as a packed operand's are");
            require(!g.b_packed || packed(g.b, g.b_pitch, g.b_scales, g.b_scales_pitch),
                    "b's rows are not aligned as a packed operand's are");
        }
        const int64_t needed = mdx::matmul_fp8_workspace(g);
        require(needed == 0
                    || (g.workspace != nullptr && g.workspace_bytes >= needed
                        && reinterpret_cast<uintptr_t>(g.workspace) % 16 == 0),
                "the workspace is smaller than mdx_hip_matmul_fp8_workspace says, or not 16-byte aligned");
        OnDevice on(device);
        mdx::matmul_fp8(g, static_cast<hipStream_t>(stream));
    });
}

int mdx_hip_adamw_step(int device, const mdx_adamw_args* args, void* stream) {
    return mdx_hip_adamw_step_at(device, args, nullptr, nullptr, stream);
}

int mdx_hip_adamw_step_at(int device, const mdx_adamw_args* args, const int64_t* step_at, const int64_t* seed_at,
                          void* stream) {
    return mdx::guarded_call([&] {
        require(args != nullptr, "arguments must not be null");
        const mdx_adamw_args& g = *args;
        check_dtype(g.grad_dtype);
        require(g.bits == 8 || g.bits == 32, "states have 8 or 32 bits");
        require(g.count >= 0 && g.count < kMostRows && (g.count == 0 || g.tensors != nullptr),
                "the tensors must not be null");
        require(step_at != nullptr || g.step >= 1, "step must be at least 1");
        require(reinterpret_cast<uintptr_t>(step_at) % 8 == 0 && reinterpret_cast<uintptr_t>(seed_at) % 8 == 0,
                "step_at and seed_at must be aligned to their numbers");
        require(std::isfinite(g.lr) && g.lr >= 0.0, "lr must be finite and not negative");
        require(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0, "betas must lie in [0, 1)");
        // the kernel multiplies by the device's reciprocal, which is infinite below the normal numbers
        require(std::isfinite(g.eps) && float(g.eps) >= 0x1p-126f, "eps must be finite and at least 2^-126");
        require(std::isfinite(g.weight_decay) && g.weight_decay >= 0.0, "weight_decay must be finite and not negative");
        for (int64_t i = 0; i < g.count; ++i) {
            const mdx_adamw_tensor& x = g.tensors[i];
            require(x.n >= 0 && x.n <= mdx::kAdamwMost, "a tensor's size must lie in [0, 2^35 - 2^11]");
            if (x.n == 0) continue;
            check_matrix(x.params, x.n, x.n, MDX_FLOAT32, "params");
            check_matrix(x.grads, x.n, x.n, g.grad_dtype, "grads");
            check_matrix(x.first, x.n, x.n, g.bits == 8 ? MDX_FLOAT8 : MDX_FLOAT32, "first");
            check_matrix(x.second, x.n, x.n, g.bits == 8 ? MDX_FLOAT8 : MDX_FLOAT32, "second");
            require(g.bits == 32 || (x.first_scales != nullptr && x.second_scales != nullptr),
                    "states in 8 bits need scales");
        }
        check_apart(g);
        OnDevice on(device);
        mdx::adamw_step(g, step_at, seed_at, static_cast<hipStream_t>(stream));
    });
}

} // extern "C"
