// The operators behind the C ABI: arguments are checked by their entry
// points (rows_api.hip), rows and widths are over zero here.
#pragma once

#include <algorithm>

#include "mdx_internal.h"

namespace mdx {

// A grid takes fewer than 2^32 lanes along a dimension.  Work that needs more
// goes in several launches of 2^28 each: such a launch takes long enough
// (a millisecond for the fastest kernel here) for the next one's cost not to show.
constexpr int64_t kLaunchLanes = int64_t(1) << 28;

// Calls launch(first, count) over runs of `groups` workgroups of `threads` lanes.
template <typename Launch> void in_runs(int64_t groups, int threads, Launch&& launch) {
    const int64_t most = kLaunchLanes / threads;
    for (int64_t first = 0; first < groups; first += most) launch(first, std::min(groups - first, most));
}

constexpr int64_t kAdamwChunk = 2048; // elements per workgroup of the AdamW step
constexpr int64_t kAdamwMost = ((int64_t(1) << 24) - 1) * kAdamwChunk; // of a tensor: one launch of 256 lanes a chunk

void rms_norm(const mdx_norm_args& args, hipStream_t stream);
int64_t rms_norm_backward_workspace(int64_t rows, int64_t width);
void rms_norm_backward(const mdx_norm_backward_args& args, hipStream_t stream);
void quantize_fp8(const mdx_quantize_args& args, hipStream_t stream);
int64_t matmul_fp8_workspace(const mdx_matmul_args& args);
void matmul_fp8(const mdx_matmul_args& args, hipStream_t stream);
void adamw_step(const mdx_adamw_args& args, const int64_t* step_at, const int64_t* seed_at, hipStream_t stream);

// Calls run() and turns what it throws into a status and this thread's last error.
int guarded_call(const std::function<void()>& run);

} // namespace mdx
