// Float8 codes with one power-of-two scale per block of 128, or 128 x 128.
//
// The matrix is read once and written once at a quarter or half its size:
// the kernels are bound by HBM.  Sixteen lanes hold the 128 elements of a
// row's block, so its maximum stays in a DPP row; a 128 x 128 tile stays in a
// workgroup's registers until its maxima are known.  65,536 x 3,696 float32 takes
// 214 us (5.7 TB/s), its transpose 255 us (4.8); 65,536 x 1,024 bfloat16 34 us
// either way (6.0, the memory-side cache holds part of it).
#include "rows_device.h"

#include <algorithm>

#include "rows_internal.h"

namespace mdx {
namespace {

using namespace rows;

struct QuantizeView {
    int64_t rows, width;
    const void* x;
    int64_t x_pitch;
    uint8_t* codes;
    int64_t codes_pitch;
    uint8_t* scales;
    int64_t scales_pitch;
};

// One scale per row and block: sixteen lanes a block, one unit a lane.
template <typename T> __global__ __launch_bounds__(256) void k_quantize_rows(const QuantizeView a, int64_t blocks, int64_t first) {
    const int64_t at = ((first + int64_t(blockIdx.x)) * 256 + threadIdx.x) / 16;
    if (at >= a.rows * blocks) return;
    const int64_t row = at / blocks, block = at - row * blocks;
    const int64_t col = block * kScaleBlock + (threadIdx.x % 16) * kUnit;
    float v[kUnit];
    load_unit(static_cast<const T*>(a.x) + row * a.x_pitch, col, a.width, v);
    const int byte = scale_byte(row_max(unit_max(v)));
    *reinterpret_cast<u2*>(a.codes + row * a.codes_pitch + col) = unit_codes(v, byte);
    if (threadIdx.x % 16 == 0) a.scales[row * a.scales_pitch + block] = uint8_t(byte);
}

// A tile of 128 x 128 per workgroup: lane (p, q) = (t / 16, t % 16) holds Rows
// rows from Rows p on and columns 8q..8q+7.  Whole: one scale for the tile,
// else one per column (the result is the transpose, whose rows are the
// columns).  Turned: the codes are written transposed.
//
// The transpose goes through 16 KB of LDS, four rows of one column at a time:
// the 16 bytes of rows 16g..16g+15 of column c lie at place g ^ (c / 8 % 8), so
// that lanes which write together use different banks.
template <typename T, bool Whole, bool Turned, int Rows>
__global__ __launch_bounds__(16 * kScaleBlock / Rows) void k_quantize_tile(const QuantizeView a) {
    static_assert(Whole || Turned, "rows of 128 have a kernel of their own");
    static_assert(!Turned || Rows == 4, "the transpose moves four rows at a time");
    constexpr int kWaves = 16 * kScaleBlock / Rows / kWave;
    __shared__ uint32_t most[kWaves][Whole ? 1 : kScaleBlock];
    __shared__ __align__(16) uint8_t turned[Turned ? kScaleBlock * kScaleBlock : 16];
    const int p = threadIdx.x / 16, q = threadIdx.x % 16, wave = threadIdx.x / kWave;
    const int64_t row0 = int64_t(blockIdx.y) * kScaleBlock, col0 = int64_t(blockIdx.x) * kScaleBlock;
    const int64_t col = col0 + q * kUnit;
    float v[Rows][kUnit];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int64_t row = row0 + p * Rows + r;
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[r][i] = 0.0f;
        if (row < a.rows) load_unit(static_cast<const T*>(a.x) + row * a.x_pitch, col, a.width, v[r]);
    }
    uint32_t m[kUnit];
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        m[i] = 0;
#pragma unroll
        for (int r = 0; r < Rows; ++r) m[i] = max(m[i], size_bits(v[r][i]));
        if constexpr (!Whole) {
            m[i] = across_max(m[i]);
        }
    }
    int byte[kUnit];
    if constexpr (Whole) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kUnit; ++i) top = max(top, m[i]);
        top = across_max(row_max(top));
        if (threadIdx.x % kWave == 0) most[wave][0] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = max(top, most[w][0]);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) byte[i] = scale_byte(top);
        if (threadIdx.x == 0) {
            uint8_t* to = Turned ? a.scales + int64_t(blockIdx.x) * a.scales_pitch + blockIdx.y
                                 : a.scales + int64_t(blockIdx.y) * a.scales_pitch + blockIdx.x;
            *to = uint8_t(byte[0]);
        }
    } else {
        __shared__ __align__(8) uint8_t bytes[kScaleBlock];
        if (threadIdx.x % kWave < 16) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) most[wave][q * kUnit + i] = m[i];
        }
        __syncthreads();
        if (threadIdx.x < kScaleBlock) { // a lane a column
            const int c = threadIdx.x;
            uint32_t top = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = max(top, most[w][c]);
            bytes[c] = uint8_t(scale_byte(top));
            if (col0 + c < a.width) a.scales[(col0 + c) * a.scales_pitch + blockIdx.y] = bytes[c];
        }
        __syncthreads();
        const u2 mine = *reinterpret_cast<const u2*>(&bytes[q * kUnit]);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) byte[i] = int(mine[i / 4] >> (8 * (i % 4)) & 255u);
    }
    if constexpr (!Turned) {
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const int64_t row = row0 + p * Rows + r;
            if (row < a.rows)
                *reinterpret_cast<u2*>(a.codes + row * a.codes_pitch + col) = unit_codes(v[r], byte[0]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const int c = q * kUnit + i;
            *reinterpret_cast<uint32_t*>(&turned[c * kScaleBlock + ((p / 4) ^ (q % 8)) * 16 + p % 4 * 4]) =
                four_codes(v[0][i], v[1][i], v[2][i], v[3][i], byte[i]);
        }
        __syncthreads();
        // eight lanes a column of the tile, sixteen of its rows each
        constexpr int kThreads = kWaves * kWave;
#pragma unroll
        for (int k = 0; k < kScaleBlock * 8 / kThreads; ++k) {
            const int c = k * (kThreads / 8) + threadIdx.x / 8, piece = threadIdx.x % 8;
            if (col0 + c >= a.width) continue;
            *reinterpret_cast<u4*>(a.codes + (col0 + c) * a.codes_pitch + row0 + piece * 16) =
                *reinterpret_cast<const u4*>(&turned[c * kScaleBlock + (piece ^ (c / 8 % 8)) * 16]);
        }
    }
}

template <typename T> void choose_quantize(const QuantizeView& a, bool whole, bool turned, hipStream_t s) {
    const int64_t across = (a.width + kScaleBlock - 1) / kScaleBlock, down = (a.rows + kScaleBlock - 1) / kScaleBlock;
    if (!whole && !turned) {
        in_runs((a.rows * across + 15) / 16, 256, [&](int64_t first, int64_t count) {
            k_quantize_rows<T><<<dim3(unsigned(count)), 256, 0, s>>>(a, across, first);
            MDX_HIP(hipGetLastError());
        });
        return;
    }
    constexpr int64_t kMostDown = 32768; // tiles in the grid's second dimension
    for (int64_t first = 0; first < down; first += kMostDown) {
        QuantizeView b = a;
        const int64_t skip = first * kScaleBlock;
        b.x = static_cast<const T*>(a.x) + skip * a.x_pitch;
        b.rows = std::min<int64_t>(a.rows - skip, kMostDown * kScaleBlock);
        b.codes = a.codes + (turned ? skip : skip * a.codes_pitch);
        b.scales = a.scales + (turned ? first : (whole ? first : skip) * a.scales_pitch);
        in_runs(across, 1024, [&](int64_t left, int64_t count) {
            QuantizeView c = b;
            const int64_t over = left * kScaleBlock;
            c.x = static_cast<const T*>(b.x) + over;
            c.width = std::min<int64_t>(b.width - over, count * kScaleBlock);
            c.codes = b.codes + (turned ? over * b.codes_pitch : over);
            c.scales = b.scales + (turned ? (whole ? left : over) * b.scales_pitch : left);
            const dim3 grid(unsigned(count), unsigned((b.rows + kScaleBlock - 1) / kScaleBlock));
            // many lanes a tile: 1,024 x 3,696 has fewer tiles than the device CUs (whole tiles 4.6 us, 7.0 with 256 lanes)
            if (whole && turned) k_quantize_tile<T, true, true, 4><<<grid, 512, 0, s>>>(c);
            else if (whole) k_quantize_tile<T, true, false, 2><<<grid, 1024, 0, s>>>(c);
            else k_quantize_tile<T, false, true, 4><<<grid, 512, 0, s>>>(c);
            MDX_HIP(hipGetLastError());
        });
    }
}

} // namespace

void quantize_fp8(const mdx_quantize_args& g, hipStream_t s) {
    const QuantizeView a{g.rows, g.width, g.x, g.x_pitch, g.codes, g.codes_pitch, g.scales, g.scales_pitch};
    const bool whole = g.tile == kScaleBlock, turned = g.transpose != 0;
    if (g.dtype == MDX_FLOAT32) choose_quantize<float>(a, whole, turned, s);
    else if (g.dtype == MDX_BFLOAT16) choose_quantize<__bf16>(a, whole, turned, s);
    else choose_quantize<_Float16>(a, whole, turned, s);
}

} // namespace mdx
