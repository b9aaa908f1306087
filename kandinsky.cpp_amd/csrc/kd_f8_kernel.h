// kd_f8_kernel.h - launch arguments shared by the host glue (kd_f8_host.cpp)
// and the gfx950 kernels of the 8-bit linear path (kd_f8_rows.hip,
// kd_f8_mm.hip).  Internal to libkd_fa.so.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kdfa {

constexpr int kF8Block = 128;   // values of one scale

// Rows into 8 bits: quantize_kernel (x only) and norm_kernel.
struct F8RowsArgs {
    const char *x;          // rows of x, stride x_nb1 bytes
    const char *residual;   // norm: or nullptr
    const float *weight;    // norm
    char *sum;              // norm: with residual
    char *codes;            // [M][K]
    char *scales;           // [M][blocks]
    int64_t x_nb1, r_nb1, s_nb1, c_nb1, e_nb1;
    int32_t x_type, s_type; // KD_F8_TYPE_* of x; of residual and sum
    int32_t M, K, blocks;
    float eps;
    double inv_k;           // norm: 1 / K
};

constexpr int kF8NormMaxK = 32768;
constexpr int kF8QuantBlocks = 64;   // blocks of 128 values per workgroup of quantize_kernel
hipError_t launch_f8_quantize(const F8RowsArgs &a, hipStream_t stream);
hipError_t launch_f8_norm(const F8RowsArgs &a, hipStream_t stream);

struct F8MmArgs {
    const char *w, *x;      // code rows [N][K], [M][K]
    const char *ws, *xs;    // scale rows
    const float *bias;      // F32 [N] or nullptr
    char *dst;              // BF16 rows [M][N]
    int64_t w_nb1, x_nb1, ws_nb1, xs_nb1, d_nb1;
    int32_t M, N, K;
    int32_t tiles_m, tiles_n, n_blocks, cols;
    int32_t lines;          // f8_mm_ring's and f8_mm_grid's LINES
};

constexpr int64_t kF8MmMaxBlocks = 1 << 23;   // workgroups of 256 threads in one launch, with room to spare
// Tiles of 16 * (tile / 100 % 100) outputs x 16 * (tile % 100) tokens: below
// 10000 f8_mm_ring's, above f8_mm_grid's, 11616 f8_mm_tile's.
hipError_t launch_f8_mm(const F8MmArgs &a, int tile, hipStream_t stream);

}  // namespace kdfa
