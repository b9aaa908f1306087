// kd_f8_rows.hip - rows into 8 bits (include/kd_f8.h): e4m3 codes with one
// E8M0 scale for each block of 128 values.
//
//   quantize_kernel  rows of F32, BF16 or F16
//   norm_kernel      residual addition and RMS norm (RMSNorm,
//                    src/core/module.hpp:163-180), its output in 8 bits
//
// In both a thread holds 8 consecutive values, so that the 16 lanes of a
// DPP row hold one block: its largest magnitude takes four DPP steps, and
// the scale and the codes follow without LDS.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/kd_f8.h"
#include "kd_f8_kernel.h"
#include "kd_fa_device.h"

namespace kdfa {

// Eight values as loaded, and as F32.
template <int TYPE> struct F8Src;
template <> struct F8Src<KD_F8_TYPE_F32> {
    f32x4 u, v;
    __device__ __forceinline__ void load(const char *row, int col) {
        u = *reinterpret_cast<const f32x4 *>(row + (int64_t)col * 4);
        v = *reinterpret_cast<const f32x4 *>(row + (int64_t)col * 4 + 16);
    }
    __device__ __forceinline__ void get(float y[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { y[e] = u[e]; y[4 + e] = v[e]; }
    }
    // F32 rounds to itself
    static __device__ __forceinline__ void round_store(char *row, int col, float y[8], bool in) {
        if (in) {
            *reinterpret_cast<f32x4 *>(row + (int64_t)col * 4) = (f32x4){y[0], y[1], y[2], y[3]};
            *reinterpret_cast<f32x4 *>(row + (int64_t)col * 4 + 16) = (f32x4){y[4], y[5], y[6], y[7]};
        }
    }
};
template <> struct F8Src<KD_F8_TYPE_BF16> {
    u32x4 w;
    __device__ __forceinline__ void load(const char *row, int col) { w = ld16(row + (int64_t)col * 2); }
    __device__ __forceinline__ void get(float y[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { y[2 * e] = bf16_lo(w[e]); y[2 * e + 1] = bf16_hi(w[e]); }
    }
    static __device__ __forceinline__ void round_store(char *row, int col, float y[8], bool in) {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] = Elem<__bf16>::pack2(y[2 * e], y[2 * e + 1]);
            y[2 * e] = bf16_lo(o[e]);
            y[2 * e + 1] = bf16_hi(o[e]);
        }
        if (in) *reinterpret_cast<u32x4 *>(row + (int64_t)col * 2) = o;
    }
};
template <> struct F8Src<KD_F8_TYPE_F16> {
    u32x4 w;
    __device__ __forceinline__ void load(const char *row, int col) { w = ld16(row + (int64_t)col * 2); }
    __device__ __forceinline__ void get(float y[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { y[2 * e] = f16_lo(w[e]); y[2 * e + 1] = f16_hi(w[e]); }
    }
};

// the larger of x and x of the lane that DPP control CTRL names
template <int CTRL>
static __device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
    return x > o ? x : o;
}

// the sum over each LANES (16, 32 or 64) lanes, in every lane: of 16 by DPP,
// then by swaps of rows of 16 and of 32 (a shuffle through LDS takes its
// latency each step)
template <int CTRL>
static __device__ __forceinline__ double add_dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return x + __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
template <int LANES>
static __device__ __forceinline__ double lane_sum(double x) {
    x = add_dpp<0xb1>(x);    // lane ^ 1
    x = add_dpp<0x4e>(x);    // lane ^ 2
    x = add_dpp<0x141>(x);   // 7 - lane of each 8
    x = add_dpp<0x140>(x);   // 15 - lane
    if constexpr (LANES >= 32) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        x = __builtin_bit_cast(double, (uint64_t)lo[0] | ((uint64_t)hi[0] << 32)) +
            __builtin_bit_cast(double, (uint64_t)lo[1] | ((uint64_t)hi[1] << 32));
    }
    if constexpr (LANES >= 64) x = pair_sum_f64(x);
    return x;
}

// 1 / sqrt(v) of v >= 0 within 2^-50: v_rsq_f64 and two steps of Newton's
// method, each of which squares its error (a division and a square root in
// double are three times the instructions).  0 of infinity.
static __device__ __forceinline__ double rsqrt_f64(double v) {
    double r = __builtin_amdgcn_rsq(v);
#pragma unroll
    for (int n = 0; n < 2; ++n) r = __builtin_fma(r, __builtin_fma(-0.5 * v * r, r, 0.5), r);
    return __builtin_isinf(v) ? 0.0 : r;
}

// Eight values of a block (its 16 lanes call together) as codes; the block's
// scale byte.  Magnitudes are compared as bits, where NaN is above infinity
// and infinity above every number.  max|y| = f * 2^E with 1 <= f < 2: 2^e is
// 2^(E - 8) for f <= 1.75 (448 = 1.75 * 2^8), else 2^(E - 7): adding
// 0x1fffff to the bits carries into the exponent for f > 1.75 alone.  A
// magnitude with an exponent field below 8 takes byte 0, so does zero.  2^-e
// is a normal number for every byte up to 247, the largest number's, and the
// product by it is exact (what underflows is far below half a code), so that
// the conversion's is the only rounding.
static __device__ __forceinline__ u32x2 to_f8(const float y[8], uint32_t &byte) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    m = max_dpp<0xb1>(m);    // lane ^ 1
    m = max_dpp<0x4e>(m);    // lane ^ 2
    m = max_dpp<0x141>(m);   // 7 - lane of each 8
    m = max_dpp<0x140>(m);   // 15 - lane
    const uint32_t f = (m + 0x1fffffu) >> 23;
    const bool bad = m >= 0x7f800000u;
    byte = bad ? 255u : (f > 8 ? f - 8 : 0);
    const float inv = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - byte) << 23);
    u32x2 c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int w = 0;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h] * inv, y[4 * h + 1] * inv, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2] * inv, y[4 * h + 3] * inv, w, true);
        c[h] = (uint32_t)w;
    }
    return c;
}

// ---------------------------------------------------------------------------
// quantize_kernel: bound by HBM (16,000 x 16384 BF16: 137 us, 5.7 TB/s; 4096
// x 4096 F16 10 us).  16 lanes take a block; the blocks of all
// rows are counted through, 64 to a workgroup, four of them (64 bytes of
// 16-bit x a lane) loaded before the first is stored.
// ---------------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(256) void quantize_kernel(F8RowsArgs a) {
    constexpr int kU = kF8QuantBlocks / 16;
    const int lane16 = threadIdx.x & 15;
    const int team = threadIdx.x >> 4;
    const float rcp = 1.0f / (float)a.blocks;
    const int64_t total = (int64_t)a.M * a.blocks;
    for (int64_t t0 = (int64_t)blockIdx.x * kF8QuantBlocks; t0 < total; t0 += (int64_t)gridDim.x * kF8QuantBlocks) {
        const int64_t row0 = (int64_t)((uint64_t)t0 / (uint32_t)a.blocks);
        const int rem0 = (int)(t0 - row0 * a.blocks);
        F8Src<TYPE> s[kU];
        int64_t row[kU];
        int col[kU], blk[kU];
        bool in[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = 16 * u + team;
            // past the end, the last block again (not stored)
            const int j = t0 + i < total ? i : (int)(total - 1 - t0);
            const int r = div_small(rem0 + j, a.blocks, rcp);
            row[u] = row0 + r;
            blk[u] = rem0 + j - r * a.blocks;
            col[u] = blk[u] * kF8Block + 8 * lane16;
            in[u] = col[u] < a.K;
            s[u].load(a.x + row[u] * a.x_nb1, in[u] ? col[u] : 0);
            in[u] = in[u] && t0 + i < total;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float y[8];
            s[u].get(y);
            if (col[u] >= a.K) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = 0.0f;
            }
            uint32_t byte;
            const u32x2 c = to_f8(y, byte);
            if (in[u]) {
                *reinterpret_cast<u32x2 *>(a.codes + row[u] * a.c_nb1 + col[u]) = c;
                if (lane16 == 0) a.scales[row[u] * a.e_nb1 + blk[u]] = (char)byte;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// norm_kernel: LANES lanes of a wave to a row of up to 8 LANES values, or
// (LANES = 0) a workgroup to a row, C chunks of 8 values a thread; the whole
// row in registers between its one reading and its writing.  Bound by HBM for
// many rows (63,488 x 4096, BF16 onto an F32 stream, 2.86 GB: 0.52 ms, 5.5
// TB/s, what a copy reaches), by one row's latency for few (2 x 3584: 2.8 us).
// A code is a rounding to 4 bits, and a value next to its border goes to the
// wrong side by an error of the value's last bits: so the squares are summed in
// double and each value of the norm is rounded once (both under the loads).
// ---------------------------------------------------------------------------
template <int XT, int ST, bool RES, int LANES, int C>
__global__ __launch_bounds__(LANES ? 256 : 1024) void norm_kernel(F8RowsArgs a) {
    constexpr int kRows = LANES ? 256 / LANES : 1;   // rows at once in a workgroup
    __shared__ double part[2][16];
    const int T = LANES ? LANES : blockDim.x;
    const int tid = LANES ? threadIdx.x % LANES : threadIdx.x;
    const int lane = threadIdx.x & 63;
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.M; base += (int64_t)gridDim.x * kRows) {
        // past the end, the last row again (not stored)
        const int64_t mine = base + (LANES ? threadIdx.x / LANES : 0);
        const bool live = mine < a.M;
        const int64_t row = live ? mine : a.M - 1;
        F8Src<XT> x[C];
        F8Src<ST> r[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = 8 * (tid + T * c);
            x[c].load(a.x + row * a.x_nb1, col < a.K ? col : 0);
            if constexpr (RES) r[c].load(a.residual + row * a.r_nb1, col < a.K ? col : 0);
        }
        // the weights with them, where registers are plenty: few rows' latency
        f32x4 w0[C], w1[C];
        auto load_weight = [&](int c) __attribute__((always_inline)) {
            const int col = 8 * (tid + T * c);
            w0[c] = *reinterpret_cast<const f32x4 *>(a.weight + (col < a.K ? col : 0));
            w1[c] = *reinterpret_cast<const f32x4 *>(a.weight + (col < a.K ? col : 0) + 4);
        };
        if constexpr (C <= 2) {
#pragma unroll
            for (int c = 0; c < C; ++c) load_weight(c);
        }
        float y[C][8];
        double ss = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = 8 * (tid + T * c);
            const bool in = col < a.K;
            x[c].get(y[c]);
            if constexpr (RES) {
                float z[8];
                r[c].get(z);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[c][e] += z[e];
                F8Src<ST>::round_store(a.sum + row * a.s_nb1, col, y[c], in && live);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[c][e] = in ? y[c][e] : 0.0f;
                ss += (double)y[c][e] * (double)y[c][e];
            }
        }
        ss = lane_sum<LANES ? LANES : 64>(ss);
        if constexpr (LANES == 0) {
            // two buffers in turn: a row's partial sums are read before the
            // next row's barrier, the row after that writes over them behind it
            if (lane == 0) part[turn][threadIdx.x >> 6] = ss;
            __syncthreads();
            ss = lane_sum<16>((lane & 15) < T >> 6 ? part[turn][lane & 15] : 0.0);
            turn ^= 1;
        }
        // 1 / rms as the sum of two F32; of rows so small or large that these
        // would not be normal numbers, 2^100 goes over to y (exact, but for
        // what is nothing beside the row's largest)
        double rstd = rsqrt_f64(__builtin_fma(ss, a.inv_k, (double)a.eps));
        if (!(rstd >= 0x1p-100 && rstd <= 0x1p100)) {
            const float up = rstd > 1.0 ? 0x1p100f : 0x1p-100f;
            rstd *= rstd > 1.0 ? 0x1p-100 : 0x1p100;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) y[c][e] *= up;
        }
        float r0 = (float)rstd;
        if ((double)r0 > rstd) r0 = __uint_as_float(__float_as_uint(r0) - 1);   // (r1 >= 0)
        const float r1 = (float)(rstd - (double)r0);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = 8 * (tid + T * c);
            const bool in = col < a.K;
            if constexpr (C > 2) load_weight(c);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // y / rms * weight, rounded once: the product with what its
                // rounding left (a zero with the product's sign, so that -0
                // stays what it is)
                const float w = e < 4 ? w0[c][e] : w1[c][e - 4], p = y[c][e] * r0;
                const float q = __builtin_fmaf(y[c][e], r1, -__builtin_fmaf(-y[c][e], r0, p));
                v[e] = in ? __builtin_fmaf(p, w, q * w) : 0.0f;
            }
            uint32_t byte;
            const u32x2 q = to_f8(v, byte);
            if (in && live) {
                *reinterpret_cast<u32x2 *>(a.codes + row * a.c_nb1 + col) = q;
                if ((tid & 15) == 0) a.scales[row * a.e_nb1 + (col >> 7)] = (char)byte;
            }
        }
    }
}

hipError_t launch_f8_quantize(const F8RowsArgs &a, hipStream_t s) {
    const int64_t want = ((int64_t)a.M * a.blocks + kF8QuantBlocks - 1) / kF8QuantBlocks;
    const dim3 grid((unsigned)(want < (1 << 22) ? want : 1 << 22));
    if (a.x_type == KD_F8_TYPE_F32)
        hipLaunchKernelGGL((quantize_kernel<KD_F8_TYPE_F32>), grid, dim3(256), 0, s, a);
    else if (a.x_type == KD_F8_TYPE_BF16)
        hipLaunchKernelGGL((quantize_kernel<KD_F8_TYPE_BF16>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((quantize_kernel<KD_F8_TYPE_F16>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int XT, int ST, bool RES, int LANES, int C>
static void launch_norm_c(const F8RowsArgs &a, hipStream_t s) {
    constexpr int kRows = LANES ? 256 / LANES : 1;
    const int64_t want = ((int64_t)a.M + kRows - 1) / kRows;
    const dim3 grid((unsigned)(want < (1 << 20) ? want : 1 << 20));
    const int threads = LANES ? 256 : (a.K + 512 * C - 1) / (512 * C) * 64;
    hipLaunchKernelGGL((norm_kernel<XT, ST, RES, LANES, C>), grid, dim3(threads), 0, s, a);
}

template <int XT, int ST, bool RES>
static void launch_norm_t(const F8RowsArgs &a, hipStream_t s) {
    // as few values a thread as a workgroup allows: at any number of rows no
    // slower than a wave to a row, which 2 rows of 3,584 take 5.5 us and 8,192
    // rows 72 (here 2.8 and 63).  What a wave does once a row is half of its
    // instructions, and they bind where lanes are idle: so no more lanes than
    // have values (63,488 rows of F32: 128 long 7.9 us on 16 lanes, 22.7 on 64;
    // 528 long 37 on two waves, 80 on four)
    if (a.K <= 128) launch_norm_c<XT, ST, RES, 16, 1>(a, s);
    else if (a.K <= 256) launch_norm_c<XT, ST, RES, 32, 1>(a, s);
    else if (a.K <= 512) launch_norm_c<XT, ST, RES, 64, 1>(a, s);
    else if (a.K <= 8192) launch_norm_c<XT, ST, RES, 0, 1>(a, s);
    else if (a.K <= 16384) launch_norm_c<XT, ST, RES, 0, 2>(a, s);
    else launch_norm_c<XT, ST, RES, 0, 4>(a, s);
}

hipError_t launch_f8_norm(const F8RowsArgs &a, hipStream_t s) {
    const bool f32 = a.x_type == KD_F8_TYPE_F32;
    constexpr int F = KD_F8_TYPE_F32, B = KD_F8_TYPE_BF16;
    if (!a.residual)
        f32 ? launch_norm_t<F, F, false>(a, s) : launch_norm_t<B, B, false>(a, s);
    else if (a.s_type == F)
        f32 ? launch_norm_t<F, F, true>(a, s) : launch_norm_t<B, F, true>(a, s);
    else
        f32 ? launch_norm_t<F, B, true>(a, s) : launch_norm_t<B, B, true>(a, s);
    return hipGetLastError();
}

}  // namespace kdfa
