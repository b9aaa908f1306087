// kd_f8_mm.hip - the linear-layer product on rows in 8 bits
// (include/kd_f8.h): e4m3 codes with an E8M0 scale for each 128 k, on
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes one block of a row and its
// scale at a time: the scales cost no instruction beside the product, and
// the sums stay in the accumulators over all of k.
//
// The product computes D^T = W X^T (A = W, outputs on M; B = X^T, tokens on
// N), so that each lane ends with 4 consecutive outputs of one token.  A
// fragment is 16 rows x 128 k: lane l holds chunks l / 16 and l / 16 + 4 (of
// 16 bytes) of row l % 16 -- which k stand where is free as long as W and X
// agree, since a row's 128 k share one scale.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/kd_f8.h"
#include "kd_f8_kernel.h"
#include "kd_fa_device.h"

namespace kdfa {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// D += A B, each row's codes times the scale in byte SEL of its word
template <int SEL>
static __device__ __forceinline__ f32x4 mfma_f8(i32x8 a, i32x8 b, f32x4 c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SEL, (int)sa, SEL, (int)sb);
}

static __device__ __forceinline__ i32x8 join(u32x4 lo, u32x4 hi) {
    return (i32x8){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// The tile of a workgroup: XCD-contiguous runs, dealt in columns of `cols`
// output tiles, the token tiles of a column one after another.
static __device__ __forceinline__ void f8_tile(const F8MmArgs &a, int &nt, int &mt) {
    const int pid = blockIdx.x;
    const int per = a.n_blocks >> 3;
    const int lid = pid < per * 8 ? (pid & 7) * per + (pid >> 3) : pid;
    const int64_t area = (int64_t)a.tiles_m * a.cols;
    const int col = (int)(lid / area), rem = (int)(lid - col * area);
    const int width = min(a.cols, a.tiles_n - col * a.cols);
    mt = rem / width;
    nt = col * a.cols + rem - mt * width;
}

// ---------------------------------------------------------------------------
// f8_mm_stream: 16 NB outputs x 16 MB tokens per workgroup, the four waves
// splitting k (whole words of scales, 512 k, each).  A wave computes the
// whole tile over its own k, so nothing that it loads is another wave's: the
// rows go from memory straight into registers, D blocks ahead.  The four
// partial sums meet in LDS, in wave order.
// Rows past N or M are the last row again (not stored); k past K reads the
// row's last 16 bytes, X's then zeroed.
// ---------------------------------------------------------------------------
template <int NB, int MB, int D>
__global__ __launch_bounds__(256) void f8_mm_stream(F8MmArgs a) {
    constexpr int PN = NB * MB <= 16 ? NB : 16 / MB;   // fragments of outputs that are joined at once
    constexpr int kPart = 16 * MB * 16 * PN * 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * kPart];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15;
    const int q4 = lane >> 4;
    int nt, mt;
    f8_tile(a, nt, mt);
    const int n0 = nt * (16 * NB), m0 = mt * (16 * MB);

    uint32_t w_off[NB], x_off[MB], ws_off[NB], xs_off[MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const uint32_t r = (uint32_t)min(16 * i + l16, a.N - 1 - n0);
        w_off[i] = r * (uint32_t)a.w_nb1;
        ws_off[i] = r * (uint32_t)a.ws_nb1;
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const uint32_t r = (uint32_t)min(16 * j + l16, a.M - 1 - m0);
        x_off[j] = r * (uint32_t)a.x_nb1;
        xs_off[j] = r * (uint32_t)a.xs_nb1;
    }
    const char *const wt = a.w + (int64_t)n0 * a.w_nb1;
    const char *const xt = a.x + (int64_t)m0 * a.x_nb1;
    const char *const wst = a.ws + (int64_t)n0 * a.ws_nb1;
    const char *const xst = a.xs + (int64_t)m0 * a.xs_nb1;

    // this wave's groups of four blocks
    const int ng = (int)(((uint32_t)a.K + 511) >> 9);
    const int g0 = (int)((int64_t)wave * ng >> 2), g1 = (int)((int64_t)(wave + 1) * ng >> 2);

    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = (f32x4){};
    u32x4 fw[D][NB][2], fx[D][MB][2];
    auto load = [&](int kt, auto d_c) __attribute__((always_inline)) {
        constexpr int d = decltype(d_c)::value;
        const uint32_t k0 = min((uint32_t)kt * 128 + 16 * q4, (uint32_t)a.K - 16);
        const uint32_t k1 = min((uint32_t)kt * 128 + 16 * q4 + 64, (uint32_t)a.K - 16);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            fw[d][i][0] = ld16(wt + (uint64_t)(w_off[i] + k0));
            fw[d][i][1] = ld16(wt + (uint64_t)(w_off[i] + k1));
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            fx[d][j][0] = ld16(xt + (uint64_t)(x_off[j] + k0));
            fx[d][j][1] = ld16(xt + (uint64_t)(x_off[j] + k1));
        }
    };
    uint32_t sw[NB], sx[MB], nw[NB], nx[MB];
    auto load_scales = [&](int g) __attribute__((always_inline)) {
        const uint32_t o = (uint32_t)min(g, ng - 1) * 4;
#pragma unroll
        for (int i = 0; i < NB; ++i) nw[i] = *reinterpret_cast<const uint32_t *>(wst + (uint64_t)(ws_off[i] + o));
#pragma unroll
        for (int j = 0; j < MB; ++j) nx[j] = *reinterpret_cast<const uint32_t *>(xst + (uint64_t)(xs_off[j] + o));
    };
    // the products of block kt (byte s of the scales' words)
    auto products = [&](int kt, auto s_c, auto end_c) __attribute__((always_inline)) {
        constexpr int s = decltype(s_c)::value, d = s % D;
        // past K the scales' bytes are anything, NaN too
        if (decltype(end_c)::value && kt * 128 >= a.K) return;
        i32x8 b[MB];
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            u32x4 lo = fx[d][j][0], hi = fx[d][j][1];
            if constexpr (decltype(end_c)::value) {
                const int left = a.K - kt * 128 - 16 * q4;   // > 0: chunk q4 is a part of the row
                lo = left > 0 ? lo : (u32x4){};
                hi = left > 64 ? hi : (u32x4){};
            }
            b[j] = join(lo, hi);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const i32x8 w = join(fw[d][i][0], fw[d][i][1]);
#pragma unroll
            for (int j = 0; j < MB; ++j) acc[i][j] = mfma_f8<s>(w, b[j], acc[i][j], sw[i], sx[j]);
        }
    };
    auto group = [&](int g, auto end_c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; ++i) sw[i] = nw[i];
#pragma unroll
        for (int j = 0; j < MB; ++j) sx[j] = nx[j];
        load_scales(g + 1);
        products(4 * g, IC<0>(), end_c);
        load(4 * g + D, IC<0>());
        products(4 * g + 1, IC<1>(), end_c);
        load(4 * g + 1 + D, IC<1 % D>());
        products(4 * g + 2, IC<2>(), end_c);
        load(4 * g + 2 + D, IC<2 % D>());
        products(4 * g + 3, IC<3>(), end_c);
        load(4 * g + 3 + D, IC<3 % D>());
    };
    static_assert(D == 1 || D == 2 || D == 4, "a block's registers by its byte");
    if (g0 < g1) {
        load_scales(g0);
        load(4 * g0, IC<0>());
        if constexpr (D > 1) load(4 * g0 + 1, IC<1 % D>());
        if constexpr (D > 2) {
            load(4 * g0 + 2, IC<2 % D>());
            load(4 * g0 + 3, IC<3 % D>());
        }
        // the last group may end inside a block, or before one
        const int whole = (a.K & 511) == 0 ? g1 : min(g1, ng - 1);
        int g = g0;
        for (; g < whole; ++g) group(g, BC<false>());
        if (g < g1) group(g, BC<true>());
    }

    // ---- the four partial sums, 16 PN outputs of every token at a time: row
    // m of 64 PN bytes, 16-byte chunk c at c ^ its swizzle
    lds_t *const sp = LDS_PTR(char, lds);
    constexpr int kChunks = 4 * PN;
    auto swz = [](int m) { return PN == 1 ? (m >> 2) & 3 : PN == 2 ? (m >> 1) & 7 : m & (kChunks - 1); };
#pragma unroll
    for (int p = 0; p < NB / PN; ++p) {
        if (p) __syncthreads();
#pragma unroll
        for (int i = 0; i < PN; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                const int m = 16 * j + l16;
                *reinterpret_cast<__attribute__((address_space(3))) f32x4 *>(
                    sp + wave * kPart + m * (64 * PN) + (((4 * i + q4) ^ swz(m)) << 4)) = acc[p * PN + i][j];
            }
        __syncthreads();
#pragma unroll
        for (int t = tid; t < 16 * MB * kChunks; t += 256) {
            const int m = t / kChunks, c = t % kChunks;
            const int n = n0 + 16 * PN * p + 4 * c;
            if (m0 + m >= a.M || n >= a.N) continue;
            const lds_t *q = sp + m * (64 * PN) + ((c ^ swz(m)) << 4);
            f32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) f32x4 *>(q);
#pragma unroll
            for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const __attribute__((address_space(3))) f32x4 *>(q + w * kPart);
            if (a.bias) v += *reinterpret_cast<const f32x4 *>(a.bias + n);
            const u32x2 o = {Elem<__bf16>::pack2(v.x, v.y), Elem<__bf16>::pack2(v.z, v.w)};
            __builtin_nontemporal_store(o, reinterpret_cast<u32x2 *>(a.dst + (int64_t)(m0 + m) * a.d_nb1 + (int64_t)n * 2));
        }
    }
}

template <int NB, int MB, int D>
static void launch_stream(const F8MmArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((f8_mm_stream<NB, MB, D>), dim3(a.n_blocks), dim3(256), 0, s, a);
}

hipError_t launch_f8_mm(const F8MmArgs &a, int tile, hipStream_t s) {
    switch (tile) {
    case 401: launch_stream<4, 1, 4>(a, s); break;
    case 404: launch_stream<4, 4, 2>(a, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kdfa
