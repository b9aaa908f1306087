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

#include <utility>

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

// f(IC<0>()) ... f(IC<N - 1>()): a loop that is unrolled whatever its size.
template <class F, int... I>
static __device__ __forceinline__ void static_for(F f, std::integer_sequence<int, I...>) {
    (f(IC<I>()), ...);
}
template <int N, class F>
static __device__ __forceinline__ void static_for(F f) {
    static_for(f, std::make_integer_sequence<int, N>());
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

// ---------------------------------------------------------------------------
// f8_mm_tile: 256 outputs x 256 tokens per workgroup, 4 waves (one per SIMD,
// 512 registers each), wave w the 128 x 128 quarter (w & 1, w >> 1) as 8 x 8
// accumulator blocks (256 AGPRs).
//
// K advances 128 per stage, whole 128-byte lines of W's and X's rows, which
// come by DMA into two buffers of W and three of X (32 KB each: all of LDS).
// In LDS 16-byte chunk c of row r lies at c ^ ((r >> 1) & 7), which spreads
// the 16 rows of a fragment read over the 64 banks.
//
// Step kt goes through W's eight fragments: 8 products of each with the X
// fragments, which are in registers since the step before.  Meanwhile W's
// fragments are read two ahead of their products and stage kt + 1's X
// fragments into the other set, so that LDS is read evenly (32 reads over 64
// products).  The one barrier stands behind the last of those reads, three
// quarters of the step through: it frees W's buffer of stage kt and X's of
// stage kt + 1 for stages kt + 2 and kt + 4, and publishes W of stage kt + 1
// and X of stage kt + 2.  X, which is another for every workgroup of a
// column, so has almost two steps for its way; W, whose lines the XCD's other
// workgroups ask for too, one.
//
// A row's scales come as words of four stages, loaded by the lanes that hold
// the row, a step ahead of their first use.
// Rows past M or N are the last row again (not stored).  The last steps bring
// nothing past K: a stage that is not there is the tile's first chunk for
// every lane, a chunk past K its row's first of that stage, and X's are
// zeroed in their registers.
// ---------------------------------------------------------------------------
constexpr int kTileBuf = 32768;   // 256 rows x 128 k

template <int SEL>
static __device__ __forceinline__ void mfma_f8_asm(f32x4 &c, const i32x8 &a, const i32x8 &b, uint32_t sa, uint32_t sb) {
    if constexpr (SEL == 0)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (SEL == 1)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]" : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (SEL == 2)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0]" : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0]" : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
void f8_mm_tile(F8MmArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[5 * kTileBuf];
    lds_t *const sbase = LDS_PTR(char, lds);
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15;
    const int q4 = lane >> 4;
    const int wn = wave & 1, wm = wave >> 1;
    int nt, mt;
    f8_tile(a, nt, mt);
    const int n0 = nt * 256, m0 = mt * 256;
    const int nk = (int)(((uint32_t)a.K + 127) >> 7);   // stages
    const int whole = a.K >> 7;                         // those of 128 k
    const int ng = (nk + 3) >> 2;                       // words of scales

    // DMA j of a wave: rows 8 (wave + 4 j) .. +7, lane l the chunk that lies
    // at l % 8 of row l / 8.  Row offsets are made where they are used (a few
    // instructions under a product), not kept in registers: `fresh` hides from
    // the compiler that they are the same every time.
    const int dr = 8 * wave + (lane >> 3);
    const int dc = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
    const int w_last = a.N - 1 - n0, x_last = a.M - 1 - m0;
    auto fresh = [](int v) __attribute__((always_inline)) {
        asm volatile("" : "+v"(v));
        return v;
    };
    auto row_off = [](int r, int last, int64_t nb1) __attribute__((always_inline)) {
        return __umul24((uint32_t)min(r, last), (uint32_t)nb1);   // (strides are below 2^24: kd_f8_host.cpp)
    };
    const char *const wtile = a.w + (int64_t)n0 * a.w_nb1;
    const char *const xtile = a.x + (int64_t)m0 * a.x_nb1;
    const char *const wst = a.ws + (int64_t)n0 * a.ws_nb1;
    const char *const xst = a.xs + (int64_t)m0 * a.xs_nb1;
    // Stage kt of W or X: its first byte of the tile's first row, the tile's
    // last row and the lane's chunk.  A stage that is not there is the tile's
    // first chunk for every lane, a chunk past K its row's first.
    struct Stage { const char *at; int last; uint32_t chunk; };
    auto stage = [&](const char *tile, int last, int kt, auto end_c) __attribute__((always_inline)) {
        Stage t = {tile + (int64_t)kt * 128, last, (uint32_t)(dc << 4)};
        if constexpr (decltype(end_c)::value) {
            t.chunk = kt * 128 + 16 * dc < a.K ? t.chunk : 0;
            t.last = kt < nk ? last : 0;
            t.at = kt < nk ? t.at : tile;
        }
        return t;
    };
    auto dma_w = [&](const Stage &t, int buf, int j) __attribute__((always_inline)) {
        dma16(t.at, row_off(fresh(dr) + 32 * j, t.last, a.w_nb1) + t.chunk, sbase + buf * kTileBuf + (wave + 4 * j) * 1024);
    };
    auto dma_x = [&](const Stage &t, int buf, int j) __attribute__((always_inline)) {
        dma16(t.at, row_off(fresh(dr) + 32 * j, t.last, a.x_nb1) + t.chunk, sbase + (2 + buf) * kTileBuf + (wave + 4 * j) * 1024);
    };

    // scales: sw[i], sx[j] the words of row 16 i + l16 of this wave's halves.
    // Lane l loads those of rows l and 64 + l, once each and four words (16
    // stages) at a time; three swaps then give four fragments' words.  (A
    // load's lines are what it costs: each is 128 bytes out of the L2.  Rows
    // loaded by four lanes each 1.03 -> 0.88 ms at 63,488 x 4096 x 4096.)
    typedef uint32_t u32x4_4 __attribute__((ext_vector_type(4), aligned(4)));
    uint32_t sw[8], sx[8], nw[8], nx[8];
    u32x4 raw[4];
    auto load_scales = [&](int b) __attribute__((always_inline)) {   // words 4 b .. +3
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool w = q < 2;
            const uint32_t r = row_off(fresh(lane) + (w ? 128 * wn : 128 * wm) + 64 * (q & 1), w ? w_last : x_last, w ? a.ws_nb1 : a.xs_nb1);
            const char *const row = (w ? wst : xst) + (uint64_t)r;
            if (4 * b + 4 <= ng) {
                raw[q] = *reinterpret_cast<const u32x4_4 *>(row + 16 * b);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[q][e] = *reinterpret_cast<const uint32_t *>(row + 4 * min(4 * b + e, ng - 1));
            }
        }
    };
    // the next word of rows q
    auto spread_scales = [&](int q) __attribute__((always_inline)) {
        uint32_t *const to = (q < 2 ? nw : nx) + 4 * (q & 1);
        const auto h = __builtin_amdgcn_permlane32_swap(raw[q].x, raw[q].x, false, false);
        const auto u = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
        const auto v = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
        to[0] = u[0]; to[1] = u[1]; to[2] = v[0]; to[3] = v[1];
        raw[q] = (u32x4){raw[q].y, raw[q].z, raw[q].w, raw[q].w};
    };
    auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 8; ++q) { sw[q] = nw[q]; sx[q] = nx[q]; }
        asm volatile("s_nop 4" ::: "memory");   // (the products are asm: VALU results before they read them)
    };

    // fragments
    typedef const __attribute__((address_space(3))) u32x4 lds_u4;
    const uint32_t f_rd = (uint32_t)(l16 * 128 + ((q4 ^ ((l16 >> 1) & 7)) << 4));
    const uint32_t w_rd = f_rd + 128 * 128 * wn, x_rd = f_rd + 128 * 128 * wm + 2 * kTileBuf;
    u32x4 fw[4][2], fx[2][8][2];
    auto read_w = [&](int buf, int i, int h) __attribute__((always_inline)) {
        fw[i & 3][h] = *reinterpret_cast<lds_u4 *>(sbase + buf * kTileBuf + (w_rd ^ (h << 6)) + i * 2048);
    };
    auto read_x = [&](int buf, auto set_c, int j, int h) __attribute__((always_inline)) {
        fx[decltype(set_c)::value][j][h] = *reinterpret_cast<lds_u4 *>(sbase + buf * kTileBuf + (x_rd ^ (h << 6)) + j * 2048);
    };

    f32x4 acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = (f32x4){};

    int xb = 1;   // the X buffer of stage kt + 1
    // step kt: byte SEL of the scales' words, W buffer and X set SEL & 1
    auto step = [&](int kt, auto sel_c, auto end_c) __attribute__((always_inline)) {
        constexpr int S = decltype(sel_c)::value, P = S & 1;
        constexpr bool END = decltype(end_c)::value;
        const int xprev = xb == 0 ? 2 : xb - 1;   // freed by the last step's barrier
        const Stage next_w = stage(wtile, w_last, kt + 2, end_c), next_x = stage(xtile, x_last, kt + 3, end_c);
        if constexpr (END) {
            if (kt >= whole) {
                // the one stage that ends inside: what lies past K is zero
                const int left = a.K - kt * 128 - 16 * q4;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    fx[P][j][0] = left > 0 ? fx[P][j][0] : (u32x4){};
                    fx[P][j][1] = left > 64 ? fx[P][j][1] : (u32x4){};
                }
                asm volatile("s_nop 4" ::: "memory");   // (the products are asm: VALU results before they read them)
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        static_for<64>([&](auto p_c) __attribute__((always_inline)) {
            constexpr int p = decltype(p_c)::value, i = p >> 3, j = p & 7;
            if constexpr (p == 48) {
                if constexpr (S == 3) {
                    // the next words of scales, loaded a step ago (the
                    // compiler waits for them here)
#pragma unroll
                    for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(raw[q]));
                }
                // all but the 8 DMAs of X of stage kt + 3 have landed
                asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
                __syncthreads();
                __builtin_amdgcn_sched_barrier(0);
            }
            mfma_f8_asm<S>(acc[i][j], join(fw[i & 3][0], fw[i & 3][1]), join(fx[P][j][0], fx[P][j][1]), sw[i], sx[j]);
            __builtin_amdgcn_sched_barrier(0);
            // X of stage kt + 3, into the buffer that the last step freed
            if constexpr (p < 32 && p % 4 == 0) dma_x(next_x, xprev, p / 4);
            // W's fragment two on
            if constexpr (i < 6 && (j == 1 || j == 3)) read_w(P, i + 2, j >> 1);
            // X of stage kt + 1
            if constexpr (i < 4 && (j == 2 || j == 4 || j == 5 || j == 7)) {
                constexpr int q = 4 * i + (j == 2 ? 0 : j == 4 ? 1 : j == 5 ? 2 : 3);
                read_x(xb, IC<1 - P>(), q >> 1, q & 1);
            }
            if constexpr (p >= 48) {
                if constexpr (j % 2 == 0) dma_w(next_w, P, (p - 48) / 2);
                if constexpr (j == 1 || j == 3) read_w(1 - P, i - 6, j >> 1);
                // the next four groups' scales, ahead of W's last DMAs
                if constexpr (S == 2 && p == 49) {
                    if (((kt >> 2) & 3) == 3) load_scales(((kt >> 2) + 1) >> 2);
                }
                if constexpr (S == 3 && j % 4 == 0) spread_scales((p - 48) >> 2);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        xb = xb == 2 ? 0 : xb + 1;
        if constexpr (S == 3) take_scales();
    };

    load_scales(0);
    {
        const Stage x0 = stage(xtile, x_last, 0, BC<true>()), w0 = stage(wtile, w_last, 0, BC<true>()),
                    x1 = stage(xtile, x_last, 1, BC<true>()), w1 = stage(wtile, w_last, 1, BC<true>()),
                    x2 = stage(xtile, x_last, 2, BC<true>());
#pragma unroll
        for (int j = 0; j < 8; ++j) dma_x(x0, 0, j);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma_w(w0, 0, j);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma_x(x1, 1, j);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma_w(w1, 1, j);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma_x(x2, 2, j);
    }
    asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) read_x(0, IC<0>(), j, h);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) read_w(0, i, h);
#pragma unroll
    for (int q = 0; q < 4; ++q) spread_scales(q);
    take_scales();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();

    int kt = 0;
    for (; kt + 7 <= whole; kt += 4) {   // the last step's X is stage kt + 6
        step(kt, IC<0>(), BC<false>());
        step(kt + 1, IC<1>(), BC<false>());
        step(kt + 2, IC<2>(), BC<false>());
        step(kt + 3, IC<3>(), BC<false>());
    }
    for (; kt < nk; kt += 4) {
        step(kt, IC<0>(), BC<true>());
        if (kt + 1 < nk) step(kt + 1, IC<1>(), BC<true>());
        if (kt + 2 < nk) step(kt + 2, IC<2>(), BC<true>());
        if (kt + 3 < nk) step(kt + 3, IC<3>(), BC<true>());
    }
    // (the products are asm: the wait states between the last and a read of
    // its accumulators are ours to give, and the accumulators pass through
    // what follows the wait, so that no read of them can stand before it)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("; accumulator complete" : "+a"(acc[i][j]));
    __syncthreads();

    // ---- epilogue: dst[m][n .. n+3] = acc (+ bias) in BF16.  The wave's 128
    // tokens x 256 bytes go through its own region of LDS (chunk c of row r at
    // c ^ (r & 15)), so that a store instruction writes four rows' 256 bytes.
    // A wave touches only its own region (its LDS operations complete in order).
    lds_t *const so = sbase + wave * 32768;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = n0 + 128 * wn + 16 * i + 4 * q4;
        f32x4 bias = {0.f, 0.f, 0.f, 0.f};
        if (a.bias && n < a.N) bias = *reinterpret_cast<const f32x4 *>(a.bias + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const f32x4 v = acc[i][j] + bias;
            *reinterpret_cast<__attribute__((address_space(3))) u32x2 *>(
                so + (16 * j + l16) * 256 + (((2 * i + (q4 >> 1)) ^ l16) << 4) + ((q4 & 1) << 3)) =
                (u32x2){Elem<__bf16>::pack2(v.x, v.y), Elem<__bf16>::pack2(v.z, v.w)};
        }
    }
    typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));   // dst rows lie at multiples of 8 bytes
    const int n = n0 + 128 * wn + 8 * l16;
#pragma unroll
    for (int t = 0; t < 32; ++t) {
        const int r = 4 * t + q4, m = m0 + 128 * wm + r;
        const u32x4 v = *reinterpret_cast<lds_u4 *>(so + r * 256 + ((l16 ^ (r & 15)) << 4));
        char *const p = a.dst + (int64_t)m * a.d_nb1 + (int64_t)n * 2;
        if (m < a.M) {
            if (n + 8 <= a.N)
                __builtin_nontemporal_store((u32x4_8)v, reinterpret_cast<u32x4_8 *>(p));
            else if (n < a.N)
                __builtin_nontemporal_store((u32x2){v.x, v.y}, reinterpret_cast<u32x2 *>(p));
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
    case 1616: hipLaunchKernelGGL(f8_mm_tile, dim3(a.n_blocks), dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kdfa
