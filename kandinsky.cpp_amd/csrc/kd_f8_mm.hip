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

// D += A B, each row's codes times the scale in byte 0 of its word
static __device__ __forceinline__ f32x4 mfma_f8(i32x8 a, i32x8 b, f32x4 c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}

// DMAs into LDS, 16 bytes a lane at base + its offset, or one word a lane at
// its own address; the destination is wave-uniform, the lanes' pieces lie there
// in lane order.  The compiler does not track them: every consumer waits with
// an explicit s_waitcnt vmcnt.  (m0 names the destination and takes a wait
// state between its writing and the DMA.)
static __device__ __forceinline__ void dma_16b(const char *base, uint32_t lane_off, lds_t *lds_wave_base) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds_wave_base);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(lane_off), "s"(base), "{m0}"(m0));
}
static __device__ __forceinline__ void dma_word(const char *p, lds_t *lds_wave_base) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds_wave_base);
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(p), "{m0}"(m0));
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

// A wave's part of dst out of LDS: R rows of C chunks of 16 bytes, chunk c of
// row r at c ^ swz(r), to tokens m0 .. and outputs n0 ..
template <int R, int C, class Swz>
static __device__ __forceinline__ void store_rows(const F8MmArgs &a, const lds_t *from, Swz swz, int m0, int n0, int lane) {
    typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));   // dst rows lie at multiples of 8 bytes
    const int c = lane % C, n = n0 + 8 * c;
#pragma unroll
    for (int t = 0; t < R * C / 64; ++t) {
        const int r = t * (64 / C) + lane / C, m = m0 + r;
        const u32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>(from + r * (16 * C) + ((c ^ swz(r)) << 4));
        char *const p = a.dst + (int64_t)m * a.d_nb1 + (int64_t)n * 2;
        if (m < a.M) {
            if (n + 8 <= a.N)
                __builtin_nontemporal_store((u32x4_8)v, reinterpret_cast<u32x4_8 *>(p));
            else if (n < a.N)
                __builtin_nontemporal_store((u32x2){v.x, v.y}, reinterpret_cast<u32x2 *>(p));
        }
    }
}

// ---------------------------------------------------------------------------
// f8_mm_ring: 16 NB outputs x 16 MB tokens per workgroup, for calls of few
// tokens or few tiles.  The four waves split k, each a run of stages of 128 k,
// and compute the whole tile over it: nothing that a wave loads is another's,
// so each keeps its own ring of S stages in LDS, filled by DMA, and no barrier
// stands before the four partial sums meet, in wave order.  A stage's
// fragments go into registers at once, and its buffer to stage S on: what is
// on its way is the whole of LDS, whatever the tile.
//
// The scales come row by row in words of four stages, into one of two slots
// ahead of the first of the four, and are read a byte at a time.
// In LDS 16-byte chunk c of row r lies at c ^ ((r >> 1) & 7).  Rows past N or
// M are the last row again (not stored); a chunk past K is its row's first of
// the stage, X's then zeroed in the registers.
//
// With few tokens it is bound by W's way from HBM: 2 x 16384 x 4096 (67 MB)
// 12.3 us, 5.5 TB/s, what a copy reaches.  300 x 4096 x 4096 takes 12.0 us
// (256 tiles of 64 x 80, one on each CU): 4 of it the first loads, the sums and
// the stores, and 0.2 for each of the 32 stages, whose 18 KB then come into LDS
// at 23 TB/s over all CUs, out of the L2s.
//
// LINES, for code rows that do not all start on 128-byte lines: a stage brings
// a line of each row in place of 128 k, what is not the row's its first or last
// chunk again, and a block's chunks are read out of two stages: 128 k of such a
// row cross two lines, each of which came twice.  From K = 1024 on (packed rows,
// 300 x 4096 x 4112 15.3 us, so 13.0; x 1040 7.6 and 7.4; x 528 5.9 and 6.4; 17 x
// 260 x 4112, where it only waits longer, 4.7 and 5.5).
// ---------------------------------------------------------------------------
template <int NB, int MB, int S, bool LINES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void f8_mm_ring(F8MmArgs a) {
    constexpr int kRows = 16 * (NB + MB);
    constexpr int kStage = kRows * 128;
    constexpr int kDma = kRows / 8;                         // of a stage
    constexpr int kWordRows = (kRows + 63) / 64 * 64;       // rows of a word's DMAs
    constexpr int kSlot = kWordRows * 4;
    constexpr int kWave = S * kStage + 2 * kSlot;
    constexpr int PN = NB % 4 == 0 ? 4 : NB % 2 == 0 ? 2 : 1;   // fragments of outputs that are joined at once
    constexpr int kPart = 16 * MB * 16 * PN * 4;
    constexpr int kLds = 4 * (kWave > kPart ? kWave : kPart);
    static_assert(kLds <= 163840 && S >= 1 + LINES && S <= 4 && (S - 1) * kDma <= 63, "LDS, a slot of words that is read before it is written again, and the counter of what is on its way");
    __shared__ __attribute__((aligned(1024))) char lds[kLds];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15;
    const int q4 = lane >> 4;
    int nt, mt;
    f8_tile(a, nt, mt);
    const int n0 = nt * (16 * NB), m0 = mt * (16 * MB);
    const int w_last = a.N - 1 - n0, x_last = a.M - 1 - m0;
    const char *const wt = a.w + (int64_t)n0 * a.w_nb1;
    const char *const xt = a.x + (int64_t)m0 * a.x_nb1;
    lds_t *const ring = LDS_PTR(char, lds) + wave * kWave;
    lds_t *const words = ring + S * kStage;

    // DMA j of a stage: rows 8 j .. +7 (W's, then X's), lane l the chunk that
    // lies at l % 8 of row l / 8
    uint32_t off[kDma];
#pragma unroll
    for (int j = 0; j < kDma; ++j) {
        const int r = 8 * j + (lane >> 3);
        off[j] = j < 2 * NB ? (uint32_t)min(r, w_last) * (uint32_t)a.w_nb1 : (uint32_t)min(r - 16 * NB, x_last) * (uint32_t)a.x_nb1;
    }
    const int c0 = (lane & 7) ^ (lane >> 4), c1 = c0 ^ 4;   // chunks of even and odd j
    // LINES: where a row begins in its line, in chunks (row r as r + 8)
    const int w_step = (int)(a.w_nb1 >> 4) & 7, x_step = (int)(a.x_nb1 >> 4) & 7;
    const int w_at = (int)((uintptr_t)wt >> 4) & 7, x_at = (int)((uintptr_t)xt >> 4) & 7;
    const int w_sh = (w_at + (lane >> 3) * w_step) & 7, x_sh = (x_at + (lane >> 3) * x_step) & 7;
    const int nk = (int)(((uint32_t)a.K + 127) >> 7);
    // this wave's stages
    const int k0 = (int)((int64_t)wave * nk >> 2), k1 = (int)((int64_t)(wave + 1) * nk >> 2);
    // word g of the tile's rows: W's, then X's, then X's last again
    const char *word_at[kWordRows / 64];
#pragma unroll
    for (int h = 0; h < kWordRows / 64; ++h) {
        const int r = 64 * h + lane, rx = r - 16 * NB;
        word_at[h] = rx < 0 ? a.ws + (int64_t)(n0 + min(r, w_last)) * a.ws_nb1
                            : a.xs + (int64_t)(m0 + min(min(rx, 16 * MB - 1), x_last)) * a.xs_nb1;
    }
    auto issue_word = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < kWordRows / 64; ++h) dma_word(word_at[h] + 4 * (int64_t)g, words + (g & 1) * kSlot + h * 256);
    };
    // stage kt into ring buffer buf, its word before the first of four; past
    // this wave's last, the tile's first chunk for every lane (not used), so
    // that the counter counts alike (the words are not counted: a wait is then
    // for up to as many operations of the next stage too)
    auto issue = [&](int kt, int buf) __attribute__((always_inline)) {
        lds_t *const to = ring + buf * kStage;
        if (kt < k1 + LINES) {
            if ((kt & 3) == 0 && kt < k1) issue_word(kt >> 2);
            if constexpr (LINES) {
                // (from 128 bytes before the tile, so that no offset is
                // negative); outside of the row, its first or last chunk
                const int line = kt * 128;
                auto at = [&](int c, int sh) __attribute__((always_inline)) {
                    return (uint32_t)(min(max(line + 16 * (((c + sh) & 7) - sh), 0), a.K - 16) - line + 128);
                };
                const uint32_t w0 = at(c0, w_sh), w1 = at(c1, w_sh), x0 = at(c0, x_sh), x1 = at(c1, x_sh);
#pragma unroll
                for (int j = 0; j < kDma; ++j)
                    dma_16b((j < 2 * NB ? wt : xt) + (int64_t)line - 128, off[j] + (j < 2 * NB ? (j & 1 ? w1 : w0) : (j & 1 ? x1 : x0)), to + j * 1024);
                return;
            }
            const int64_t kb = (int64_t)kt * 128;
            const int left = a.K - kt * 128;
            const uint32_t b0 = 16 * c0 < left ? 16 * c0 : 0, b1 = 16 * c1 < left ? 16 * c1 : 0;
#pragma unroll
            for (int j = 0; j < kDma; ++j) dma_16b((j < 2 * NB ? wt : xt) + kb, off[j] + (j & 1 ? b1 : b0), to + j * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < kDma; ++j) dma_16b(j < 2 * NB ? wt : xt, 0, to + j * 1024);
        }
    };

    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = (f32x4){};
    typedef const __attribute__((address_space(3))) u32x4 lds_u4;
    const uint32_t f_rd = (uint32_t)(l16 * 128 + ((q4 ^ ((l16 >> 1) & 7)) << 4));
    // LINES: all bits where chunk q4 or q4 + 4 of a block is in the next line
    uint32_t w_next[2], x_next[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w_next[h] = 0u - (uint32_t)((q4 + 4 * h + ((w_at + l16 * w_step) & 7)) >> 3);
        x_next[h] = 0u - (uint32_t)((q4 + 4 * h + ((x_at + l16 * x_step) & 7)) >> 3);
    }
    if (k0 < k1) {
        if (k0 & 3) issue_word(k0 >> 2);
#pragma unroll
        for (int s = 0; s < S; ++s) issue(k0 + s, s);
        int buf = 0;
        for (int kt = k0; kt < k1; ++kt) {
            asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S - 1 - LINES) * kDma) : "memory");
            const lds_t *const from = ring + buf * kStage;
            const uint32_t on = LINES ? (buf == S - 1 ? 0u - (S - 1) * kStage : kStage) : 0u;
            const lds_t *const w_from[2] = {from + f_rd + (w_next[0] & on), from + (f_rd ^ 64) + (w_next[1] & on)};
            const lds_t *const x_from[2] = {from + f_rd + (x_next[0] & on), from + (f_rd ^ 64) + (x_next[1] & on)};
            u32x4 fw[NB][2], fx[MB][2];
            uint32_t sw[NB], sx[MB];
            const lds_t *const sp = words + ((kt >> 2) & 1) * kSlot + (kt & 3) + l16 * 4;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                sw[i] = *reinterpret_cast<const __attribute__((address_space(3))) uint8_t *>(sp + 64 * i);
                fw[i][0] = *reinterpret_cast<lds_u4 *>(w_from[0] + i * 2048);
                fw[i][1] = *reinterpret_cast<lds_u4 *>(w_from[1] + i * 2048);
            }
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                sx[j] = *reinterpret_cast<const __attribute__((address_space(3))) uint8_t *>(sp + 64 * (NB + j));
                fx[j][0] = *reinterpret_cast<lds_u4 *>(x_from[0] + (NB + j) * 2048);
                fx[j][1] = *reinterpret_cast<lds_u4 *>(x_from[1] + (NB + j) * 2048);
            }
            // the buffer is free when its reads have returned
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            issue(kt + S, buf);
            buf = buf == S - 1 ? 0 : buf + 1;
            if (kt * 128 + 128 > a.K) {
                const int left = a.K - kt * 128 - 16 * q4;
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    fx[j][0] = left > 0 ? fx[j][0] : (u32x4){};
                    fx[j][1] = left > 64 ? fx[j][1] : (u32x4){};
                }
            }
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j)
                    acc[i][j] = mfma_f8(join(fw[i][0], fw[i][1]), join(fx[j][0], fx[j][1]), acc[i][j], sw[i], sx[j]);
        }
        // what is still on its way is nobody's
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    // ---- the four partial sums, 16 PN outputs of every token at a time: row
    // m of 64 PN bytes, 16-byte chunk c at c ^ its swizzle
    lds_t *const sp = LDS_PTR(char, lds);
    constexpr int kChunks = 4 * PN;
    auto swz = [](int m) { return PN == 1 ? (m >> 2) & 3 : PN == 2 ? (m >> 1) & 7 : m & 15; };
#pragma unroll
    for (int p = 0; p < NB / PN; ++p) {
        __syncthreads();
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
// f8_mm_grid: 32 NB outputs x 32 MB tokens per workgroup, its four waves a 2 x
// 2 grid of 16 NB x 16 MB each: for calls whose 256 x 256 tiles would leave
// CUs idle, and whose tiles of f8_mm_ring (where a wave holds the whole tile's
// sums) would have to be so small that W and X come too often.
//
// S stages of 128 k in LDS, one barrier a step: step kt publishes stage kt + 1
// -- behind the barrier every wave's reads of stage kt have returned -- reads
// its fragments into the other set, and sends stage kt + S into stage kt's
// buffer while the products of stage kt run.  Words of scales come ahead of
// each fourth stage, into one of two slots.  LDS rows, rows past N or M and k
// past K are f8_mm_ring's; a stage past the last is the tile's first chunk for
// every lane, so that the counter counts alike.
//
// 1,280 x 4096 x 4096 takes 23.5 us (256 tiles of 128 x 160, one on each CU):
// 0.46 us a stage for the CU's 36 KB into LDS, 20 TB/s over all of them out of
// the L2s, where the products would take 0.31 at the rate they sustain.  997 x
// 1540 x 3600: 14 us (208 tiles of 128 x 64).
//
// LINES as f8_mm_ring's: 997 x 1540 x 3600 (rows packed) 17.8 us without, 14.0
// with; 1,280 x 4096 x 3600 26.2 and 22.3; 1500 x 1500 x 400 6.8 and 7.1.
// ---------------------------------------------------------------------------
template <int NB, int MB, int S, bool LINES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void f8_mm_grid(F8MmArgs a) {
    constexpr int kRows = 32 * (NB + MB);
    constexpr int kStage = kRows * 128;
    constexpr int kDma = NB + MB;                     // of a wave and stage
    constexpr int kWordDma = (kRows + 255) / 256;     // of a wave and word
    constexpr int kSlot = kWordDma * 1024;
    constexpr int kWaveOut = 16 * MB * 32 * NB;       // a wave's part of dst
    constexpr int kUse = S * kStage + 2 * kSlot;
    constexpr int kLds = kUse > 4 * kWaveOut ? kUse : 4 * kWaveOut;
    static_assert(kLds <= 163840 && S >= 2 + LINES && S <= 8, "LDS, and a slot of words that is read before it is written again");
    __shared__ __attribute__((aligned(1024))) char lds[kLds];
    lds_t *const sbase = LDS_PTR(char, lds);
    lds_t *const words = sbase + S * kStage;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15;
    const int q4 = lane >> 4;
    const int wn = wave & 1, wm = wave >> 1;
    int nt, mt;
    f8_tile(a, nt, mt);
    const int n0 = nt * (32 * NB), m0 = mt * (32 * MB);
    const int w_last = a.N - 1 - n0, x_last = a.M - 1 - m0;
    const char *const wt = a.w + (int64_t)n0 * a.w_nb1;
    const char *const xt = a.x + (int64_t)m0 * a.x_nb1;
    const int nk = (int)(((uint32_t)a.K + 127) >> 7);   // stages
    const int whole = a.K >> 7;                         // those of 128 k
    const int ng = (nk + 3) >> 2;                       // words of scales

    // DMA j of a wave: rows 8 (wave + 4 j) .. +7 of W, then of X; lane l the
    // chunk that lies at l % 8 of row l / 8
    uint32_t off[kDma];
    const int dc = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
    // LINES: row r begins (at + r * step) % 8 chunks of 16 bytes into a line,
    // rows r + 8, r + 16 .. too.  A row's chunk c of a block then lies at the
    // same place of the buffer as without (no other banks), of this stage's
    // line or of the next one; rel is the byte of line 0, from the row's
    // first, that this lane brings.
    const int w_step = (int)(a.w_nb1 >> 4) & 7, x_step = (int)(a.x_nb1 >> 4) & 7;
    const int w_at = (int)((uintptr_t)wt >> 4) & 7, x_at = (int)((uintptr_t)xt >> 4) & 7;
    const int w_sh = (w_at + (lane >> 3) * w_step) & 7, x_sh = (x_at + (lane >> 3) * x_step) & 7;
    const int w_rel = 16 * (((dc + w_sh) & 7) - w_sh), x_rel = 16 * (((dc + x_sh) & 7) - x_sh);
#pragma unroll
    for (int j = 0; j < kDma; ++j) {
        const int r = 8 * (wave + 4 * j) + (lane >> 3);
        off[j] = j < NB ? (uint32_t)min(r, w_last) * (uint32_t)a.w_nb1 : (uint32_t)min(r - 32 * NB, x_last) * (uint32_t)a.x_nb1;
        if constexpr (LINES) off[j] += 128 + (j < NB ? w_rel : x_rel);
    }
    // DMA h of a word: rows 256 h + 64 wave + lane (W's, X's, X's last again)
    const char *word_at[kWordDma];
#pragma unroll
    for (int h = 0; h < kWordDma; ++h) {
        const int r = 256 * h + 64 * wave + lane, rx = r - 32 * NB;
        word_at[h] = rx < 0 ? a.ws + (int64_t)(n0 + min(r, w_last)) * a.ws_nb1
                            : a.xs + (int64_t)(m0 + min(min(rx, 32 * MB - 1), x_last)) * a.xs_nb1;
    }
    // DMA j of stage kt, its words before its first
    auto dma_j = [&](int kt, int buf, int j, auto word_c, auto end_c) __attribute__((always_inline)) {
        if constexpr (decltype(word_c)::value) {
            if (j == 0) {
                const int g = min(kt >> 2, ng - 1);
#pragma unroll
                for (int h = 0; h < kWordDma; ++h) dma_word(word_at[h] + 4 * (int64_t)g, words + ((kt >> 2) & 1) * kSlot + h * 1024 + wave * 256);
            }
        }
        if constexpr (LINES) {
            // (from 128 bytes before the tile, so that no offset is negative)
            const char *at = (j < NB ? wt : xt) + ((int64_t)kt - 1) * 128;
            uint32_t o = off[j];
            if constexpr (decltype(end_c)::value) {
                // outside of the row, its first or last chunk
                const int rel = kt * 128 + (j < NB ? w_rel : x_rel);
                o = kt > nk ? 128 : o + (uint32_t)(min(max(rel, 0), a.K - 16) - rel);
                at = kt > nk ? (j < NB ? wt : xt) - 128 : at;
            }
            dma_16b(at, o, sbase + buf * kStage + (wave + 4 * j) * 1024);
            return;
        }
        const char *at = (j < NB ? wt : xt) + (int64_t)kt * 128;
        uint32_t o = off[j] + (uint32_t)(dc << 4);
        if constexpr (decltype(end_c)::value) {
            o = kt >= nk ? 0 : kt * 128 + 16 * dc < a.K ? o : off[j];
            at = kt >= nk ? (j < NB ? wt : xt) : at;
        }
        dma_16b(at, o, sbase + buf * kStage + (wave + 4 * j) * 1024);
    };

    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = (f32x4){};
    typedef const __attribute__((address_space(3))) u32x4 lds_u4;
    typedef const __attribute__((address_space(3))) uint32_t lds_u1;
    const uint32_t f_rd = (uint32_t)(l16 * 128 + ((q4 ^ ((l16 >> 1) & 7)) << 4));
    const uint32_t w_rd = f_rd + 16 * NB * wn * 128, x_rd = f_rd + (32 * NB + 16 * MB * wm) * 128;
    u32x4 fw[2][NB][2], fx[2][MB][2];
    uint32_t sw[NB], sx[MB], nw[NB], nx[MB];
    // LINES: all bits where chunk q4 or q4 + 4 of a block is in the next line
    uint32_t w_next[2], x_next[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w_next[h] = 0u - (uint32_t)((q4 + 4 * h + ((w_at + l16 * w_step) & 7)) >> 3);
        x_next[h] = 0u - (uint32_t)((q4 + 4 * h + ((x_at + l16 * x_step) & 7)) >> 3);
    }
    auto read = [&](int buf, auto set_c) __attribute__((always_inline)) {
        constexpr int set = decltype(set_c)::value;
        const lds_t *const from = sbase + buf * kStage;
        if constexpr (LINES) {
            const uint32_t here = buf * kStage, on = buf == S - 1 ? 0u - (S - 1) * kStage : kStage;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const lds_t *const wf = sbase + ((w_rd ^ (h << 6)) + here + (w_next[h] & on));
                const lds_t *const xf = sbase + ((x_rd ^ (h << 6)) + here + (x_next[h] & on));
#pragma unroll
                for (int i = 0; i < NB; ++i) fw[set][i][h] = *reinterpret_cast<lds_u4 *>(wf + i * 2048);
#pragma unroll
                for (int j = 0; j < MB; ++j) fx[set][j][h] = *reinterpret_cast<lds_u4 *>(xf + j * 2048);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) fw[set][i][h] = *reinterpret_cast<lds_u4 *>(from + (w_rd ^ (h << 6)) + i * 2048);
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) fx[set][j][h] = *reinterpret_cast<lds_u4 *>(from + (x_rd ^ (h << 6)) + j * 2048);
    };
    auto read_words = [&](int g) __attribute__((always_inline)) {
        const lds_t *const from = words + (g & 1) * kSlot + l16 * 4;
#pragma unroll
        for (int i = 0; i < NB; ++i) nw[i] = *reinterpret_cast<lds_u1 *>(from + (16 * NB * wn + 16 * i) * 4);
#pragma unroll
        for (int j = 0; j < MB; ++j) nx[j] = *reinterpret_cast<lds_u1 *>(from + (32 * NB + 16 * MB * wm + 16 * j) * 4);
    };
    // operations behind stage s + 1's, when stages up to s + S - 1 are issued
    // (s as far as it counts: its place in a group of four)
    auto later = [](int s, int from) constexpr {
        int n = 0;
        for (int t = s + from; t < s + S; ++t) n += kDma + (t % 4 == 0 ? kWordDma : 0);
        return n;
    };

    int buf = 0;   // of stage kt
    auto step = [&](int kt, auto sel_c, auto end_c) __attribute__((always_inline)) {
        constexpr int Q = decltype(sel_c)::value, P = Q & 1;
        const int here = buf;
        buf = buf == S - 1 ? 0 : buf + 1;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(later(Q, 2 + LINES)) : "memory");
        __syncthreads();
        read(buf, IC<1 - P>());
        if constexpr (Q == 3) read_words((kt >> 2) + 1);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(end_c)::value) {
            if (kt >= whole) {
                const int left = a.K - kt * 128 - 16 * q4;
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    fx[P][j][0] = left > 0 ? fx[P][j][0] : (u32x4){};
                    fx[P][j][1] = left > 64 ? fx[P][j][1] : (u32x4){};
                }
            }
        }
        static_for<NB * MB>([&](auto p_c) __attribute__((always_inline)) {
            constexpr int p = decltype(p_c)::value, i = p / MB, j = p % MB;
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(fw[P][i][0], fw[P][i][1]), join(fx[P][j][0], fx[P][j][1]), acc[i][j],
                                                                         0, 0, Q, (int)sw[i], Q, (int)sx[j]);
            __builtin_amdgcn_sched_barrier(0);
            static_for<kDma>([&](auto d_c) __attribute__((always_inline)) {
                constexpr int d = decltype(d_c)::value;
                if constexpr (d * (NB * MB) / kDma == p) dma_j(kt + S, here, d, BC<(Q + S) % 4 == 0>(), end_c);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (Q == 3) {
#pragma unroll
            for (int i = 0; i < NB; ++i) sw[i] = nw[i];
#pragma unroll
            for (int j = 0; j < MB; ++j) sx[j] = nx[j];
        }
    };

    static_for<S>([&](auto s_c) __attribute__((always_inline)) {
        constexpr int s = decltype(s_c)::value;
#pragma unroll
        for (int j = 0; j < kDma; ++j) dma_j(s, s, j, BC<s % 4 == 0>(), BC<true>());
    });
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(later(0, 1 + LINES)) : "memory");
    __syncthreads();
    read(0, IC<0>());
    read_words(0);
#pragma unroll
    for (int i = 0; i < NB; ++i) sw[i] = nw[i];
#pragma unroll
    for (int j = 0; j < MB; ++j) sx[j] = nx[j];
    int kt = 0;
    for (; kt + 3 + S < whole; kt += 4) {   // the last step's DMAs are of stage kt + 3 + S
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
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();

    // ---- dst[m][n .. n+3] = acc (+ bias) in BF16, through the wave's own
    // region of LDS (its operations complete in order): rows of 32 NB bytes,
    // 16-byte chunk c of row r at c ^ swz(r), stored as whole rows
    constexpr int kC = 2 * NB;
    auto swz = [](int r) { return (r / (16 / kC)) & (kC - 1); };
    lds_t *const so = sbase + wave * kWaveOut;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int n = n0 + 16 * NB * wn + 16 * i + 4 * q4;
        f32x4 bias = {0.f, 0.f, 0.f, 0.f};
        if (a.bias && n < a.N) bias = *reinterpret_cast<const f32x4 *>(a.bias + n);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int r = 16 * j + l16;
            const f32x4 v = acc[i][j] + bias;
            *reinterpret_cast<__attribute__((address_space(3))) u32x2 *>(
                so + r * (32 * NB) + (((2 * i + (q4 >> 1)) ^ swz(r)) << 4) + ((q4 & 1) << 3)) =
                (u32x2){Elem<__bf16>::pack2(v.x, v.y), Elem<__bf16>::pack2(v.z, v.w)};
        }
    }
    store_rows<16 * MB, kC>(a, so, swz, m0 + 16 * MB * wm, n0 + 16 * NB * wn, lane);
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
//
// 63,488 x 4096 x 4096 takes 0.85-0.88 ms (2.4-2.5 PFLOP/s), 15,872 x 4096 x 16384
// 0.72-0.75 (2.9); the products alone (no loads, no LDS reads) would take 0.50 of
// the former, the DMAs alone 0.53-0.62.  Both together draw the chip down to
// 2.0-2.1 GHz, and the two run at once but for what the barrier holds up.
// Tiles kept up by persistent workgroups (the next tile's first stages under
// the stores), lines asked into the L2 ahead, other cache hints of the DMAs, 2,
// 8 or 16 tile columns at a time in place of 4 and the barrier elsewhere in the
// step left the time where it was or made it longer.
// M and N are at least 256: a last tile that would end past them begins earlier
// instead, and what it has in common with the one before is written twice, the
// same bits.  The last steps bring nothing past K: a stage that is not there is
// the tile's first chunk for every lane, a chunk past K its row's first of that
// stage, and X's are zeroed in their registers.
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
    const int n0 = min(nt * 256, a.N - 256), m0 = min(mt * 256, a.M - 256);
    const int nk = (int)(((uint32_t)a.K + 127) >> 7);   // stages
    const int whole = a.K >> 7;                         // those of 128 k
    const int ng = (nk + 3) >> 2;                       // words of scales

    const char *const wtile = a.w + (int64_t)n0 * a.w_nb1;
    const char *const xtile = a.x + (int64_t)m0 * a.x_nb1;
    const char *const wst = a.ws + (int64_t)n0 * a.ws_nb1;
    const char *const xst = a.xs + (int64_t)m0 * a.xs_nb1;
    // DMA j of a wave: rows 8 (wave + 4 j) .. +7, lane l the chunk that lies
    // at l % 8 of row l / 8: one offset a lane, and a scalar step from j to j
    // + 1.  (Offsets clamped to the last row were four vector instructions a
    // DMA, as many as products: 903 us, without them 873, at 63,488 x 4096 x
    // 4096.)
    const int dr = 8 * wave + (lane >> 3);
    const int dc = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
    const uint32_t w_row = __umul24(dr, (uint32_t)a.w_nb1), x_row = __umul24(dr, (uint32_t)a.x_nb1);   // (strides are below 2^24)
    const uint32_t w_off = w_row + (dc << 4), x_off = x_row + (dc << 4);
    // Stage kt of W or X.  One that is not there is the tile's first chunk for
    // every lane, a chunk past K its row's first.
    struct Stage { const char *at; int64_t step; uint32_t off; };
    auto stage = [&](bool w, int kt, auto end_c) __attribute__((always_inline)) {
        const char *const tile = w ? wtile : xtile;
        Stage t = {tile + (int64_t)kt * 128, 32 * (w ? a.w_nb1 : a.x_nb1), w ? w_off : x_off};
        if constexpr (decltype(end_c)::value) {
            t.off = kt * 128 + 16 * dc < a.K ? t.off : kt < nk ? (w ? w_row : x_row) : 0;
            t.at = kt < nk ? t.at : tile;
            t.step = kt < nk ? t.step : 0;
        }
        return t;
    };
    auto dma_w = [&](const Stage &t, int buf, int j) __attribute__((always_inline)) {
        dma_16b(t.at + j * t.step, t.off, sbase + buf * kTileBuf + (wave + 4 * j) * 1024);
    };
    auto dma_x = [&](const Stage &t, int buf, int j) __attribute__((always_inline)) {
        dma_16b(t.at + j * t.step, t.off, sbase + (2 + buf) * kTileBuf + (wave + 4 * j) * 1024);
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
            const uint32_t r = __umul24(lane + (w ? 128 * wn : 128 * wm) + 64 * (q & 1), (uint32_t)(w ? a.ws_nb1 : a.xs_nb1));
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
        const Stage next_w = stage(true, kt + 2, end_c), next_x = stage(false, kt + 3, end_c);
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
        const Stage x0 = stage(false, 0, BC<true>()), w0 = stage(true, 0, BC<true>()), x1 = stage(false, 1, BC<true>()),
                    w1 = stage(true, 1, BC<true>()), x2 = stage(false, 2, BC<true>());
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
        if (a.bias) bias = *reinterpret_cast<const f32x4 *>(a.bias + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const f32x4 v = acc[i][j] + bias;
            *reinterpret_cast<__attribute__((address_space(3))) u32x2 *>(
                so + (16 * j + l16) * 256 + (((2 * i + (q4 >> 1)) ^ l16) << 4) + ((q4 & 1) << 3)) =
                (u32x2){Elem<__bf16>::pack2(v.x, v.y), Elem<__bf16>::pack2(v.z, v.w)};
        }
    }
    store_rows<128, 16>(a, so, [](int r) { return r & 15; }, m0 + 128 * wm, n0 + 128 * wn, lane);
}

template <int NB, int MB, int S, int LS>
static void launch_ring(const F8MmArgs &a, hipStream_t s) {
    if (a.lines) {
        hipLaunchKernelGGL((f8_mm_ring<NB, MB, LS, true>), dim3(a.n_blocks), dim3(256), 0, s, a);
        return;
    }
    hipLaunchKernelGGL((f8_mm_ring<NB, MB, S, false>), dim3(a.n_blocks), dim3(256), 0, s, a);
}

// (with 256 tokens three stages are all of LDS, and LINES leaves too little on
// its way: 3,000 x 2500 x 2320 27.4 us, without 26.6)
template <int NB, int MB, int S>
static void launch_grid(const F8MmArgs &a, hipStream_t s) {
    if constexpr (S > 3) {
        if (a.lines) {
            hipLaunchKernelGGL((f8_mm_grid<NB, MB, S, true>), dim3(a.n_blocks), dim3(256), 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((f8_mm_grid<NB, MB, S, false>), dim3(a.n_blocks), dim3(256), 0, s, a);
}

hipError_t launch_f8_mm(const F8MmArgs &a, int tile, hipStream_t s) {
    switch (tile) {
    case 101: launch_ring<1, 1, 4, 4>(a, s); break;
    case 202: launch_ring<2, 2, 4, 4>(a, s); break;
    case 401: launch_ring<4, 1, 3, 3>(a, s); break;
    case 402: launch_ring<4, 2, 3, 3>(a, s); break;
    case 405: launch_ring<4, 5, 1, 2>(a, s); break;
    case 10804: launch_grid<4, 2, 5>(a, s); break;
    case 10806: launch_grid<4, 3, 5>(a, s); break;
    case 10810: launch_grid<4, 5, 4>(a, s); break;
    case 10816: launch_grid<4, 8, 3>(a, s); break;
    case 11616: hipLaunchKernelGGL(f8_mm_tile, dim3(a.n_blocks), dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kdfa
