// kd_f8_host.cpp - C ABI of the 8-bit linear path (include/kd_f8.h):
// validation of the three descriptors, the choice of the product's tile and
// the launches.  Nothing here allocates device memory, synchronises or keeps
// pointers past the call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/kd_f8.h"
#include "kd_f8_kernel.h"
#include "kd_fa_kernel.h"

namespace {

constexpr int64_t kI32Max = 0x7fffffff;
constexpr uint64_t kU32Max = 0xffffffffull;

bool aligned(uint64_t x, uint64_t to) { return x % to == 0; }
bool aligned(const void *p, uint64_t to) { return aligned((uint64_t)reinterpret_cast<uintptr_t>(p), to); }

int64_t blocks_of(int64_t K) { return (K + kdfa::kF8Block - 1) / kdfa::kF8Block; }

// The rows of a [ne0, ne1, ne2, ne3] view and the bytes from one to the next
// (0 for a single row).  rows is -1 on a layout that has no one stride, or
// more rows than 32 bits count.
struct Rows { int64_t rows; uint64_t stride; };
Rows flat_rows(const kd_fa_tensor &t) {
    Rows r = {1, 0};
    for (int i = 1; i < 4; ++i) {
        if (t.ne[i] < 0) return {-1, 0};
        if (t.ne[i] == 0) return {0, 0};
    }
    for (int i = 1; i < 4; ++i) {
        if (t.ne[i] == 1) continue;
        if (r.rows == 1) r.stride = t.nb[i];
        else if (t.nb[i] != r.stride * (uint64_t)r.rows) return {-1, 0};
        if (t.ne[i] > kI32Max / r.rows) return {-1, 0};
        r.rows *= t.ne[i];
    }
    return r;
}

bool same_rows(const kd_fa_tensor &a, const kd_fa_tensor &b) {
    return a.ne[1] == b.ne[1] && a.ne[2] == b.ne[2] && a.ne[3] == b.ne[3];
}

// A view of width `width`, elements of `size` bytes back to back, rows at
// multiples of `align` that do not overlap.
int check_rows(const kd_fa_tensor &t, int64_t width, size_t size, size_t align) {
    if (t.ne[0] != width) return KD_FA_ERR_SHAPE;
    const Rows r = flat_rows(t);
    if (r.rows < 0) return KD_FA_ERR_LAYOUT;
    if (r.rows == 0 || width == 0) return KD_FA_OK;
    if (!t.data) return KD_FA_ERR_NULL;
    if (t.nb[0] != size && width > 1) return KD_FA_ERR_LAYOUT;
    if (!aligned(t.data, align)) return KD_FA_ERR_LAYOUT;
    if (r.rows > 1 && (!aligned(r.stride, align) || r.stride < (uint64_t)width * size)) return KD_FA_ERR_LAYOUT;
    return KD_FA_OK;
}

int check_f8(const kd_f8_rows &r, int64_t K) {
    if (r.codes.type != KD_F8_TYPE_E4M3 || r.scales.type != KD_F8_TYPE_E8M0) return KD_FA_ERR_TYPE;
    if (!same_rows(r.codes, r.scales)) return KD_FA_ERR_SHAPE;
    const int st = check_rows(r.codes, K, 1, 16);
    if (st != KD_FA_OK) return st;
    return check_rows(r.scales, blocks_of(K), 1, 4);
}

// K values a row: whole 16-byte chunks of codes, 32-bit indexes
int check_k(int64_t K) { return K <= 0 || K % 16 != 0 || K > kI32Max - 65536 ? KD_FA_ERR_SHAPE : KD_FA_OK; }

// tiles of 16 * sixteens rows that cover `rows`
int64_t tiles(int sixteens, int64_t rows) { return (rows + 16 * sixteens - 1) / (16 * sixteens); }

size_t type_size(int type) {
    return type == KD_F8_TYPE_F32 ? 4 : type == KD_F8_TYPE_BF16 || type == KD_F8_TYPE_F16 ? 2 : 0;
}

int validate(const kd_f8_quantize_desc *d) {
    if (!d) return KD_FA_ERR_NULL;
    if (!type_size(d->x.type)) return KD_FA_ERR_TYPE;
    const int64_t K = d->x.ne[0];
    int st = check_k(K);
    if (st != KD_FA_OK) return st;
    if (!same_rows(d->x, d->out.codes)) return KD_FA_ERR_SHAPE;
    st = check_rows(d->x, K, type_size(d->x.type), 16);
    return st != KD_FA_OK ? st : check_f8(d->out, K);
}

int validate(const kd_f8_norm_desc *d) {
    if (!d) return KD_FA_ERR_NULL;
    const auto two_types = [](int t) { return t == KD_F8_TYPE_F32 || t == KD_F8_TYPE_BF16; };
    if (!two_types(d->x.type)) return KD_FA_ERR_TYPE;
    const int64_t K = d->x.ne[0];
    int st = check_k(K);
    if (st != KD_FA_OK) return st;
    if (K > kdfa::kF8NormMaxK) return KD_FA_ERR_SHAPE;
    if (!same_rows(d->x, d->out.codes)) return KD_FA_ERR_SHAPE;
    st = check_rows(d->x, K, type_size(d->x.type), 16);
    if (st != KD_FA_OK) return st;
    const kd_fa_tensor &r = d->residual, &s = d->sum, &w = d->weight;
    if (flat_rows(d->x).rows > 0 && !r.data != !s.data) return KD_FA_ERR_NULL;
    if (r.data) {
        if (!two_types(r.type) || s.type != r.type) return KD_FA_ERR_TYPE;
        if (!same_rows(d->x, r) || !same_rows(d->x, s)) return KD_FA_ERR_SHAPE;
        st = check_rows(r, K, type_size(r.type), 16);
        if (st != KD_FA_OK) return st;
        st = check_rows(s, K, type_size(s.type), 16);
        if (st != KD_FA_OK) return st;
    }
    if (w.type != KD_F8_TYPE_F32) return KD_FA_ERR_TYPE;
    if (w.ne[1] != 1 || w.ne[2] != 1 || w.ne[3] != 1) return KD_FA_ERR_SHAPE;
    st = check_rows(w, K, 4, 16);
    if (st != KD_FA_OK) return st;
    if (!std::isfinite(d->eps) || d->eps < 0.0f) return KD_FA_ERR_PARAM;
    return check_f8(d->out, K);
}

int validate(const kd_f8_mm_desc *d) {
    if (!d) return KD_FA_ERR_NULL;
    const kd_fa_tensor &o = d->dst, &b = d->bias;
    if (o.type != KD_F8_TYPE_BF16) return KD_FA_ERR_TYPE;
    if (b.data && b.type != KD_F8_TYPE_F32) return KD_FA_ERR_TYPE;
    const int64_t K = d->w.codes.ne[0], N = d->w.codes.ne[1];
    int st = check_k(K);
    if (st != KD_FA_OK) return st;
    if (d->w.codes.ne[2] != 1 || d->w.codes.ne[3] != 1) return KD_FA_ERR_SHAPE;
    if (N < 0 || N > kI32Max - 256 || N % 4 != 0) return KD_FA_ERR_SHAPE;
    st = check_f8(d->w, K);
    if (st != KD_FA_OK) return st;
    st = check_f8(d->x, K);
    if (st != KD_FA_OK) return st;
    if (!same_rows(o, d->x.codes)) return KD_FA_ERR_SHAPE;
    const int64_t M = flat_rows(o).rows;
    if (M > kI32Max - 256 || tiles(8, N) * tiles(16, M) > kdfa::kF8MmMaxBlocks) return KD_FA_ERR_SHAPE;
    st = check_rows(o, N, 2, 8);
    if (st != KD_FA_OK) return st;
    if (b.data) {
        if (b.ne[1] != 1 || b.ne[2] != 1 || b.ne[3] != 1) return KD_FA_ERR_SHAPE;
        st = check_rows(b, N, 4, 16);
        if (st != KD_FA_OK) return st;
    }
    // a tile's rows are addressed with 32-bit offsets from its first
    for (const kd_fa_tensor *t : {&d->w.codes, &d->w.scales, &d->x.codes, &d->x.scales})
        if (flat_rows(*t).stride > kU32Max / 256) return KD_FA_ERR_LAYOUT;
    return KD_FA_OK;
}

int64_t stride_of(const kd_fa_tensor &t) { return (int64_t)flat_rows(t).stride; }

kdfa::F8RowsArgs rows_args(const kd_fa_tensor &x, const kd_f8_rows &out) {
    kdfa::F8RowsArgs a = {};
    a.x = static_cast<const char *>(x.data);
    a.x_nb1 = stride_of(x);
    a.x_type = x.type;
    a.codes = static_cast<char *>(out.codes.data);
    a.c_nb1 = stride_of(out.codes);
    a.scales = static_cast<char *>(out.scales.data);
    a.e_nb1 = stride_of(out.scales);
    a.M = (int32_t)flat_rows(x).rows;
    a.K = (int32_t)x.ne[0];
    a.blocks = (int32_t)blocks_of(x.ne[0]);
    return a;
}

int launched(hipError_t e) { return e == hipSuccess ? KD_FA_OK : KD_FA_ERR_LAUNCH; }

// The tile of a call: the one whose rounds of workgroups (256 CUs, `at_once`
// on each) take least time.  A round's time with every CU at it is `fixed`
// (first loads, sums and stores) + `stage` * the stages of 128 k; and the
// rounds' stages take no less than the call's bytes from HBM (4.8 TB/s).  The
// two figures of a tile are fitted to its times over 106 shapes (1 to 63,488
// tokens, 4 to 16,384 outputs, 16 to 16,384 k); over these the tile taken is
// in the mean 1.7% slower than the fastest of sixteen, at worst 21% (12,768 x
// 1448 x 224, 31 us).  Six more tiles tried were never more than 1% of that
// mean.
int choose_tile(int64_t M, int64_t N, int64_t K) {
    constexpr struct { int tile, at_once; double fixed, stage; } kTiles[] = {
        {101, 2, 3.2, 0.067},   {202, 1, 3.2, 0.099},   {401, 1, 3.8, 0.072},   {402, 1, 3.9, 0.088},   {405, 1, 4.0, 0.20},
        {10804, 1, 4.1, 0.22},  {10806, 1, 4.2, 0.29},  {10810, 1, 4.4, 0.455}, {10816, 1, 4.8, 0.68},  {11616, 1, 6.5, 1.14}};
    const double stream = ((double)(M + N) * (double)K + 2.0 * (double)M * (double)N) / 4.8e6;   // us
    const double stages = (double)blocks_of(K);
    int best = 10816;   // (the largest that takes any size)
    double least = 1e300;
    for (const auto &t : kTiles) {
        const int64_t n = tiles(t.tile / 100 % 100, N) * tiles(t.tile % 100, M);
        if (n > kdfa::kF8MmMaxBlocks || (t.tile == 11616 && (M < 256 || N < 256))) continue;
        const double rounds = (double)((n + 256 * t.at_once - 1) / (256 * t.at_once));
        const double cost = rounds * t.fixed + std::max(rounds * t.stage * stages, stream);
        if (cost < least) { least = cost; best = t.tile; }
    }
    return best;
}

}  // namespace

extern "C" {

int kd_f8_quantize_supports(const kd_f8_quantize_desc *desc, int *reason) {
    const int st = validate(desc);
    if (reason) *reason = st;
    return st == KD_FA_OK ? 1 : 0;
}

int kd_f8_norm_supports(const kd_f8_norm_desc *desc, int *reason) {
    const int st = validate(desc);
    if (reason) *reason = st;
    return st == KD_FA_OK ? 1 : 0;
}

int kd_f8_mm_supports(const kd_f8_mm_desc *desc, int *reason) {
    const int st = validate(desc);
    if (reason) *reason = st;
    return st == KD_FA_OK ? 1 : 0;
}

int kd_f8_quantize(const kd_f8_quantize_desc *desc, void *stream) {
    int st = validate(desc);
    if (st != KD_FA_OK) return st;
    const kdfa::F8RowsArgs a = rows_args(desc->x, desc->out);
    if (a.M == 0) return KD_FA_OK;
    st = kdfa::device_gfx950();
    if (st != KD_FA_OK) return st;
    return launched(kdfa::launch_f8_quantize(a, static_cast<hipStream_t>(stream)));
}

int kd_f8_norm_run(const kd_f8_norm_desc *desc, void *stream) {
    int st = validate(desc);
    if (st != KD_FA_OK) return st;
    kdfa::F8RowsArgs a = rows_args(desc->x, desc->out);
    if (a.M == 0) return KD_FA_OK;
    a.residual = static_cast<const char *>(desc->residual.data);
    a.r_nb1 = stride_of(desc->residual);
    a.sum = static_cast<char *>(desc->sum.data);
    a.s_nb1 = stride_of(desc->sum);
    a.s_type = desc->residual.type;
    a.weight = static_cast<const float *>(desc->weight.data);
    a.eps = desc->eps;
    a.inv_k = 1.0 / a.K;
    st = kdfa::device_gfx950();
    if (st != KD_FA_OK) return st;
    return launched(kdfa::launch_f8_norm(a, static_cast<hipStream_t>(stream)));
}

int kd_f8_mm_run(const kd_f8_mm_desc *desc, void *stream) {
    int st = validate(desc);
    if (st != KD_FA_OK) return st;
    const int64_t K = desc->w.codes.ne[0], N = desc->w.codes.ne[1], M = flat_rows(desc->x.codes).rows;
    if (M == 0 || N == 0) return KD_FA_OK;
    const int tile = choose_tile(M, N, K);
    const int64_t tiles_n = tiles(tile / 100 % 100, N), tiles_m = tiles(tile % 100, M);
    st = kdfa::device_gfx950();
    if (st != KD_FA_OK) return st;
    kdfa::F8MmArgs a;
    a.w = static_cast<const char *>(desc->w.codes.data);
    a.w_nb1 = stride_of(desc->w.codes);
    a.ws = static_cast<const char *>(desc->w.scales.data);
    a.ws_nb1 = stride_of(desc->w.scales);
    a.x = static_cast<const char *>(desc->x.codes.data);
    a.x_nb1 = stride_of(desc->x.codes);
    a.xs = static_cast<const char *>(desc->x.scales.data);
    a.xs_nb1 = stride_of(desc->x.scales);
    a.bias = static_cast<const float *>(desc->bias.data);
    a.dst = static_cast<char *>(desc->dst.data);
    a.d_nb1 = stride_of(desc->dst);
    a.M = (int32_t)M;
    a.N = (int32_t)N;
    a.K = (int32_t)K;
    a.tiles_n = (int32_t)tiles_n;
    a.tiles_m = (int32_t)tiles_m;
    a.n_blocks = (int32_t)(tiles_n * tiles_m);
    a.cols = 4;
    // (code rows that do not all start on 128-byte lines, where that pays)
    a.lines = K >= 1024 && (!aligned(desc->w.codes.data, 128) || !aligned(desc->x.codes.data, 128) || !aligned((uint64_t)(a.w_nb1 | a.x_nb1), 128));
    return launched(kdfa::launch_f8_mm(a, tile, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
