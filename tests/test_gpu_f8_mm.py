"""GPU checks of the product on 8-bit rows (include/kd_f8.h): bitwise on
operands whose sums are exact in F32 in any order (f8_common.exact_rows), so
that any row, block, scale or token out of place shows; within the derived
bound on random ones."""
import numpy as np
import pytest
import torch

import kd_f8
import kd_oracle_f8 as of
from f8_common import BF16_HALF, DEV, announce, exact_rows, linear_tol, random_rows, round_bf16, to_rows

pytestmark = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# M, N, K, bias: one token to many, sizes at, below and past the tiles of
# every kernel, a last block of 16 to 128 values, one block to many
CASES = [
    (1, 4, 16, False), (1, 4, 128, True), (2, 20, 144, True), (3, 64, 112, False), (5, 132, 1040, True), (8, 260, 4096, True),
    (16, 68, 528, False), (16, 1000, 2064, True), (17, 64, 128, True), (31, 36, 640, False), (33, 100, 256, True), (47, 516, 1536, True),
    (64, 64, 512, False), (65, 68, 4112, True), (100, 1028, 272, True), (128, 128, 1024, False), (129, 132, 1040, True),
    (200, 260, 3600, True), (256, 256, 2048, False), (257, 516, 1168, True), (300, 4096, 128, True), (513, 772, 640, True),
    (700, 1540, 912, False), (1280, 512, 256, True), (1999, 1024, 144, True), (4100, 300, 400, True), (434, 372, 608, True),
    (97, 2164, 672, False), (34, 5576, 528, True), (290, 3816, 416, False), (1878, 788, 640, True), (3266, 856, 528, True),
    (947, 3244, 784, False), (1531, 4720, 336, True), (2594, 6704, 192, True),
]
# each tile's steady loop: many stages, the last whole or not
DEEP = [
    (3, 420, 5232, True), (17, 8, 6144, False), (18, 4104, 2240, True), (559, 444, 2048, False), (77, 2732, 3120, True),
    (765, 260, 4096, False), (108, 2332, 4112, True), (1730, 136, 6144, True), (1556, 604, 2384, False), (1386, 544, 4096, True),
    (176, 5716, 2384, True), (3695, 396, 3328, False), (1118, 1812, 4128, True), (4103, 412, 2304, False), (773, 4364, 6192, False),
    (3461, 792, 2048, True), (1292, 3732, 2096, True), (1406, 4208, 4352, False), (1558, 6684, 2080, False), (3539, 2836, 4352, True),
]
# tokens and outputs that take the same tile for every K of STAGE_K: one to
# thirteen stages, whole and not, through every kernel's first and last steps
STAGES = [(1, 4), (46, 76), (27, 4880), (36, 4180), (238, 1128), (3000, 132), (888, 1616), (877, 2592), (3062, 1244), (5275, 1016), (3154, 3324)]
STAGE_K = [16, 112, 128, 144, 256, 272, 384, 400, 512, 624, 640, 768, 784, 896, 1008, 1024, 1152, 1168, 1280, 1424, 1536, 1552, 1664]


def _exact(M, N, K, bias, seed=0):
    rng = np.random.default_rng(seed + M * 3 + N * 5 + K)
    xc, xs = exact_rows(rng, M, K)
    wc, ws = exact_rows(rng, N, K)
    b = rng.integers(-64, 65, N).astype(np.float32) if bias else None
    # (float64 products of exact values, on the GPU where they are many)
    xv, wv = (torch.from_numpy(of.decode(c, t)) for c, t in ((xc, xs), (wc, ws)))
    if M * N * K > 1e9:
        xv, wv = xv.to(DEV), wv.to(DEV)
    want = (xv @ wv.t()).cpu().numpy()
    if b is not None:
        want = want + b.astype(np.float64)
    return (to_rows(xc, xs, DEV), to_rows(wc, ws, DEV), None if b is None else torch.from_numpy(b).to(DEV), round_bf16(want))


@pytest.mark.parametrize("M,N,K,bias", CASES + DEEP)
def test_exact_sums(M, N, K, bias):
    _need_gpu()
    announce(f"mm exact {M} x {N} x {K}")
    x, w, b, want = _exact(M, N, K, bias)
    # dst inside a larger tensor: what lies around it stays
    store = torch.full((M + 2, N + 8), 77.0, dtype=torch.bfloat16, device=DEV)
    kd_f8.linear(x, w, b, dst=store[1:M + 1, 4:4 + N])
    torch.cuda.synchronize()
    assert torch.equal(store[1:M + 1, 4:4 + N].cpu(), want)
    store[1:M + 1, 4:4 + N] = 77.0
    assert bool((store == 77.0).all()), "written outside dst"


@pytest.mark.parametrize("M,N", STAGES)
def test_every_number_of_stages(M, N):
    _need_gpu()
    for K in STAGE_K:
        announce(f"mm stages {M} x {N} x {K}")
        x, w, b, want = _exact(M, N, K, True)
        got = kd_f8.linear(x, w, b)
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), want), K


@pytest.mark.parametrize("M,N,K,bias", [(2, 512, 4096, True), (16, 260, 3600, False), (60, 132, 992, True), (300, 516, 4096, True),
                                        (700, 260, 16384, True), (1500, 1028, 1040, False)])
def test_random_values(M, N, K, bias):
    _need_gpu()
    announce(f"mm random {M} x {N} x {K}")
    rng = np.random.default_rng(M + N + K)
    xc, xs = random_rows(rng, M, K)
    wc, ws = random_rows(rng, N, K)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    x, w = of.decode(xc, xs), of.decode(wc, ws)
    got = kd_f8.linear(to_rows(xc, xs, DEV), to_rows(wc, ws, DEV), None if b is None else torch.from_numpy(b).to(DEV))
    again = kd_f8.linear(to_rows(xc, xs, DEV), to_rows(wc, ws, DEV), None if b is None else torch.from_numpy(b).to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(got, again)
    ref = of.linear(x, w, b)
    err = np.abs(got.cpu().double().numpy() - ref)
    tol = linear_tol(x, w, ref)
    assert np.all(err <= tol), f"worst {np.max(err / tol):.3g} of the bound"
    # in norm the sums are far below dst's own rounding (half a step is 2^-8
    # at most, and 2^-8 / sqrt(3) at most in the root mean square)
    assert np.linalg.norm(err) <= 2.0 ** -8 / np.sqrt(3) * 1.05 * np.linalg.norm(ref)


def test_every_scale_reaches_its_own_block():
    """One block and one row at a time: scales over the whole range whose
    products stay in BF16's."""
    _need_gpu()
    announce("mm scales")
    M, N, K = 20, 36, 1200
    rng = np.random.default_rng(3)
    xc, _ = exact_rows(rng, M, K)
    wc, _ = exact_rows(rng, N, K)
    nb = 10
    # a row's blocks all but one are zero, so that no sum mixes magnitudes
    keep = rng.integers(0, nb, M)
    for m in range(M):
        xc[m] = np.where(np.arange(K) // 128 == keep[m], xc[m], 0)
    xs = rng.integers(1, 250, (M, nb)).astype(np.uint8)
    ws = np.zeros((N, nb), dtype=np.uint8)
    e = rng.integers(-30, 31, (N, nb))
    ws[:] = 127 + e
    want = of.linear(of.decode(xc, xs), of.decode(wc, ws))
    got = kd_f8.linear(to_rows(xc, xs, DEV), to_rows(wc, ws, DEV)).cpu().double().numpy()
    fine = (np.abs(want) < 1e38) & (np.abs(want) > 1e-35)
    assert fine.mean() > 0.7
    assert np.all(np.abs(got - want)[fine] <= BF16_HALF * np.abs(want)[fine])


def test_nan_rows_stay_in_their_rows():
    _need_gpu()
    announce("mm nan")
    M, N, K = 70, 132, 656
    rng = np.random.default_rng(4)
    xc, xs = exact_rows(rng, M, K)
    wc, ws = exact_rows(rng, N, K)
    want = of.linear(of.decode(xc, xs), of.decode(wc, ws))
    xc[3, 655] = 0x7F            # a NaN code in the last, shorter block
    xs[40, 2] = 255              # a NaN scale
    wc[9, 0] = 0xFF
    ws[131, 5] = 255
    bad = np.zeros((M, N), dtype=bool)
    bad[[3, 40]] = True
    bad[:, [9, 131]] = True
    got = kd_f8.linear(to_rows(xc, xs, DEV), to_rows(wc, ws, DEV)).cpu()
    assert np.array_equal(torch.isnan(got).numpy(), bad)
    keep = torch.from_numpy(~bad)
    assert torch.equal(got[keep], round_bf16(want)[keep])


@pytest.mark.parametrize("M,N,K", [(3, 64, 2064), (40, 4096, 1040), (77, 2732, 3120), (96, 3000, 4096), (300, 1500, 1552), (559, 444, 2048),
                                   (1292, 1500, 2096), (1999, 1024, 144), (700, 1028, 16), (1406, 4208, 1280), (2300, 3300, 1664)])
@pytest.mark.parametrize("lead,gap", [(16, 0), (112, 16), (0, 144), (64, 64), (48, 368)])
def test_rows_that_start_anywhere_in_a_line(M, N, K, lead, gap):
    """Codes `lead` bytes behind the start of a line, `gap` bytes between the
    rows, NaN in all that is not theirs."""
    _need_gpu()
    announce(f"mm {M} x {N} x {K} at {lead}, {gap} apart")
    x, w, b, want = _exact(M, N, K, True)

    def elsewhere(r, lead, gap):
        rows = r.codes.shape[0]
        store = torch.full((lead + rows * (K + gap) + 256,), 0x7F, dtype=torch.uint8, device=DEV)
        codes = store[lead:lead + rows * (K + gap)].view(rows, K + gap)[:, :K]
        codes.copy_(r.codes.view(torch.uint8))
        return kd_f8.Rows(codes.view(torch.float8_e4m3fn), r.scales)

    for xs, ws in (((lead, gap), (0, (-K) % 128)), ((0, (-K) % 128), (lead, gap)), ((lead, gap), (gap, lead))):
        got = kd_f8.linear(elsewhere(x, *xs), elsewhere(w, *ws), b)
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), want), (xs, ws)


def test_rows_of_three_dimensions_and_strided_operands():
    _need_gpu()
    announce("mm 3-D strided")
    B, L, N, K = 3, 40, 100, 272
    rng = np.random.default_rng(5)
    xc, xs = exact_rows(rng, B * L, K)
    wc, ws = exact_rows(rng, N, K)
    want = round_bf16(of.linear(of.decode(xc, xs), of.decode(wc, ws))).view(B, L, N)
    x = to_rows(xc, xs, DEV)
    # codes inside wider rows, scales inside wider rows
    wide = torch.zeros((B * L, K + 48), dtype=torch.uint8, device=DEV)
    wide[:, 32:32 + K] = x.codes.view(torch.uint8)
    wsc = torch.full((B * L, 12), 200, dtype=torch.uint8, device=DEV)
    wsc[:, 4:7] = x.scales.view(torch.uint8)
    xr = kd_f8.Rows(wide.view(B, L, K + 48)[..., 32:32 + K].view(torch.float8_e4m3fn),
                    wsc.view(B, L, 12)[..., 4:7].view(torch.float8_e8m0fnu))
    got = kd_f8.linear(xr, to_rows(wc, ws, DEV))
    torch.cuda.synchronize()
    assert got.shape == (B, L, N) and torch.equal(got.cpu(), want)


def test_token_rows_and_weight_rows_past_32_bits():
    """x of 4.3e9 bytes and dst rows past 2^31: the tile's offsets are its own."""
    _need_gpu()
    announce("mm 1,060,000 x 132 x 4096")
    M, N, K = 1_060_000, 132, 4096
    rng = np.random.default_rng(6)
    pc, ps = exact_rows(rng, 1000, K)
    wc, ws = exact_rows(rng, N, K)
    part = to_rows(pc, ps, DEV)
    x = kd_f8.empty_rows((M,), K, DEV)
    x.codes.view(torch.uint8).view(1060, 1000, K).copy_(part.codes.view(torch.uint8)[None])
    x.scales.view(torch.uint8).view(1060, 1000, -1).copy_(part.scales.view(torch.uint8)[None])
    got = kd_f8.linear(x, to_rows(wc, ws, DEV))
    torch.cuda.synchronize()
    want = round_bf16(of.linear(of.decode(pc, ps), of.decode(wc, ws))).to(DEV)
    for i in (0, 1, 523, 524, 1059):
        assert torch.equal(got[1000 * i:1000 * (i + 1)], want), i
