"""GPU checks of what writes 8-bit rows (include/kd_f8.h): kd_f8_quantize
bitwise against the oracle, and kd_f8_norm_run, whose F32 norm may round
differently from the oracle's float64 one by EPS_Y, so that a code is one of
the two that y (1 - EPS_Y) and y (1 + EPS_Y) round to, and a scale likewise."""
import numpy as np
import pytest
import torch

import kd_f8
import kd_oracle_f8 as of
from f8_common import DEV, announce, from_rows

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# y = s / rms * w.  rms is within a few roundings of double; as two F32 it is
# within 2^-47.  s / rms is a product and what its rounding left, the latter
# within 2^-24 of itself twice over: 2^-46 of the product; times w that rest is
# rounded again, 2^-47, and the sum once, 2^-24.  In all less than 2^-23.
EPS_Y = 2.0 ** -23


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def guarded(M, K):
    """Rows with untouched memory around them: (Rows, codes store, scales store)."""
    nb = kd_f8.blocks(K)
    words = (nb + 3) // 4 * 4 + 4
    codes = torch.full((M + 2, K + 32), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((M + 2, words), 0x55, dtype=torch.uint8, device=DEV)
    return (kd_f8.Rows(codes[1:M + 1, 16:16 + K].view(torch.float8_e4m3fn), scales[1:M + 1, :nb].view(torch.float8_e8m0fnu)),
            codes, scales)


def check_guard(codes, scales, M, K):
    c, s = codes.clone(), scales.clone()
    c[1:M + 1, 16:16 + K] = 0x55
    s[1:M + 1, :kd_f8.blocks(K)] = 0x55
    assert bool((c == 0x55).all()) and bool((s == 0x55).all()), "written outside the rows"


def same_codes(got, want):
    """Equal codes (any NaN code for a NaN)."""
    nan = (got & 127) == 127
    return np.array_equal(nan, (want & 127) == 127) and np.array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 128), (3, 272), (5, 2048), (37, 144), (130, 1552), (7, 4096), (2, 16400)])
def test_quantize(dt, M, K):
    _need_gpu()
    announce(f"quantize {M} x {K} {dt}")
    rng = np.random.default_rng(M * K)
    lo, hi = (-8, 3) if dt == F16 else (-30, 30)
    x = torch.from_numpy((rng.standard_normal((M, K)) * np.exp(rng.uniform(lo, hi, (M, 1)))).astype(np.float32)).to(dt)
    out, codes, scales = guarded(M, K)
    kd_f8.run(kd_f8.quantize_desc(x.to(DEV), out))
    torch.cuda.synchronize()
    c, s = of.quantize(x.float().numpy())
    gc, gs = from_rows(out)
    assert np.array_equal(gs, s)
    assert np.array_equal(gc, c)
    check_guard(codes, scales, M, K)


def test_quantize_every_f16_value():
    """Every finite F16 value beside the largest of a block, so that both the
    scale and the rounding meet every mantissa."""
    _need_gpu()
    announce("quantize all F16 values")
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(F16)
    v = v[torch.isfinite(v)]
    x = v[:v.numel() // 128 * 128].view(-1, 128)
    for tops in (448.0, 450.0, 65504.0, 0.0):
        y = torch.cat([x, torch.full((x.shape[0], 16), tops, dtype=F16)], 1)
        y = torch.cat([y[:, 128:], y[:, :112]], 1).contiguous()
        r = kd_f8.quantize(y.to(DEV))
        gc, gs = from_rows(r)
        c, s = of.quantize(y.float().numpy())
        assert np.array_equal(gs, s) and np.array_equal(gc, c), tops


def test_quantize_borders_and_specials():
    _need_gpu()
    announce("quantize borders")
    big = float(np.finfo(np.float32).max)
    tops = [0.0, -0.0, 1e-45, 1e-40, 2.0 ** -126, 448 * 2.0 ** -127, 2.0 ** -118, 1.75, 1.7500001, -1.75, 448.0, 448.00003, 3e38, big,
            -big, np.inf, -np.inf, np.nan]
    x = np.zeros((len(tops), 272), dtype=np.float32)
    for i, t in enumerate(tops):
        x[i, 5], x[i, 130], x[i, 271] = t, t / 3 if np.isfinite(t) else 1.0, t / 64 if np.isfinite(t) else 2.0
    for dt in (F32, BF16):
        xt = torch.from_numpy(x).to(dt)
        gc, gs = from_rows(kd_f8.quantize(xt.to(DEV)))
        with np.errstate(invalid="ignore"):
            c, s = of.quantize(xt.float().numpy())
        assert np.array_equal(gs, s)
        assert same_codes(gc, c)


def test_quantize_rows_of_three_dimensions_and_strides():
    _need_gpu()
    announce("quantize 3-D strided")
    x = torch.randn((4, 6, 640), generator=torch.Generator().manual_seed(5)).to(DEV)
    part = x[..., 128:128 + 272]
    r = kd_f8.quantize(part)
    assert r.codes.shape == (4, 6, 272) and r.scales.shape == (4, 6, 3)
    c, s = of.quantize(part.cpu().numpy().reshape(24, 272))
    gc, gs = from_rows(r)
    assert np.array_equal(gc, c) and np.array_equal(gs, s)


def test_quantize_more_rows_than_one_sweep_of_workgroups():
    """Offsets past 32 bits: 2.2e9 values in rows of 16."""
    _need_gpu()
    announce("quantize 140,000,000 x 16")
    M = 140_000_000
    out = kd_f8.empty_rows((M,), 16, DEV)
    out.codes.view(torch.uint8).fill_(0x55)
    out.scales.view(torch.uint8).fill_(0x55)
    x = torch.zeros((M, 16), dtype=BF16, device=DEV)
    x[:, 3] = (torch.arange(M, device=DEV) % 251 - 125).to(BF16)
    kd_f8.run(kd_f8.quantize_desc(x, out))
    torch.cuda.synchronize()
    at = torch.randint(0, M, (4096,), generator=torch.Generator().manual_seed(6)).to(DEV)
    at = torch.cat([at, torch.arange(M - 512, M, device=DEV), torch.arange(512, device=DEV)])
    c, s = of.quantize(x[at].float().cpu().numpy())
    assert np.array_equal(out.codes.view(torch.uint8)[at].cpu().numpy(), c)
    assert np.array_equal(out.scales.view(torch.uint8)[at].cpu().numpy(), s)


def check_norm(x, residual, weight, eps, out, total):
    """out and total against the oracle."""
    s = x.float().cpu()
    if residual is not None:
        s = (s + residual.float().cpu()).to(residual.dtype)
        assert torch.equal(total.cpu().view(torch.uint8), s.view(torch.uint8)), "sum"
        s = s.float()
    K = s.shape[-1]
    y = of.rms_norm(s.double().numpy().reshape(-1, K), weight.cpu().numpy(), eps)
    gc, gs = from_rows(out)
    lo, hi = y * (1 - EPS_Y), y * (1 + EPS_Y)
    s_lo, s_hi = of.scale_bytes(lo), of.scale_bytes(hi)
    assert np.all((gs == s_lo) | (gs == s_hi)), "scales"
    factor = np.repeat(2.0 ** (127.0 - gs.astype(np.float64)), 128, axis=1)[:, :K]
    assert np.all((gc == of.round_e4m3(np.clip(lo * factor, -448, 448))) | (gc == of.round_e4m3(np.clip(hi * factor, -448, 448)))), "codes"


@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, None), (F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("M,K", [(1, 16), (2, 3584), (3, 272), (9, 512), (4, 528), (1030, 2064), (5, 2048), (1025, 1552), (1500, 4096),
                                 (3, 4112), (2, 16384), (3, 16400), (2, 32768)])
def test_norm(xt, rt, M, K):
    _need_gpu()
    announce(f"norm {M} x {K} {xt} {rt}")
    g = torch.Generator().manual_seed(M * 7 + K)
    x = torch.randn((M, K), generator=g).to(xt).to(DEV)
    r = None if rt is None else (3 * torch.randn((M, K), generator=g)).to(rt).to(DEV)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(DEV)
    out, codes, scales = guarded(M, K)
    total = None if r is None else torch.empty_like(r)
    kd_f8.run(kd_f8.norm_desc(x, w, out, r, total))
    torch.cuda.synchronize()
    check_norm(x, r, w, 1e-6, out, total)
    check_guard(codes, scales, M, K)


@pytest.mark.parametrize("M", [4, 1100])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_norm_in_place(into, M):
    """The sum over its own operand: the same bits as into another tensor."""
    _need_gpu()
    announce(f"norm in place {into} {M}")
    g = torch.Generator().manual_seed(8)
    x, r = (torch.randn((M, 3584), generator=g).to(DEV) for _ in range(2))
    w = torch.rand(3584, generator=g).to(DEV)
    want, total = kd_f8.add_rms_norm(x, w, r)
    out = kd_f8.empty_rows((M,), 3584, DEV)
    kd_f8.run(kd_f8.norm_desc(x, w, out, r, r if into == "residual" else x))
    torch.cuda.synchronize()
    assert torch.equal(r if into == "residual" else x, total)
    assert all(np.array_equal(a, b) for a, b in zip(from_rows(out), from_rows(want)))


def test_norm_of_zeros_specials_and_large_values():
    _need_gpu()
    announce("norm specials")
    K = 400
    x = torch.randn((6, K), generator=torch.Generator().manual_seed(9))
    x[0] = 0.0
    x[1, 200] = float("nan")
    x[2, 130] = float("inf")
    x[3] *= 1e12
    x[4] *= 1e-15
    x[5, :] = 0.0
    x[5, 399] = 1e-3
    w = torch.ones(K)
    out, same = kd_f8.add_rms_norm(x.to(DEV), w.to(DEV))
    torch.cuda.synchronize()
    gc, gs = from_rows(out)
    assert np.all(gs[0] == 0) and np.all(gc[0] & 127 == 0)
    # a NaN makes its row's mean NaN, and with it every value of the row
    assert np.all(gs[1] == 255) and np.all(gc[1] & 127 == 127)
    # an infinity: NaN in its own block, zero elsewhere (finite / infinity)
    assert gs[2].tolist() == [0, 255, 0, 0] and np.all(gc[2, :128] & 127 == 0) and np.all(gc[2, 128:256] & 127 == 127)
    keep = [3, 4, 5]
    part = kd_f8.Rows(out.codes[keep], out.scales.view(torch.uint8)[keep].view(torch.float8_e8m0fnu))
    check_norm(x[keep], None, w, 1e-6, part, None)


def test_norm_without_eps_and_with_a_large_one():
    _need_gpu()
    announce("norm eps")
    x = torch.randn((5, 256), generator=torch.Generator().manual_seed(10)).to(DEV)
    w = torch.ones(256, device=DEV)
    for eps in (0.0, 1e-6, 10.0):
        out, _ = kd_f8.add_rms_norm(x, w, eps=eps)
        torch.cuda.synchronize()
        check_norm(x, None, w, eps, out, None)


@pytest.mark.parametrize("K", [256, 3600, 16400])
def test_norm_of_rows_at_either_end_of_f32(K):
    """Without eps: 1 / rms beyond F32, below its normal numbers, and near."""
    _need_gpu()
    announce(f"norm ends of F32, {K}")
    x = torch.randn((9, K), generator=torch.Generator().manual_seed(11)).clamp(-4, 4)
    for i, top in enumerate((1e-44, 1e-40, 1e-38, 2.0 ** -99, 2.0 ** 99, 1e37, 8e37)):
        x[i] *= top
    x[7] = 0.0
    x[7, K - 1] = 1e-45
    x[8] = float(np.finfo(np.float32).max)
    w = 1 + 0.3 * torch.rand(K, generator=torch.Generator().manual_seed(12))
    for r in (None, torch.zeros_like(x)):
        out, total = kd_f8.add_rms_norm(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV), eps=0.0)
        torch.cuda.synchronize()
        check_norm(x, r, w, 0.0, out, total)


def test_norm_of_more_rows_than_workgroups():
    """Rows past the grid's first sweep, in each of the row layouts."""
    _need_gpu()
    for M, K in ((4_300_000, 16), (1_060_000, 528)):
        announce(f"norm {M} x {K}")
        x = (torch.arange(M, device=DEV, dtype=F32)[:, None] % 97 + torch.arange(K, device=DEV)[None] % 13 - 5).to(BF16)
        w = torch.ones(K, device=DEV)
        out, _ = kd_f8.add_rms_norm(x, w)
        torch.cuda.synchronize()
        at = torch.cat([torch.arange(64), torch.arange(M - 64, M), torch.randint(0, M, (512,), generator=torch.Generator().manual_seed(1))]).to(DEV)
        part = kd_f8.Rows(out.codes.view(torch.uint8)[at].view(torch.float8_e4m3fn), out.scales.view(torch.uint8)[at].view(torch.float8_e8m0fnu))
        check_norm(x[at], None, w, 1e-6, part, None)
        del x, out
