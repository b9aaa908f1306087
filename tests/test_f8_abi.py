"""Host-side checks of the 8-bit linear path's C ABI (include/kd_f8.h), no
GPU: exports, struct layout, what each *_supports accepts and refuses with
its reason, and that a refused call enqueues nothing."""
import ctypes
import re

import pytest
import torch

import kd_f8
import kd_fa

T = ctypes.sizeof(kd_fa.KdFaTensor)
E4M3, E8M0, BF16, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


def rows(*shape):
    return kd_f8.empty_rows(shape[:-1], shape[-1], "cpu")


def reason(make):
    """The status that a descriptor is refused with."""
    with pytest.raises(kd_fa.KdFaError) as e:
        make()
    return e.value.status


def test_library_exports_every_symbol():
    syms = kd_f8.header_symbols()
    assert set(syms) == {"kd_f8_quantize_supports", "kd_f8_quantize", "kd_f8_norm_supports", "kd_f8_norm_run",
                         "kd_f8_mm_supports", "kd_f8_mm_run"}
    for s in syms:
        assert hasattr(kd_fa.lib(), s), s


def test_structs_and_type_ids_equal_the_header():
    assert ctypes.sizeof(kd_f8.KdF8Rows) == 2 * T
    assert ctypes.sizeof(kd_f8.KdF8QuantizeDesc) == 3 * T
    assert ctypes.sizeof(kd_f8.KdF8NormDesc) == 6 * T + 8
    assert ctypes.sizeof(kd_f8.KdF8MmDesc) == 6 * T
    text = open(kd_f8.HEADER_PATH).read()
    ids = {m.group(1): int(m.group(2)) for m in re.finditer(r"\bKD_F8_(TYPE_[A-Z0-9]+)\s*=\s*(-?\d+)", text)}
    assert len(ids) == 5
    for name, value in ids.items():
        assert getattr(kd_f8, name) == value, name
    assert int(re.search(r"#define KD_F8_BLOCK (\d+)", text).group(1)) == kd_f8.BLOCK


def test_rows_hold_codes_and_their_scales():
    r = rows(2, 3, 272)
    assert r.codes.shape == (2, 3, 272) and r.scales.shape == (2, 3, 3) and r.scales.stride() == (12, 4, 1)
    r.scales.view(torch.uint8).fill_(127)
    assert torch.equal(r.to("cpu").scales.view(torch.uint8), r.scales.view(torch.uint8))
    assert rows(3, 1040).codes.stride() == (1152, 1) and rows(3, 1040).codes.shape == (3, 1040)
    with pytest.raises(ValueError):
        kd_f8.Rows(torch.zeros((4, 128)), r.scales)
    with pytest.raises(ValueError):
        kd_f8.Rows(torch.zeros((4, 128), dtype=torch.uint8).view(E4M3), torch.zeros((4, 2), dtype=torch.uint8).view(E8M0))


@pytest.mark.parametrize("dt", [F32, BF16, torch.float16])
def test_quantize_accepts(dt):
    kd_f8.quantize_desc(torch.zeros((3, 5, 272), dtype=dt), rows(3, 5, 272))
    kd_f8.quantize_desc(torch.zeros((1, 16), dtype=dt), rows(1, 16))
    kd_f8.quantize_desc(torch.zeros((0, 128), dtype=dt), rows(0, 128))
    kd_f8.quantize_desc(torch.zeros(128, dtype=dt), rows(128))
    kd_f8.quantize_desc(torch.zeros((4, 512), dtype=dt)[:, 128:384], rows(4, 256))     # strided rows
    kd_f8.quantize_desc(torch.zeros((4, 7, 32), dtype=dt)[:, -1:], rows(4, 1, 32))     # each sequence's last row


def test_quantize_refuses():
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 24)), rows(2, 24))) == kd_fa.ERR_SHAPE       # K % 16
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 0)), rows(2, 0))) == kd_fa.ERR_SHAPE
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 32)), rows(3, 32))) == kd_fa.ERR_SHAPE       # rows
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 32)), rows(2, 48))) == kd_fa.ERR_SHAPE       # K
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 34))[:, 1:33], rows(2, 32))) == kd_fa.ERR_LAYOUT
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((32, 2)).t(), rows(2, 32))) == kd_fa.ERR_LAYOUT  # K strided
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((4, 3, 32))[:, :2], rows(4, 2, 32))) == kd_fa.ERR_LAYOUT
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((1, 32)).expand(2, 32), rows(2, 32))) == kd_fa.ERR_LAYOUT
    r = rows(2, 32)
    packed = kd_f8.Rows(r.codes, torch.zeros((2, 1), dtype=torch.uint8).view(E8M0))    # scale rows 1 byte apart
    assert reason(lambda: kd_f8.quantize_desc(torch.zeros((2, 32)), packed)) == kd_fa.ERR_LAYOUT
    d = kd_f8.quantize_desc(torch.zeros((2, 32)), r)
    d.x.type = kd_f8.TYPE_E4M3
    assert _status(d) == kd_fa.ERR_TYPE
    d = kd_f8.quantize_desc(torch.zeros((2, 32)), r)
    d.out.scales.type = kd_f8.TYPE_E4M3
    assert _status(d) == kd_fa.ERR_TYPE
    d = kd_f8.quantize_desc(torch.zeros((2, 32)), r)
    d.x.data = None
    assert _status(d) == kd_fa.ERR_NULL


def _status(d):
    """What the entry point itself returns (no device is touched before)."""
    return kd_f8._RUN[type(d)][1](ctypes.byref(d), None)


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("rt", [F32, BF16, None])
def test_norm_accepts(xt, rt):
    x, w = torch.zeros((3, 5, 272), dtype=xt), torch.ones(272)
    r = None if rt is None else torch.zeros((3, 5, 272), dtype=rt)
    kd_f8.norm_desc(x, w, rows(3, 5, 272), r, None if r is None else torch.empty_like(r))
    if r is not None:
        kd_f8.norm_desc(x, w, rows(3, 5, 272), r, r)                    # in place
    if xt == rt:
        kd_f8.norm_desc(x, w, rows(3, 5, 272), r, x)
    kd_f8.norm_desc(torch.zeros((0, 64), dtype=xt), torch.ones(64), rows(0, 64))
    kd_f8.norm_desc(torch.zeros((1, 32768), dtype=xt), torch.ones(32768), rows(1, 32768), eps=0.0)


def test_norm_refuses():
    x, w, out = torch.zeros((2, 32)), torch.ones(32), rows(2, 32)
    assert reason(lambda: kd_f8.norm_desc(x, w, out, residual=x)) == kd_fa.ERR_NULL                 # no sum
    assert reason(lambda: kd_f8.norm_desc(x, w, out, sum=x)) == kd_fa.ERR_NULL                      # no residual
    assert reason(lambda: kd_f8.norm_desc(x, w, out, x, x.bfloat16())) == kd_fa.ERR_TYPE
    assert reason(lambda: kd_f8.norm_desc(x.half(), w, out)) == kd_fa.ERR_TYPE
    assert reason(lambda: kd_f8.norm_desc(x, w.bfloat16(), out)) == kd_fa.ERR_TYPE
    assert reason(lambda: kd_f8.norm_desc(x, torch.ones(48), out)) == kd_fa.ERR_SHAPE
    assert reason(lambda: kd_f8.norm_desc(x, torch.ones((2, 32)), out)) == kd_fa.ERR_SHAPE
    assert reason(lambda: kd_f8.norm_desc(x, torch.ones(64)[::2], out)) == kd_fa.ERR_LAYOUT
    assert reason(lambda: kd_f8.norm_desc(x, torch.ones(33)[1:], out)) == kd_fa.ERR_LAYOUT
    assert reason(lambda: kd_f8.norm_desc(x, w, out, torch.zeros((3, 32)), torch.zeros((3, 32)))) == kd_fa.ERR_SHAPE
    for eps in (-1e-6, float("nan"), float("inf")):
        assert reason(lambda: kd_f8.norm_desc(x, w, out, eps=eps)) == kd_fa.ERR_PARAM
    big = 32768 + 16
    assert reason(lambda: kd_f8.norm_desc(torch.zeros((1, big)), torch.ones(big), rows(1, big))) == kd_fa.ERR_SHAPE


def test_linear_accepts():
    kd_f8.linear_desc(rows(3, 5, 272), rows(64, 272), torch.empty((3, 5, 64), dtype=BF16), torch.ones(64))
    kd_f8.linear_desc(rows(1, 16), rows(4, 16), torch.empty((1, 4), dtype=BF16))
    kd_f8.linear_desc(rows(0, 16), rows(4, 16), torch.empty((0, 4), dtype=BF16))
    kd_f8.linear_desc(rows(3, 16), rows(0, 16), torch.empty((3, 0), dtype=BF16))
    kd_f8.linear_desc(rows(3, 16), rows(4, 16), torch.empty((3, 12), dtype=BF16)[:, 4:8])           # strided dst


def test_linear_refuses():
    x, w, dst = rows(3, 32), rows(8, 32), torch.empty((3, 8), dtype=BF16)
    assert reason(lambda: kd_f8.linear_desc(x, w, dst.float())) == kd_fa.ERR_TYPE
    assert reason(lambda: kd_f8.linear_desc(x, w, dst, torch.ones(8, dtype=BF16))) == kd_fa.ERR_TYPE
    assert reason(lambda: kd_f8.linear_desc(x, w, dst, torch.ones(7))) == kd_fa.ERR_SHAPE
    assert reason(lambda: kd_f8.linear_desc(x, w, dst, torch.ones(9)[1:])) == kd_fa.ERR_LAYOUT
    assert reason(lambda: kd_f8.linear_desc(x, rows(8, 48), dst)) == kd_fa.ERR_SHAPE                # K
    assert reason(lambda: kd_f8.linear_desc(x, rows(2, 4, 32), dst)) == kd_fa.ERR_SHAPE             # w of rank 3
    assert reason(lambda: kd_f8.linear_desc(x, rows(6, 32), torch.empty((3, 6), dtype=BF16))) == kd_fa.ERR_SHAPE   # N % 4
    assert reason(lambda: kd_f8.linear_desc(x, w, torch.empty((4, 8), dtype=BF16))) == kd_fa.ERR_SHAPE
    assert reason(lambda: kd_f8.linear_desc(x, w, torch.empty((3, 12), dtype=BF16)[:, 2:10])) == kd_fa.ERR_LAYOUT
    wide = torch.zeros((3, 48), dtype=torch.uint8).view(E4M3)[:, 8:40]                              # rows not at 16 bytes
    assert reason(lambda: kd_f8.linear_desc(kd_f8.Rows(wide, x.scales), w, dst)) == kd_fa.ERR_LAYOUT
    d = kd_f8.linear_desc(x, w, dst)
    d.x.codes.nb[1] = 1 << 24                                          # 256 rows past 32 bits
    assert _status(d) == kd_fa.ERR_LAYOUT
    d = kd_f8.linear_desc(x, w, dst)
    d.w.scales.data = None
    assert _status(d) == kd_fa.ERR_NULL


def test_sizes_beyond_32_bits_are_refused():
    d = kd_f8.linear_desc(rows(3, 32), rows(8, 32), torch.empty((3, 8), dtype=BF16))
    for t in (d.x.codes, d.x.scales, d.dst):
        t.ne[1] = 2 ** 31
    assert _status(d) == kd_fa.ERR_LAYOUT
    d = kd_f8.quantize_desc(torch.zeros((2, 32)), rows(2, 32))
    for t in (d.x, d.out.codes, d.out.scales):
        t.ne[1], t.ne[2] = 2 ** 20, 2 ** 20
        t.nb[2] = t.nb[1] * 2 ** 20
    assert _status(d) == kd_fa.ERR_LAYOUT


def test_null_descriptors():
    kd_f8._lib()
    for desc, (sup, run) in kd_f8._RUN.items():
        why = ctypes.c_int(0)
        assert sup(None, ctypes.byref(why)) == 0 and why.value == kd_fa.ERR_NULL
        assert run(None, None) == kd_fa.ERR_NULL


def test_tensors_off_the_gpu_are_not_launched():
    with pytest.raises(ValueError):
        kd_f8.quantize(torch.zeros((2, 32)))
    with pytest.raises(ValueError):
        kd_f8.linear(rows(3, 32), rows(8, 32))
    with pytest.raises(ValueError):
        kd_f8.add_rms_norm(torch.zeros((2, 32)), torch.ones(32))


def test_no_rows_and_no_outputs_do_nothing():
    """Returned before any device work: also without a GPU."""
    assert _status(kd_f8.quantize_desc(torch.zeros((0, 128)), rows(0, 128))) == kd_fa.OK
    assert _status(kd_f8.norm_desc(torch.zeros((0, 64)), torch.ones(64), rows(0, 64))) == kd_fa.OK
    assert _status(kd_f8.linear_desc(rows(0, 16), rows(4, 16), torch.empty((0, 4), dtype=BF16))) == kd_fa.OK
    assert _status(kd_f8.linear_desc(rows(3, 16), rows(0, 16), torch.empty((3, 0), dtype=BF16))) == kd_fa.OK
