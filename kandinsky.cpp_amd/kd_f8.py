"""ctypes binding of the 8-bit linear path (include/kd_f8.h) in libkd_fa.so:
rows as e4m3 codes with one E8M0 scale (a power of two) for each 128
consecutive values, what makes them -- `quantize`, and `add_rms_norm`, the
residual addition and RMS norm ahead of a layer -- and the linear layer on
them, `linear`, beside kd_mm.linear.

`Rows` holds such rows: `codes` torch.float8_e4m3fn (..., K) and `scales`
torch.float8_e8m0fnu (..., ceil(K / 128)), whose rows start at multiples of 4
bytes (`empty_rows` makes them so, and lays the codes out as the product
reads them fastest).  Each operator has a descriptor over
existing tensors (`quantize_desc`, `norm_desc`, `linear_desc`), checked when
it is made, which `run` launches any number of times; the functions above
make their outputs -- tensors of the stream they run on -- and run once.  Inference only: no gradient is recorded.
There is no fallback path: the library must be built.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import re

import kd_fa

HEADER_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "kd_f8.h")

TYPE_F32 = 0
TYPE_F16 = 1
TYPE_BF16 = 30
TYPE_E4M3 = 4096
TYPE_E8M0 = 4097
BLOCK = 128


class KdF8Rows(ctypes.Structure):
    """struct kd_f8_rows: codes and scales."""

    _fields_ = [("codes", kd_fa.KdFaTensor), ("scales", kd_fa.KdFaTensor)]


class KdF8QuantizeDesc(ctypes.Structure):
    """struct kd_f8_quantize_desc."""

    _fields_ = [("x", kd_fa.KdFaTensor), ("out", KdF8Rows)]


class KdF8NormDesc(ctypes.Structure):
    """struct kd_f8_norm_desc."""

    _fields_ = [
        ("x", kd_fa.KdFaTensor),
        ("residual", kd_fa.KdFaTensor),
        ("weight", kd_fa.KdFaTensor),
        ("sum", kd_fa.KdFaTensor),
        ("out", KdF8Rows),
        ("eps", ctypes.c_float),
    ]


class KdF8MmDesc(ctypes.Structure):
    """struct kd_f8_mm_desc."""

    _fields_ = [("w", KdF8Rows), ("x", KdF8Rows), ("bias", kd_fa.KdFaTensor), ("dst", kd_fa.KdFaTensor)]


class Rows:
    """Rows in 8 bits: `codes` float8_e4m3fn (..., K), `scales`
    float8_e8m0fnu (..., ceil(K / 128)); value = code * scale."""

    def __init__(self, codes, scales):
        torch = kd_fa._torch()
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float8_e8m0fnu:
            raise ValueError(f"codes are float8_e4m3fn and scales float8_e8m0fnu, not {codes.dtype} and {scales.dtype}")
        if codes.dim() < 1 or tuple(scales.shape) != tuple(codes.shape[:-1]) + (blocks(codes.shape[-1]),):
            raise ValueError(f"codes {tuple(codes.shape)} need scales (..., ceil(K / {BLOCK})), not {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    def to(self, device):
        """The same rows on `device`."""
        out = empty_rows(self.codes.shape[:-1], self.codes.shape[-1], device)
        out.codes.copy_(self.codes)
        out.scales.copy_(self.scales)
        return out


def blocks(K: int) -> int:
    """Scales of a row of K values."""
    return (K + BLOCK - 1) // BLOCK


def empty_rows(rows, K: int, device) -> Rows:
    """Uninitialised Rows of shape (*rows, K): the scales' rows padded to
    words, the codes' to whole 128-byte lines from K = 1024 on (the product
    reads its operands by such pieces: packed rows of 3,600 take it 14.0 us at
    997 x 1540, padded ones 13.0, and many tokens 12% longer; below, the padding
    would weigh more)."""
    torch = kd_fa._torch()
    rows = tuple(rows)
    words, wide = (blocks(K) + 3) // 4 * 4, blocks(K) * BLOCK if K >= 1024 else K
    scales = torch.empty(rows + (words,), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    codes = torch.empty(rows + (wide,), dtype=torch.float8_e4m3fn, device=device)
    return Rows(codes[..., :K], scales[..., :blocks(K)])


_RUN = {}
_current_device = _current_stream = None   # () -> index, index -> handle


def _lib():
    global _current_device, _current_stream
    lib = kd_fa.lib()
    if not _RUN:
        torch = kd_fa._torch()
        # a small call is the host's time: torch.cuda's functions of these are
        # 2.5 of its 7 us (current_stream makes a Stream object)
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda i: torch.cuda.current_stream(i).cuda_stream)
        P, ci, cv = ctypes.POINTER, ctypes.c_int, ctypes.c_void_p
        for desc, sup, run_ in ((KdF8QuantizeDesc, lib.kd_f8_quantize_supports, lib.kd_f8_quantize),
                                (KdF8NormDesc, lib.kd_f8_norm_supports, lib.kd_f8_norm_run),
                                (KdF8MmDesc, lib.kd_f8_mm_supports, lib.kd_f8_mm_run)):
            sup.argtypes, sup.restype = [P(desc), P(ci)], ci
            run_.argtypes, run_.restype = [P(desc), cv], ci
            _RUN[desc] = (sup, run_)
    return lib


def header_symbols(path: str = HEADER_PATH) -> list[str]:
    """Function names declared in include/kd_f8.h."""
    with open(path) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    return sorted(set(re.findall(r"\b(kd_f8_\w+)\s*\(", text)))


def view(t) -> kd_fa.KdFaTensor:
    """ggml view of a torch tensor, the 8-bit types included."""
    torch = kd_fa._torch()
    eight = {torch.float8_e4m3fn: TYPE_E4M3, torch.float8_e8m0fnu: TYPE_E8M0}
    return kd_fa.view(t, None if t is None else eight.get(t.dtype))


def rows_view(r: Rows) -> KdF8Rows:
    out = KdF8Rows()
    out.codes, out.scales = view(r.codes), view(r.scales)
    return out


def _checked(d, what, *tensors):
    """d, if the library can execute it; it keeps the tensors alive."""
    d._keep = tuple(t for t in tensors if t is not None)
    d._device = d._keep[0].device
    d._index = d._device.index if d._device.type == "cuda" else None
    d._ref = ctypes.byref(d)
    if any(t.device != d._device for t in d._keep):
        raise ValueError(f"{what}: the tensors are on different devices")
    _lib()
    supports, d._enqueue = _RUN[type(d)]
    reason = ctypes.c_int(0)
    if not supports(d._ref, ctypes.byref(reason)):
        raise kd_fa.KdFaError(reason.value, what)
    return d


def quantize_desc(x, out: Rows) -> KdF8QuantizeDesc:
    """x (..., K) float32 / bfloat16 / float16 into `out`."""
    d = KdF8QuantizeDesc()
    d.x, d.out = view(x), rows_view(out)
    return _checked(d, "kd_f8_quantize", x, out.codes, out.scales)


def norm_desc(x, weight, out: Rows, residual=None, sum=None, eps=1e-6) -> KdF8NormDesc:
    """The RMS norm of x (..., K), or of x + residual, times `weight` (K,)
    float32 into `out`; the addition, rounded to residual's type, into `sum`
    (which may be `residual` or `x` itself)."""
    d = KdF8NormDesc()
    d.x, d.residual, d.weight, d.sum, d.out = view(x), view(residual), view(weight), view(sum), rows_view(out)
    d.eps = float(eps)
    return _checked(d, "kd_f8_norm_run", x, residual, weight, sum, out.codes, out.scales)


def linear_desc(x: Rows, w: Rows, dst, bias=None) -> KdF8MmDesc:
    """dst (..., N) bfloat16 = x (..., K) times w (N, K), plus bias (N,) float32."""
    d = KdF8MmDesc()
    d.w, d.x, d.bias, d.dst = rows_view(w), rows_view(x), view(bias), view(dst)
    return _checked(d, "kd_f8_mm_run", x.codes, x.scales, w.codes, w.scales, bias, dst)


def run(desc, stream=None) -> None:
    """Enqueue a descriptor's operator on `stream` (default: the current
    stream of its tensors' device)."""
    on = desc._index
    if on is None:
        raise ValueError(f"the tensors are on {desc._device}, not on a GPU")
    if _current_device() != on:
        with kd_fa._torch().cuda.device(on):
            return run(desc, stream)
    st = desc._enqueue(desc._ref, _current_stream(on) if stream is None else stream.cuda_stream)
    if st != kd_fa.OK:
        raise kd_fa.KdFaError(st, type(desc).__name__)


def _made_on(stream):
    """Tensors made in this context belong to `stream`: on another stream
    their memory might still be in use by what was enqueued there."""
    return contextlib.nullcontext() if stream is None else kd_fa._torch().cuda.stream(stream)


def quantize(x, stream=None) -> Rows:
    """x (..., K) as 8-bit rows."""
    with _made_on(stream):
        out = empty_rows(x.shape[:-1], x.shape[-1], x.device)
    run(quantize_desc(x, out), stream)
    return out


def add_rms_norm(x, weight, residual=None, eps=1e-6, stream=None):
    """(Rows, sum): the RMS norm of x + residual in 8 bits, and the addition
    in residual's type -- (Rows, x) without a residual."""
    torch = kd_fa._torch()
    with _made_on(stream):
        out = empty_rows(x.shape[:-1], x.shape[-1], x.device)
        total = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    run(norm_desc(x, weight, out, residual, total, eps), stream)
    return out, x if total is None else total


def linear(x: Rows, w: Rows, bias=None, dst=None, stream=None):
    """ops::linear on 8-bit rows: x (..., K) and w (N, K) -> (..., N) bfloat16."""
    torch = kd_fa._torch()
    if dst is None:
        with _made_on(stream):
            dst = torch.empty(tuple(x.shape[:-1]) + (w.shape[0],), dtype=torch.bfloat16, device=x.codes.device)
    run(linear_desc(x, w, dst, bias), stream)
    return dst
