"""Helpers of the 8-bit linear path's tests: rows between torch and the
numpy oracle, inputs whose products are exact, and the tolerances."""
import numpy as np
import torch

import kd_f8
import kd_oracle_f8 as of

DEV = "cuda:0"


def announce(msg):
    print(f"[case] {msg}", flush=True)


def to_rows(codes, scales, device):
    """kd_f8.Rows on `device` of uint8 codes (M, K) and scale bytes; what pads
    the scales' rows is NaN."""
    M, nb = scales.shape
    store = torch.full((M, (nb + 3) // 4 * 4), of.NAN_BYTE, dtype=torch.uint8, device=device)
    r = kd_f8.Rows(torch.empty(codes.shape, dtype=torch.float8_e4m3fn, device=device),
                   store[:, :nb].view(torch.float8_e8m0fnu))
    r.codes.view(torch.uint8).copy_(torch.from_numpy(codes))
    r.scales.view(torch.uint8).copy_(torch.from_numpy(scales))
    return r


def from_rows(r):
    """(codes, scale bytes) as numpy arrays (rows flattened)."""
    K, nb = r.codes.shape[-1], r.scales.shape[-1]
    return (r.codes.cpu().contiguous().view(torch.uint8).numpy().reshape(-1, K),
            r.scales.cpu().contiguous().view(torch.uint8).numpy().reshape(-1, nb))


def exact_rows(rng, M, K):
    """Codes of integers of magnitude <= 8 and scales 1/2, 1 or 2.  The
    products of 16 neighbouring k lie within 7 bits and every partial sum of
    up to 16,384 of them is a multiple of 1/4 below 2^22: the product of two
    such operands is exact in F32 in any order."""
    codes = of.round_e4m3(rng.integers(-8, 9, (M, K)).astype(np.float64))
    return codes, rng.integers(126, 129, (M, (K + 127) // 128)).astype(np.uint8)


def random_rows(rng, M, K):
    """Normal values in 8 bits, a hundredth of the columns eight times as large."""
    y = rng.standard_normal((M, K)) * np.where(rng.random(K) < 0.01, 8.0, 1.0)
    return of.quantize(y.astype(np.float32))


def round_bf16(v):
    """float64 -> the nearest bfloat16 (through F32: exact for values of <= 24
    bits, which the exact cases' are)."""
    return torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).to(torch.bfloat16)


# Error of the product beside dst's rounding, as a part of sum |w x|.  Within
# 16 neighbouring k products are aligned to the largest exponent sum E of
# their operands and cut 13 bits below 2^E; the largest is at least 2^E, so
# the 15 others lose less than 15 * 2^-13 of it.  The F32 sums add their K /
# 16 + 8 roundings of 2^-24 each, K <= 65536: 2^-12.
SUM_TOL = 15 * 2.0 ** -13 + 2.0 ** -12
BF16_HALF = 2.0 ** -8


def linear_tol(x, w, ref):
    """Bound of |dst - ref| for float64 operands and result."""
    ab = SUM_TOL * (np.abs(x) @ np.abs(w).T)
    return BF16_HALF * (np.abs(ref) + ab) + ab
