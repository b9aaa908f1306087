"""The 8-bit oracle (oracle/kd_oracle_f8.py) against torch's own casts to
float8, closed forms of the scale rule and invariants (CPU)."""
import numpy as np
import pytest
import torch

import kd_oracle_f8 as of


def test_codes_stand_for_the_values_torch_reads():
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(v), np.isnan(of.e4m3_values()))
    assert np.array_equal(v[~np.isnan(v)], of.e4m3_values()[~np.isnan(v)])


def test_rounding_equals_torchs():
    rng = np.random.default_rng(1)
    v = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000) * 0.01, [0.0, -0.0, 448.0, -448.0]])
    mid = (of.e4m3_values()[:126] + of.e4m3_values()[1:127]) / 2       # every tie
    v = np.concatenate([v, mid, -mid]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(of.round_e4m3(v), want)


@pytest.mark.parametrize("amax,byte", [(448.0, 127), (np.nextafter(np.float32(448), np.float32(999)), 128), (896.0, 128),
                                       (1.0, 119), (1.75, 119), (1.7500001, 120), (0.0, 0), (2.0 ** -126, 0),
                                       (448 * 2.0 ** -127, 0), (448 * 2.0 ** -126, 1), (float(np.finfo(np.float32).max), 247),
                                       (np.inf, 255), (-np.inf, 255), (np.nan, 255)])
def test_scale_bytes(amax, byte):
    y = np.zeros((1, 130), dtype=np.float32)
    y[0, 7], y[0, 128] = amax, 1.0
    s = of.scale_bytes(y)
    assert s.tolist() == [[byte, 119]]


def test_quantized_values_are_within_half_a_step():
    rng = np.random.default_rng(2)
    y = (rng.standard_normal((40, 300)) * np.exp(rng.uniform(-20, 20, (40, 1)))).astype(np.float32)
    codes, s = of.quantize(y)
    scale = np.repeat(2.0 ** (s.astype(np.float64) - 127), 128, axis=1)[:, :300]
    err = np.abs(of.decode(codes, s) - y)
    assert np.all(err <= np.maximum(np.abs(y) * 2.0 ** -4, scale * 2.0 ** -10))
    # the largest code of a block uses the upper half of the range
    top = np.max(np.abs(of.blocked(of.e4m3_values()[codes])), axis=2)
    assert np.all(top >= 224)


def test_a_block_with_a_nan_or_infinity_is_nan_throughout():
    y = np.ones((2, 256), dtype=np.float32)
    y[0, 3], y[1, 200] = np.inf, np.nan
    d = of.decode(*of.quantize(y))
    assert np.all(np.isnan(d[0, :128])) and np.all(d[0, 128:] == 1)
    assert np.all(d[1, :128] == 1) and np.all(np.isnan(d[1, 128:]))


def test_norm_of_a_constant_row():
    s = np.full((1, 64), 3.0)
    y = of.rms_norm(s, np.arange(64), 0.0)
    assert np.allclose(y[0], np.arange(64), rtol=1e-14)
    assert np.array_equal(of.rms_norm(np.zeros((1, 64)), np.ones(64), 1e-6), np.zeros((1, 64)))
