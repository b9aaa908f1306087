"""The tile that kd_f8_mm_run takes (kandinsky.cpp_amd/csrc/kd_f8_host.cpp),
on the host alone."""
import math
import random

import pytest

import kd_fa
from f8_plan import TILES, desc, outputs, plan, run, tokens
from test_gpu_f8_mm import CASES, DEEP, STAGE_K, STAGES


@pytest.mark.parametrize("M,N,K", [(2 ** 31 - 257, 4, 32), (1, 2 ** 30 - 4, 32), (200, 2 ** 30 - 512, 64), (2 ** 24, 2 ** 14, 16),
                                   (1, 4, 2 ** 31 - 65536 - 16 - (2 ** 31 - 65536) % 16)])
def test_sizes_within_a_tile_of_2_31(M, N, K):
    d = desc(M, N, K)
    if K > 2 ** 24 - 16:
        # such rows lie further apart than a tile's 32-bit offsets reach, but one row has no stride
        for r in (d.w, d.x):
            assert r.codes.nb[1] == K
    st, p = run(d)
    if K > 2 ** 24 and N > 1:
        assert st == kd_fa.ERR_LAYOUT
        return
    assert st == kd_fa.OK
    assert p.tiles_m == -(-M // tokens(p.tile)) and p.tiles_n == -(-N // outputs(p.tile))
    assert p.n_blocks == p.tiles_m * p.tiles_n <= 2 ** 23   # 256 threads each: a grid of less than 2^32
    # the last tile's row and output indexes are 32-bit
    assert p.tiles_m * tokens(p.tile) <= 2 ** 31 and p.tiles_n * outputs(p.tile) <= 2 ** 31


def test_more_tiles_than_a_launch_holds_are_refused():
    for M, N in ((2 ** 26, 2 ** 21), (1, 2 ** 31 - 260), (257, 2 ** 30)):
        st, _ = run(desc(M, N, 32))
        assert st == kd_fa.ERR_SHAPE


def test_one_row_of_dst_may_have_any_stride():
    st, p = run(desc(1, 64, 128, d_nb1=0))
    assert st == kd_fa.OK and p.d_nb1 == 0
    st, _ = run(desc(2, 64, 128, d_nb1=0))
    assert st == kd_fa.ERR_LAYOUT


def test_every_size_has_a_tile_and_it_covers_the_call():
    rng = random.Random(3)
    seen = set()
    for _ in range(4000):
        M, N, K = (int(math.exp(rng.uniform(math.log(a), math.log(b)))) for a, b in ((1, 70000), (4, 20000), (16, 17000)))
        p = plan(M, N // 4 * 4, K // 16 * 16)
        seen.add(p.tile)
        assert p.n_blocks == -(-p.M // tokens(p.tile)) * -(-p.N // outputs(p.tile))
        assert p.tile != 11616 or (M >= 256 and N >= 256)      # its tiles are whole
    assert seen == set(TILES)      # none that no call reaches


def test_gpu_cases_run_every_tile():
    """Each tile by calls with partial tiles both ways; with k of one and of
    many stages, ending on a stage and inside it."""
    for cases in (CASES, DEEP):
        taken = {}
        for M, N, K, _ in cases:
            taken.setdefault(plan(M, N, K).tile, []).append((M, N, K))
        assert set(taken) == set(TILES), set(TILES) - set(taken)
        for t, c in taken.items():
            assert any(M % tokens(t) and N % outputs(t) for M, N, K in c), (t, c)
            assert any(K % 128 for M, N, K in c), (t, c)
    for M, N, K, _ in DEEP:
        assert K >= 128 * 16, (M, N, K)
    taken = [{plan(M, N, K).tile for K in STAGE_K} for M, N in STAGES]
    assert all(len(t) == 1 for t in taken) and set().union(*taken) == set(TILES)
