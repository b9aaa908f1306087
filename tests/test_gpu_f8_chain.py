"""The 8-bit linear path as it is used together, on the GPU: weights quantised
at load (from the linear layers' own block formats too), a pre-norm
feed-forward block from the residual stream to its update, captured and
replayed, and on several streams."""
import numpy as np
import pytest
import torch

import kd_f8
import kd_mm
import kd_oracle_f8 as of
import kd_oracle_quant as oq
from f8_common import DEV, announce, from_rows, linear_tol

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Block:
    """norm -> up -> GELU -> down, 8-bit weights; stream += the block."""

    def __init__(self, D, F, seed):
        g = torch.Generator().manual_seed(seed)
        self.norm = (1 + 0.2 * torch.randn(D, generator=g)).to(DEV)
        self.up = kd_f8.quantize((torch.randn((F, D), generator=g) * D ** -0.5).to(BF16).to(DEV))
        self.down = kd_f8.quantize((torch.randn((D, F), generator=g) * F ** -0.5).to(BF16).to(DEV))
        self.bias = (torch.randn(F, generator=g) * 0.1).to(DEV)

    def __call__(self, branch, stream):
        """(the block's output, the new residual stream)."""
        h, stream = kd_f8.add_rms_norm(branch, self.norm, stream)
        inner = torch.nn.functional.gelu(kd_f8.linear(h, self.up, self.bias).float())
        return kd_f8.linear(kd_f8.quantize(inner), self.down), stream


@pytest.mark.parametrize("M", [1, 16, 77, 600])
def test_block_step_by_step(M):
    """Every step of the chain against the oracle on that step's own inputs."""
    _need_gpu()
    announce(f"chain {M}")
    D, F = 400, 1040
    blk = Block(D, F, 1)
    g = torch.Generator().manual_seed(M)
    branch = torch.randn((M, D), generator=g).to(BF16).to(DEV)
    stream = (4 * torch.randn((M, D), generator=g)).to(DEV)
    h, total = kd_f8.add_rms_norm(branch, blk.norm, stream)
    assert torch.equal(total, branch.float() + stream)
    y = of.rms_norm(total.cpu().double().numpy(), blk.norm.cpu().numpy(), 1e-6)
    hv = of.decode(*from_rows(h))
    scale = np.repeat(2.0 ** (from_rows(h)[1].astype(np.float64) - 127), 128, axis=1)[:, :D]
    assert np.all(np.abs(hv - y) <= np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * scale) * (1 + 1e-4))
    u = kd_f8.linear(h, blk.up, blk.bias)
    wv = of.decode(*from_rows(blk.up))
    ref = of.linear(hv, wv, blk.bias.cpu().numpy())
    assert np.all(np.abs(u.cpu().double().numpy() - ref) <= linear_tol(hv, wv, ref))
    inner = torch.nn.functional.gelu(u.float())
    q = kd_f8.quantize(inner)
    c, s = of.quantize(inner.cpu().numpy())
    assert np.array_equal(from_rows(q)[0], c) and np.array_equal(from_rows(q)[1], s)
    got, again = blk(branch, stream)
    qv, wv = of.decode(c, s), of.decode(*from_rows(blk.down))
    ref = of.linear(qv, wv)
    assert np.all(np.abs(got.cpu().double().numpy() - ref) <= linear_tol(qv, wv, ref))
    assert torch.equal(again, total)


def test_block_weights_of_the_linear_layers():
    """A Q8_0 weight through kd_mm.dequant into 8 bits; the product near the
    16-bit one: operands are off by a sixteenth at most each."""
    _need_gpu()
    announce("chain q8_0 weight")
    M, N, K = 50, 128, 512
    rng = np.random.default_rng(2)
    blocks = oq.quantize_q8_0((rng.standard_normal((N, K)) * 0.05).astype(np.float32))
    w = kd_mm.QuantWeight(torch.from_numpy(blocks).to(DEV), kd_mm.TYPE_Q8_0, K)
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(DEV)
    full = kd_mm.linear(x, w).double()
    got = kd_f8.linear(kd_f8.quantize(x), kd_f8.quantize(kd_mm.dequant(w))).double()
    wide = kd_mm.dequant(w).double().abs()
    bound = (1.0625 ** 2 - 1 + 2.0 ** -8) * (x.double().abs() @ wide.t()) + 2.0 ** -7 * full.abs()
    assert bool(((got - full).abs() <= bound).all())


def test_captured_block_replays():
    _need_gpu()
    announce("chain graph")
    blk = Block(512, 1024, 3)
    g = torch.Generator().manual_seed(4)
    branch = torch.randn((40, 512), generator=g).to(BF16).to(DEV)
    stream = torch.randn((40, 512), generator=g).to(DEV)
    blk(branch, stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, new = blk(branch, stream)
    for i in range(4):
        branch.copy_(torch.randn((40, 512), generator=g).to(BF16))
        stream.copy_(torch.randn((40, 512), generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, total = blk(branch, stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(new, total), i


def test_two_streams_at_once():
    """No call shares state with another: several in flight equal one by one."""
    _need_gpu()
    announce("chain streams")
    blk = Block(512, 2048, 5)
    g = torch.Generator().manual_seed(6)
    ins = [(torch.randn((m, 512), generator=g).to(BF16).to(DEV), torch.randn((m, 512), generator=g).to(DEV)) for m in (3, 700, 64, 1)]
    want = [blk(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for s, i in zip(streams, ins):
        with torch.cuda.stream(s):
            got.append(blk(*i))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_an_explicit_stream_is_used():
    """A call on a stream that another holds up does not run ahead of it."""
    _need_gpu()
    announce("chain explicit stream")
    s = torch.cuda.Stream()
    x = torch.zeros((64, 4096), device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(50):
            x.add_(1.0)
    r = kd_f8.quantize(x, stream=s)
    torch.cuda.synchronize()
    want, _ = of.quantize(np.full((1, 128), 50.0, dtype=np.float32))
    assert np.all(from_rows(r)[0] == want[0, 0])


def test_outputs_of_an_explicit_stream_are_its_own():
    """What the current stream still writes to, and has given back, is not
    handed to a call on another stream."""
    _need_gpu()
    announce("chain explicit stream's outputs")
    s = torch.cuda.Stream()
    x = torch.full((4096, 4096), 50.0, device=DEV)
    w = kd_f8.quantize(torch.eye(4096, device=DEV))
    codes, scales = from_rows(kd_f8.quantize(x))
    torch.cuda.synchronize()

    def busy(shape, dtype):
        old = torch.empty(shape, dtype=dtype, device=DEV)
        for _ in range(200):
            old.fill_(7)

    busy((4096, 4096), torch.uint8)
    r = kd_f8.quantize(x, stream=s)
    torch.cuda.synchronize()
    assert np.array_equal(from_rows(r)[0], codes) and np.array_equal(from_rows(r)[1], scales)
    busy((4096, 4096), torch.bfloat16)
    y = kd_f8.linear(r, w, stream=s)
    torch.cuda.synchronize()
    # 50 lies halfway between two codes: blocks of 50s get the scale 2^-3, 400
    # = 1.5625 * 2^8 goes to 1.5 * 2^8 (of 1.5 and 1.625 the even one)
    assert bool((y == 48.0).all())
    busy((4096, 4096), torch.float32)
    _, total = kd_f8.add_rms_norm(x, torch.ones(4096, device=DEV), x, stream=s)
    torch.cuda.synchronize()
    assert bool((total == 100.0).all())


def test_last_token_of_each_sequence():
    """Rows of a slice, one of each sequence, through every operator."""
    _need_gpu()
    announce("chain last tokens")
    B, L, D = 5, 9, 512
    blk = Block(D, 1024, 7)
    g = torch.Generator().manual_seed(8)
    branch = torch.randn((B, L, D), generator=g).to(BF16).to(DEV)
    stream = torch.randn((B, L, D), generator=g).to(DEV)
    got, total = blk(branch[:, -1:], stream[:, -1:])
    want, same = blk(branch[:, -1].contiguous(), stream[:, -1].contiguous())
    torch.cuda.synchronize()
    assert got.shape == (B, 1, D) and torch.equal(got[:, 0], want) and torch.equal(total[:, 0], same)
    whole, _ = kd_f8.add_rms_norm(branch, blk.norm, stream)
    part = kd_f8.Rows(whole.codes[:, -1:], whole.scales[:, -1:])
    assert torch.equal(kd_f8.linear(part, blk.up)[:, 0], kd_f8.linear(kd_f8.add_rms_norm(branch[:, -1].contiguous(), blk.norm,
                                                                                         stream[:, -1].contiguous())[0], blk.up))
