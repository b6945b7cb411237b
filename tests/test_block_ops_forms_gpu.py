"""Every form of the 8-bit product: single CTAs by token tile, clusters that
share the k-blocks, pairs of CTAs, each with channels and tokens that end
inside a tile.  Tolerances are test_block_ops_gpu's."""
import pytest
import torch

import ppdl
from test_block_ops_gpu import LIN_SHAPES, TYPES, close, gen, lin_want, normal, q_want

TOKENS = {16: (0.27, 0.1), 32: (0.30, 0.28), 64: (0.31, 0.34), 128: (0.355, 1.03), 256: (0.42, 2.9)}


def cdiv(a, b):
    return -(-a // b)


def form(M, K, N, sms=148):
    """The kind and token tile that the library's model of the times chooses
    on a B200's 148 SMs."""
    kblocks, least, best = cdiv(K, 128), 1e30, None
    for tokens, (step, tail) in TOKENS.items():
        tiles, load = cdiv(N, 128) * cdiv(M, tokens), (128 + tokens) * 128 / 9e6
        for splits in (1, 2, 4, 8):
            if splits > 1 and (tokens > 64 or splits > kblocks):
                break
            room, ctas = (2 if splits > 1 else 1) * sms, tiles * splits
            t = 2.9 + (1.2 + 0.15 * splits if splits > 1 else 0) + cdiv(ctas, room) * (
                cdiv(kblocks, splits) * max(step, min(ctas, room) * load) + tail)
            if t < least:
                least, best = t, ("split" if splits > 1 else "whole", tokens)
    if best == ("whole", 256) and kblocks >= 8 and cdiv(N, 256) * cdiv(M, 256) > sms // 2:
        return "pair", 256
    return best


# the last pair of tiles holds 1 and 76 channels, or 220 (92 of them the second CTA's)
PAIRS = [(2570, 1024, 1537), (4001, 1111, 1100), (5003, 1300, 1500)]
SPLITS = [(20, 4096, 4097), (100, 4096, 641), (33, 2000, 4097)]


def test_every_form_is_reached():
    assert {form(*s) for s in PAIRS} == {("pair", 256)}
    assert {form(*s) for s in SPLITS} == {("split", 32), ("split", 64)}
    assert {form(*s) for s in list(LIN_SHAPES) + PAIRS + SPLITS} == {("pair", 256)} | {
        ("split", t) for t in (16, 32, 64)} | {("whole", t) for t in TOKENS}


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", PAIRS + SPLITS)
def test_linear_i8(cuda, M, K, N, t):
    T = TYPES[t]
    g = gen(M + 31 * K + 17 * N)
    x, w = normal(g, M, K, t=T), normal(g, N, K, scale=K ** -0.5)
    wq, ws = ppdl.quantize_rows(w)
    xq, xs = q_want(x)
    bias, res = normal(g, N), normal(g, M, N, t=T)
    for act, b, r in (("none", None, None), ("relu", bias, None), ("silu", bias, res), ("gelu", None, res)):
        y = ppdl.linear_i8(x, wq, ws, bias=b, act=act, residual=r)
        want, tol = lin_want(xq, xs, wq, ws, b, act, r, T)
        close(y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", PAIRS + SPLITS)
def test_whole_numbers(cuda, M, K, N):
    """Scales of one: the integer sums themselves, over all 8-bit values; no
    row behind the last is written."""
    g = gen(M + N)
    pad = cdiv(K, 16) * 16 + 16
    q = torch.randint(-128, 128, (M, pad), generator=g).to(torch.int8).cuda()
    w = torch.randint(-128, 128, (N, pad), generator=g).to(torch.int8).cuda()
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    out = torch.full((M + 2, N + 3), 5.0, device="cuda")
    ppdl.check(ppdl.lib().ppdl_linear_i8(
        q.data_ptr(), pad, one_m.data_ptr(), w.data_ptr(), pad, one_n.data_ptr(), None, None, 0, 0, 0, M, N,
        K, out[1:, 2:].data_ptr(), N + 3, torch.cuda.current_stream().cuda_stream))
    want = q[:, :K].double() @ w[:, :K].double().t()
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(out[1:-1, 2:-1].double(), want)
    assert (out[0] == 5).all() and (out[-1] == 5).all() and (out[:, :2] == 5).all() and (out[:, -1] == 5).all()


@pytest.mark.gpu
def test_pairs_among_small_kernels(cuda):
    """Pairs of CTAs with short kernels right behind them, whose blocks take
    the pair's SMs as soon as they are free: the same as with a pause after
    every call."""
    M, K, N = PAIRS[0]
    g = gen(6)
    x, few, w = normal(g, M, K, t=torch.bfloat16), normal(g, 30, K, t=torch.bfloat16), normal(g, N, K)
    wq, ws = ppdl.quantize_rows(w)

    def chain(pause):
        out = []
        for _ in range(4):
            out.append(ppdl.linear_i8(x, wq, ws))
            pause()
            out.append(ppdl.linear_i8(few, wq, ws))
            pause()
            out.append(ppdl.layernorm(out[-1]))
            pause()
        return out

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))
    torch.cuda.synchronize()
    assert ppdl.lib().ppdl_op_device_error() == 0
