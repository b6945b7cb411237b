"""The transformer-block operators against their definitions in 64 bits:
layer norm (forward, backward), 8-bit quantiser and linear layer, rotary
positions; then all of them in a row around the attention core.

Tolerances count roundings.  u = 2^-24 is half a step of FP32; half(t) that
of the result's type, relative to the result.  A sum of n terms added one
after another is off by at most n u times the sum of their magnitudes; the
kernels add at most D / 32 + 16 terms in a row along a row of D (at least 32
lanes take every row wider than 64), and at most rows / 128 + 320 down a
column.
"""
import ctypes as C

import pytest
import torch

import ppdl

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol):
    """|got - want| <= tol everywhere (tol: a tensor); want in 64 bits."""
    assert got.shape == want.shape
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got.double() - want).abs() / tol).max()):.3g} times the bound")


def normal(g, *shape, t=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(t).cuda()


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- layer norm ----------------------------------------------------------------------------------

def ln_want(x, w, b, eps, residual=None):
    s = x.double() if residual is None else (x.double() + residual.double()).to(x.dtype).double()
    D = x.shape[-1]
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    w = torch.ones(D, device=x.device) if w is None else w
    b = torch.zeros(D, device=x.device) if b is None else b
    xh = (s - mean) * rstd
    y = xh * w.double() + b.double()
    k = D / 32 + 16
    dmean = U * (k + 1) * s.abs().mean(-1, keepdim=True)          # of the mean
    # of rstd, relative: half that of variance + eps (its sum, and the mean's own error squared)
    drstd = U * (k + 4) + 0.5 * (dmean * rstd) ** 2
    tol = half(x.dtype) * y.abs() + U * y.abs() + (dmean * rstd + U * s.abs() * rstd) * w.double().abs() \
        + (drstd + 4 * U) * (xh * w.double()).abs() + U * b.double().abs()
    # FP16's smallest numbers: half a step of the subnormals
    tol = tol + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)
    return y, s, mean[..., 0], rstd[..., 0], tol, dmean[..., 0], (drstd * rstd + 1e-30)[..., 0]


SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (7, 31), (4, 32), (9, 33), (2, 64), (6, 65), (33, 100),
          (300, 256), (17, 257), (3, 512), (5, 640), (4, 1000), (2, 1024), (3, 1025), (13, 1153),
          (2, 2048), (5, 2500), (2, 4096), (3, 4097), (2, 5000), (1, 8192), (2, 8200), (1, 12289),
          (2, 16384), (1, 16385), (2, 20000), (1, 32768), (1, 40001)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,D", SHAPES)
def test_layernorm(cuda, rows, D, t):
    T = TYPES[t]
    g = gen(rows * 131 + D)
    x, r = normal(g, rows, D, t=T, scale=2.0, shift=0.7), normal(g, rows, D, t=T)
    for wt in {T, torch.float32}:
        w, b = normal(g, D, t=wt, shift=1.0, scale=0.3), normal(g, D, t=wt, scale=0.3)
        y, mean, rstd = ppdl.layernorm(x, w, b, 1e-5, return_stats=True)
        want = ln_want(x, w, b, 1e-5)
        close(y, want[0], want[4])
        close(mean, want[2], want[5] + U * want[2].abs())
        close(rstd, want[3], want[6] + U * want[3])
        y, s = ppdl.layernorm(x, w, b, 1e-5, residual=r, return_sum=True)
        want = ln_want(x, w, b, 1e-5, r)
        assert torch.equal(s.double(), want[1])
        close(y, want[0], want[4])
        assert torch.equal(ppdl.layernorm(x, w, b, 1e-5, residual=r), y)
    y = ppdl.layernorm(x)
    want = ln_want(x, None, None, 1e-5)
    close(y, want[0], want[4])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,ld,off", [(256, 264, 0), (256, 257, 0), (256, 512, 3), (100, 104, 4),
                                      (2048, 2051, 1), (4096, 8192, 8), (1000, 1008, 8)])
def test_layernorm_strided_rows(cuda, D, ld, off, t):
    """Rows inside wider rows, at any alignment; what lies between is left alone."""
    T = TYPES[t]
    g = gen(D + ld)
    wide = normal(g, 5, ld + off, t=T)
    x = wide[:, off:off + D]
    w, b = normal(g, D + 1, t=T, shift=1.0)[1:], normal(g, D, t=T)
    want = ln_want(x, w, b, 1e-5)
    close(ppdl.layernorm(x, w, b), want[0], want[4])
    # output rows with a stride of their own, through the C ABI
    out = torch.full((5, ld + off), 7.0, device="cuda", dtype=T)
    code = {"f32": 0, "bf16": 1, "f16": 2}[t]
    st = ppdl.lib().ppdl_layernorm(x.data_ptr(), ld + off, None, 0, w.data_ptr(), b.data_ptr(), code,
                                   code, 5, D, 1e-5, out[:, off:].data_ptr(), ld + off, None, 0, None,
                                   None, torch.cuda.current_stream().cuda_stream)
    ppdl.check(st)
    close(out[:, off:off + D], want[0], want[4])
    assert (out[:, :off] == 7).all() and (out[:, off + D:] == 7).all()


@pytest.mark.parametrize("D", [32, 256, 1000, 4096, 33000])
def test_layernorm_in_place(cuda, D):
    g = gen(D)
    x, r = normal(g, 6, D), normal(g, 6, D)
    w, b = normal(g, D), normal(g, D)
    y, s = ppdl.layernorm(x, w, b, residual=r, return_sum=True)
    st = ppdl.lib().ppdl_layernorm(x.data_ptr(), D, r.data_ptr(), D, w.data_ptr(), b.data_ptr(), 0, 0,
                                   6, D, 1e-5, x.data_ptr(), D, r.data_ptr(), D, None, None,
                                   torch.cuda.current_stream().cuda_stream)
    ppdl.check(st)
    assert torch.equal(x, y) and torch.equal(r, s)


def test_layernorm_hard_rows(cuda):
    """A constant row, a huge common offset, and rows with an infinity or a NaN
    (which spoil their own row only)."""
    g = gen(3)
    for D in (256, 1001, 4096):
        x = normal(g, 6, D)
        x[1] = 3.25
        x[2] += 30000.0
        x[3, 5] = float("inf")
        x[4, D - 1] = float("nan")
        w, b = normal(g, D), normal(g, D)
        y = ppdl.layernorm(x, w, b)
        want = ln_want(x, w, b, 1e-5)
        ok = [0, 1, 2, 5]
        close(y[ok], want[0][ok], want[4][ok])
        assert y[3].isnan().all() and y[4].isnan().all()


def bwd_want(dy, x, w, mean, rstd, dsum=None):
    dy, xx, D = dy.double(), x.double(), x.shape[-1]
    m, r = mean.double().unsqueeze(-1), rstd.double().unsqueeze(-1)
    xh = (xx - m) * r
    ww = torch.ones(D, device=x.device).double() if w is None else w.double()
    gg = dy * ww
    m1, m2 = gg.mean(-1, keepdim=True), (gg * xh).mean(-1, keepdim=True)
    dx = r * (gg - m1 - xh * m2)
    k = D / 32 + 24
    dxh = 2 * U * xh.abs() + U * (xx.abs() + m.abs()) * r           # of xh, once rounded
    size = gg.abs() + gg.abs().mean(-1, keepdim=True) + xh.abs() * (gg * xh).abs().mean(-1, keepdim=True)
    tol = r * (k * U * size + dxh * m2.abs() + xh.abs() * (gg.abs() * dxh).mean(-1, keepdim=True))
    if dsum is not None:
        dx = dx + dsum.double()
        tol = tol + U * dsum.double().abs()
    tol = tol + (half(x.dtype) + U) * dx.abs() + (2.0 ** -24 if x.dtype == torch.float16 else 1e-38)
    flat = lambda v: v.reshape(-1, D)  # noqa: E731
    kr = flat(xx).shape[0] / 128 + 320
    dw, db = flat(dy * xh).sum(0), flat(dy).sum(0)
    wt = x.dtype if w is None else w.dtype
    tiny = 2.0 ** -24 if wt == torch.float16 else 1e-38
    tw = kr * U * flat(dy * xh).abs().sum(0) + flat(dy.abs() * dxh).sum(0) + (half(wt) + U) * dw.abs() + tiny
    tb = kr * U * flat(dy).abs().sum(0) + (half(wt) + U) * db.abs() + tiny
    return (dx, dw, db), (tol, tw, tb)


BWD_SHAPES = [(1, 1), (4, 2), (1, 31), (7, 33), (300, 256), (2400, 256), (1000, 257), (5, 64),
              (129, 100), (64, 512), (40, 1024), (99, 1153), (700, 1000), (31, 2048), (300, 4096),
              (9, 4099), (17, 8192), (5, 8193), (6, 12000), (3, 16384), (2, 40001), (3000, 24)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,D", BWD_SHAPES)
def test_layernorm_backward(cuda, rows, D, t):
    T = TYPES[t]
    g = gen(rows * 7 + D)
    x = normal(g, rows, D, t=T, scale=2.0, shift=0.7)
    dy, ds = normal(g, rows, D, t=T), normal(g, rows, D, t=T)
    for wt in {T, torch.float32}:
        w = normal(g, D, t=wt, shift=1.0, scale=0.3)
        _, mean, rstd = ppdl.layernorm(x, w, None, return_stats=True)
        for dsum in (None, ds):
            got = ppdl.layernorm_backward(dy, x, w, mean, rstd, dsum=dsum)
            want, tol = bwd_want(dy, x, w, mean, rstd, dsum)
            for a, b, c in zip(got, want, tol):
                close(a, b, c)
            assert got[1].dtype == got[2].dtype == wt
        # the same call gives the same bits; without the weights' gradients dx is unchanged
        again = ppdl.layernorm_backward(dy, x, w, mean, rstd, dsum=dsum)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        alone = ppdl.layernorm_backward(dy, x, w, mean, rstd, dsum=dsum, param_grads=False)
        assert torch.equal(alone[0], got[0]) and alone[1] is None and alone[2] is None
    got = ppdl.layernorm_backward(dy, x, None, mean, rstd)
    want, tol = bwd_want(dy, x, None, mean, rstd)
    for a, b, c in zip(got, want, tol):
        close(a, b, c)


@pytest.mark.parametrize("D", [256, 1000, 4096])
def test_layernorm_backward_strided(cuda, D):
    g = gen(D)
    for ld, off in ((D + 8, 0), (D + 1, 1), (2 * D, 4)):
        x = normal(g, 37, ld + off, t=torch.bfloat16)[:, off:off + D]
        dy = normal(g, 37, ld + 3, t=torch.bfloat16)[:, :D]
        w = normal(g, D)
        _, mean, rstd = ppdl.layernorm(x, w, None, return_stats=True)
        got = ppdl.layernorm_backward(dy, x, w, mean, rstd)
        want, tol = bwd_want(dy, x, w, mean, rstd)
        for a, b, c in zip(got, want, tol):
            close(a, b, c)


DENSE = [(148, 1), (153, 3), (161, 33), (2501, 79), (149, 257), (1000, 322), (5, 1153), (64001, 79),
         (35003, 129), (17001, 257), (13101, 322), (8195, 513), (6601, 641), (4098, 1027), (3651, 1153),
         (3303, 1281), (2051, 2049), (1661, 2561), (1027, 4095), (1031, 4097), (50001, 100)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,D", DENSE)
def test_layernorm_dense_odd_rows(cuda, rows, D, t):
    """Dense rows that are no whole vectors, the last ones of which end inside
    one: both directions, results over inputs, and nothing behind the last row."""
    T = TYPES[t]
    g = gen(rows + D)

    def guarded(v):
        room = torch.full((rows * D + 64,), 7.0, device="cuda", dtype=T)
        room[:rows * D] = v.reshape(-1)
        return room, room[:rows * D].view(rows, D)

    (xr, x), (rr, r) = guarded(normal(g, rows, D, t=T, scale=2.0, shift=0.7)), guarded(normal(g, rows, D, t=T))
    w, b = normal(g, D, t=T, shift=1.0, scale=0.3), normal(g, D, t=T, scale=0.3)
    want = ln_want(x, w, b, 1e-5, r)
    y, s, mean, rstd = ppdl.layernorm(x, w, b, 1e-5, residual=r, return_sum=True, return_stats=True)
    close(y, want[0], want[4])
    assert torch.equal(s.double(), want[1])
    close(mean, want[2], want[5] + U * want[2].abs())
    close(rstd, want[3], want[6] + U * want[3])
    plain, bare = ppdl.layernorm(x, w, b, 1e-5), ln_want(x, w, b, 1e-5)
    close(plain, bare[0], bare[4])
    code, stream = {"f32": 0, "bf16": 1, "f16": 2}[t], torch.cuda.current_stream().cuda_stream
    dy, (outr, out) = normal(g, rows, D, t=T), guarded(torch.zeros(rows, D))
    dx, dw, db = ppdl.layernorm_backward(dy, s, w, mean, rstd, dsum=r)
    wants, tol = bwd_want(dy, s, w, mean, rstd, r)
    for got, a, c in zip((dx, dw, db), wants, tol):
        close(got, a, c)
    ppdl.check(ppdl.lib().ppdl_layernorm_backward(
        dy.data_ptr(), D, s.data_ptr(), D, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), r.data_ptr(), D,
        code, code, rows, D, out.data_ptr(), D, None, None, None, stream))
    assert torch.equal(out, dx) and (outr[rows * D:] == 7).all()
    ppdl.check(ppdl.lib().ppdl_layernorm(
        x.data_ptr(), D, r.data_ptr(), D, w.data_ptr(), b.data_ptr(), code, code, rows, D, 1e-5,
        x.data_ptr(), D, r.data_ptr(), D, None, None, stream))
    assert torch.equal(x, y) and torch.equal(r, s)
    assert (xr[rows * D:] == 7).all() and (rr[rows * D:] == 7).all()


@pytest.mark.parametrize("rows,D", [(8195, 513), (3651, 1153), (16384, 1024), (1200, 8192)])
def test_layernorm_chain(cuda, rows, D):
    """Kernels that start before the ones they follow have ended wait for all
    that those store, by bulk copies too: a chain gives what it gives with a
    pause after every call, eagerly and in a graph."""
    g = gen(rows + D)
    T = torch.bfloat16
    x, dy, w = normal(g, rows, D, t=T), normal(g, rows, D, t=T), normal(g, D, t=T, shift=1.0, scale=0.2)

    def chain(pause):
        out = [x]
        for _ in range(3):
            y, s, mean, rstd = ppdl.layernorm(out[-1], w, None, residual=dy, return_sum=True, return_stats=True)
            pause()
            dx, dw, db = ppdl.layernorm_backward(dy, s, w, mean, rstd, dsum=y)
            pause()
            q, scale = ppdl.quantize_rows(dx)
            pause()
            out += [y, s, dw, db, scale, q.contiguous(), dx]
        return out

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layernorm_backward_no_rows(cuda):
    """No rows: the weights' gradients are zeros, not what the memory held."""
    x, s = torch.empty((0, 300), device="cuda"), torch.empty(0, device="cuda")
    dx, dw, db = ppdl.layernorm_backward(x, x, torch.ones(300, device="cuda"), s, s)
    assert dx.shape == (0, 300) and (dw == 0).all() and (db == 0).all()
    assert ppdl.layernorm(x).shape == (0, 300)


def test_layernorm_gradients_by_differences(cuda):
    """The kernels' own difference quotient along a direction against their
    gradient; the same quotient in 64 bits says how far a quotient at this
    step is from the derivative."""
    g = gen(11)
    x, r, dy = (normal(g, 64, 384) for _ in range(3))
    w, b = normal(g, 384, shift=1.0, scale=0.3), normal(g, 384)
    vx, vw, vb = normal(g, 64, 384), normal(g, 384), normal(g, 384)
    y, s, mean, rstd = ppdl.layernorm(x, w, b, residual=r, return_sum=True, return_stats=True)
    dx, dw, db = ppdl.layernorm_backward(dy, s, w, mean, rstd)
    h = 2.0 ** -7

    def quotient(f):
        a = f(x + h * vx, w + h * vw, b + h * vb)
        c = f(x - h * vx, w - h * vw, b - h * vb)
        return float(((a.double() - c.double()) * dy.double()).sum()) / (2 * h)

    ours = quotient(lambda *p: ppdl.layernorm(*p, residual=r))
    true = quotient(lambda *p: ln_want(*p, 1e-5, r)[0])
    grad = float((dx.double() * vx.double()).sum() + (dw.double() * vw.double()).sum()
                 + (db.double() * vb.double()).sum())
    want, tol = bwd_want(dy, s, w, mean, rstd)
    exact = float((want[0] * vx.double()).sum() + (want[1] * vw.double()).sum()
                  + (want[2] * vb.double()).sum())
    noise = float((ln_want(x, w, b, 1e-5, r)[4] * dy.double().abs()).sum()) / h
    slack = sum(float((t * v.double().abs()).sum()) for t, v in zip(tol, (vx, vw, vb)))
    assert abs(ours - grad) <= 2 * noise + slack + abs(true - exact)


# ---- 8-bit linear layers -------------------------------------------------------------------------

def q_want(x):
    x = x.double()
    amax = x.abs().amax(-1)
    scale = (amax / 127).float()
    s = scale.double().unsqueeze(-1)
    q = torch.where((s > 0) & s.isfinite(), torch.round(x / s), torch.zeros_like(x))
    return q.nan_to_num(0.0).clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 5), (2, 16), (7, 100), (300, 256), (5, 1000), (4, 1111),
                                    (2, 4096), (3, 8191), (1, 20000), (1, 70001)])
def test_quantize_rows(cuda, rows, K, t):
    """Whole numbers: equal to the definition's, bit for bit, the scale too."""
    T = TYPES[t]
    for x in (normal(gen(rows + K), rows, K, t=T, scale=3.0),
              normal(gen(rows + K), rows, K + 3, t=T, scale=1e-3)[:, 3:]):
        q, s = ppdl.quantize_rows(x)
        wq, ws = q_want(x)
        assert q.shape == x.shape and q.stride(-2) % 16 == 0
        assert torch.equal(s, ws) and torch.equal(q, wq)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,K", [(16001, 67), (12001, 99), (8201, 131), (4099, 257), (3301, 322),
                                    (2101, 513), (1003, 1153), (901, 1281), (521, 2049), (271, 4095),
                                    (301, 4097)])
def test_quantize_dense_odd_rows(cuda, rows, K, t):
    """Dense rows that are no whole vectors, among them zeros, an infinity and
    a NaN; nothing is written past a row's K values."""
    g = gen(rows + K)
    x = normal(g, rows, K, t=TYPES[t], scale=3.0)
    x[1], x[rows - 2, K - 1], x[rows // 2, 0] = 0, float("inf"), float("nan")
    ldq = (K + 31) // 16 * 16
    q = torch.full((rows, ldq), 55, device="cuda", dtype=torch.int8)
    scale = torch.empty(rows, device="cuda")
    ppdl.check(ppdl.lib().ppdl_quantize_rows_i8(
        x.data_ptr(), K, {"f32": 0, "bf16": 1, "f16": 2}[t], rows, K, q.data_ptr(), ldq,
        scale.data_ptr(), torch.cuda.current_stream().cuda_stream))
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[rows - 2, rows // 2]] = True
    want, ws = q_want(x[~bad])
    assert torch.equal(q[~bad][:, :K], want) and torch.equal(scale[~bad], ws)
    assert (q[bad][:, :K] == 0).all() and not scale[bad].isfinite().any()
    assert (q[:, K:] == 55).all()


def test_quantize_ties_and_extremes(cuda):
    """Ties on exact halves go to the even neighbour; quotients next to a half
    fall on their own side; tiny, zero, infinite and NaN rows."""
    n = torch.arange(-126, 127, device="cuda").float()
    x = torch.zeros(12, 1024, device="cuda")
    x[:, 0] = 127.0
    x[0, 1:254] = n + 0.5
    x[1] = x[0] * 0.37                      # scale no power of two
    x[2] = torch.nextafter(x[0], x[0] * 2)
    x[2, 0] = 127.0
    x[3] = torch.nextafter(x[0], x[0] * 0)
    x[3, 0] = 127.0
    s = torch.tensor(1.1, device="cuda")
    x[4, 1:254] = (n + 0.5) * s
    x[4, 0] = 127.0 * s
    x[5] = x[0] * 2.0 ** -120
    x[6] = x[0] * 2.0 ** -140               # subnormal scale
    x[7] = 0.0
    x[8, :3] = torch.tensor([2.0 ** -149, -(2.0 ** -149), 2.0 ** -148], device="cuda")
    x[8, 3:] = 0.0
    x[9, 7] = float("inf")
    x[10, 9] = float("nan")
    x[11] = x[0] * 2.0 ** 120
    q, sc = ppdl.quantize_rows(x)
    wq, ws = q_want(x)
    assert torch.equal(sc[:10], ws[:10]) and sc[10].isnan() and torch.equal(sc[11:], ws[11:])
    assert torch.equal(q, wq)
    assert (q[7:] [:3] == wq[7:][:3]).all() and (q[9] == 0).all() and (q[10] == 0).all()


def act_want(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    return v


def lin_want(q, qs, w, ws, bias, act, residual, T):
    """The definition on the 8-bit values and its tolerance: the integer sum
    rounded to FP32, two scales, the bias' sum, an activation whose slope is
    at most 1.13 and whose own evaluation in FP32 is good to 16 u, the
    residual's sum, the result's rounding."""
    acc = q.double() @ w.double().t()
    v = acc * qs.double()[:, None] * ws.double()
    tol = 4 * U * v.abs()
    if bias is not None:
        v = v + bias.double()
        tol = tol + U * bias.double().abs()
    y = act_want(v, act)
    tol = 1.13 * (tol + U * v.abs()) + 16 * U * v.abs() * (act != "none")
    if residual is not None:
        y = y + residual.double()
        tol = tol + U * y.abs()
    return y, tol + (half(T) + U) * y.abs() + (2.0 ** -25 if T == torch.float16 else 1e-38)


LIN_SHAPES = [(16, 4096, 300), (5, 2047, 260), (1, 65000, 33), (7, 8192, 129), (1, 2048, 40000), (1, 1, 1), (1, 16, 7), (2, 17, 3), (1, 4096, 512), (1, 1000, 333), (3, 300, 129),
              (8, 2048, 256), (16, 512, 1000), (17, 515, 130), (33, 64, 64), (64, 128, 200),
              (100, 256, 300), (128, 128, 128), (129, 130, 257), (300, 256, 1024), (300, 2048, 256),
              (511, 1111, 127), (1000, 96, 2047), (2400, 256, 256), (777, 1111, 513), (5000, 40, 40),
              (1, 33000, 40), (2049, 513, 1025), (5003, 200, 2100), (3001, 70, 3333), (19000, 130, 256)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", LIN_SHAPES)
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
        # quantised before the call: the same bits
        q, s = ppdl.quantize_rows(x)
        assert torch.equal(ppdl.linear_i8(q, wq, ws, x_scale=s, bias=b, act=act, residual=r, out_dtype=T), y)


@pytest.mark.parametrize("M,K,N", [(1, 64, 20), (5, 1024, 300), (70, 127, 129), (300, 500, 260),
                                   (1500, 256, 384)])
def test_linear_i8_whole_numbers(cuda, M, K, N):
    """Scales of one: the integer sums themselves, over all 8-bit values (-128
    among them); what lies past K in the rows is not read as data."""
    g = gen(M + N)
    pad = (K + 15) // 16 * 16 + 32
    q = torch.randint(-128, 128, (M, pad), generator=g).to(torch.int8).cuda()
    w = torch.randint(-128, 128, (N, pad), generator=g).to(torch.int8).cuda()
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    y = ppdl.linear_i8(q[:, :K], w[:, :K], one_n, x_scale=one_m)
    want = q[:, :K].double() @ w[:, :K].double().t()
    assert float(want.abs().max()) < 2 ** 24 and torch.equal(y.double(), want)
    q.fill_(-128), w.fill_(-128)
    y = ppdl.linear_i8(q[:, :K], w[:, :K], one_n, x_scale=one_m)
    assert (y == K * 16384).all()


def test_linear_i8_longest_sum(cuda):
    K = 131071
    q = torch.full((2, 131072), -128, dtype=torch.int8, device="cuda")
    y = ppdl.linear_i8(q[:, :K], q[:, :K], torch.ones(2, device="cuda"), x_scale=torch.ones(2, device="cuda"))
    assert (y.double() == torch.tensor(float(K * 16384)).float().double()).all()


def test_linear_i8_strides_and_rows_left_alone(cuda):
    """Output and residual rows with strides of their own, at odd offsets."""
    g = gen(5)
    for M, K, N, T, code in ((37, 100, 45, torch.bfloat16, 1), (200, 64, 130, torch.float32, 0),
                             (3, 512, 96, torch.float16, 2)):
        x, w = normal(g, M, K), normal(g, N, K)
        q, s = ppdl.quantize_rows(x)
        wq, ws = ppdl.quantize_rows(w)
        for ld, off in ((N + 1, 1), (N + 2, 0), (2 * N, 3)):
            res = normal(g, M, ld + off + 2, t=T)
            out = torch.full((M + 2, ld + off), 5.0, device="cuda", dtype=T)
            st = ppdl.lib().ppdl_linear_i8(
                q.data_ptr(), q.stride(0), s.data_ptr(), wq.data_ptr(), wq.stride(0), ws.data_ptr(),
                None, res[:, 2:].data_ptr(), res.stride(0), code, 2, M, N, K, out[1:, off:].data_ptr(),
                out.stride(0), torch.cuda.current_stream().cuda_stream)
            ppdl.check(st)
            want, tol = lin_want(q, s, wq, ws, None, "silu", res[:, 2:2 + N], T)
            close(out[1:-1, off:off + N], want, tol)
            assert (out[0] == 5).all() and (out[-1] == 5).all()
            assert (out[:, :off] == 5).all() and (out[:, off + N:] == 5).all()


def test_linear_i8_bad_rows_stay_their_own(cuda):
    """A token with a NaN or an infinity spoils its own output row only."""
    g = gen(8)
    x, w = normal(g, 40, 256), normal(g, 96, 256)
    wq, ws = ppdl.quantize_rows(w)
    clean = ppdl.linear_i8(x, wq, ws)
    x[3, 200], x[17, 0] = float("nan"), float("inf")
    y = ppdl.linear_i8(x, wq, ws)
    keep = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(y[keep], clean[keep]) and y[3].isnan().all() and y[17].isnan().all()


@pytest.mark.parametrize("M,K", [(1, 512), (2, 300), (1, 1003), (2, 4096), (9, 300), (16, 1000)])
def test_linear_i8_few_rows(cuda, M, K):
    """Few rows in place: strided and unaligned ones, ties, and bad, zero and
    tiny rows, quantised in the product's kernel to the same bits."""
    g = gen(M + K)
    wq, ws = ppdl.quantize_rows(normal(g, 200, K))
    for T in TYPES.values():
        for x in (normal(g, M, K, t=T), normal(g, M, K + 1, t=T)[:, 1:], normal(g, M, 2 * K, t=T)[:, K:]):
            x[0, 3:40] = x.abs().max() / 2            # 63.5 steps when it is the row's largest
            if M == 2:
                x[1] = {300: 0.0, 4096: float("nan")}[K]
            if M > 8:
                x[1], x[2] = 0, x[2] * 1e-6
                x[3] = x[3] * 2.0 ** -120 if T != torch.float16 else x[3]
                x[4, K - 1], x[5, 0] = float("nan"), float("-inf")
            q, s = ppdl.quantize_rows(x)
            want = ppdl.linear_i8(q, wq, ws, x_scale=s, out_dtype=T)
            got = ppdl.linear_i8(x, wq, ws)
            assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
            if M > 8:
                assert got[4].isnan().all() and got[5].isnan().all() and (got[1] == 0).all()


def test_linear_i8_in_place_residual(cuda):
    g = gen(9)
    for M in (2, 500):
        x, w, r = normal(g, M, 128), normal(g, 70, 128), normal(g, M, 70)
        wq, ws = ppdl.quantize_rows(w)
        q, s = ppdl.quantize_rows(x)
        want = ppdl.linear_i8(x, wq, ws, residual=r)
        st = ppdl.lib().ppdl_linear_i8(q.data_ptr(), q.stride(0), s.data_ptr(), wq.data_ptr(), wq.stride(0),
                                       ws.data_ptr(), None, r.data_ptr(), 70, 0, 0, M, 70, 128,
                                       r.data_ptr(), 70, torch.cuda.current_stream().cuda_stream)
        ppdl.check(st)
        assert torch.equal(r, want)


def test_linear_i8_leading_dimensions(cuda):
    g = gen(10)
    x, w = normal(g, 2, 3, 64), normal(g, 24, 64)
    wq, ws = ppdl.quantize_rows(w)
    y = ppdl.linear_i8(x, wq, ws)
    assert y.shape == (2, 3, 24) and torch.equal(y.view(6, 24), ppdl.linear_i8(x.view(6, 64), wq, ws))
    assert ppdl.linear_i8(x[:0], wq, ws).shape == (0, 3, 24)
    with pytest.raises(RuntimeError):
        ppdl.linear_i8(x, torch.zeros(24, 72, dtype=torch.int8, device="cuda")[:, :64], ws)


# ---- rotary --------------------------------------------------------------------------------------

def rot_want(x, pos, freq, sections, interleaved, inverse):
    """The definition in 64 bits, and its tolerance: the fraction of a turn is
    rounded to FP32 and goes through a sine and cosine good to a few u (pi u of
    angle and 4 u of value), two products and their difference are rounded; the
    angle itself carries the 64-bit product's 2^-51 of its size."""
    pairs = freq.numel()
    axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], device=x.device)
    angle = pos[axis].permute(1, 2, 0).double() * freq
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None] * (-1 if inverse else 1)
    y = x.double().clone()
    idx = torch.arange(pairs, device=x.device)
    ia, ib = (2 * idx, 2 * idx + 1) if interleaved else (idx, idx + pairs)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    tol = half(x.dtype) * y.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)
    off = 10 * U + angle.abs()[:, :, None] * 2.0 ** -51
    tol[..., ia] += (a.abs() + b.abs()) * off
    tol[..., ib] += (a.abs() + b.abs()) * off
    return y, tol


ROT = [  # batch, length, q heads, k heads, dim, rotated, sections, far
    (1, 1, 1, 1, 2, 2, (1,), 10), (2, 3, 4, 2, 32, 32, (4, 6, 6), 100), (1, 5, 3, 1, 64, 32, (16,), 4096),
    (3, 7, 8, 2, 128, 128, (16, 24, 24), 1 << 20), (1, 300, 8, 8, 32, 32, (8, 8), 25),
    (2, 17, 5, 1, 80, 80, (13, 0, 27), 1000), (1, 9, 2, 2, 96, 90, (45,), 50000),
    (1, 33, 28, 4, 256, 128, (10, 20, 30, 4), 1 << 24), (64, 1, 32, 8, 128, 128, (16, 24, 24), 32768),
    (1, 2, 1, 1, 1024, 1024, (512,), 99), (2, 40, 1, 3, 6, 4, (1, 1), 7), (1, 600, 16, 16, 64, 64, (8, 12, 12), 2500),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROT)
def test_rotary(cuda, case, interleaved, t):
    B, L, qh, kh, D, R, sections, far = case
    T = TYPES[t]
    g = gen(B * L + D)
    qk = normal(g, B, L, qh + kh, D, t=T)
    q, k = qk[:, :, :qh], qk[:, :, qh:]
    pos = torch.randint(-far // 4, far, (len(sections), B, L), generator=g).cuda()
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64, device="cuda") * 2 / R)
    for inverse in (False, True):
        for p in (pos, pos.int()):
            got = ppdl.rotary(q, k, p, freq, sections, interleaved=interleaved, inverse=inverse)
            for x, y in zip((q, k), got):
                want, tol = rot_want(x, pos, freq, sections, interleaved, inverse)
                close(y, want, tol)
                assert torch.equal(y[..., R:], x[..., R:])
    # in place on views of one buffer; q alone
    alone = ppdl.rotary(q, None, pos, freq, sections, interleaved=interleaved, inverse=True)
    assert torch.equal(alone[0], got[0]) and alone[1] is None
    a, b = ppdl.rotary(q, k, pos, freq, sections, interleaved=interleaved, inverse=True, inplace=True)
    assert a.data_ptr() == q.data_ptr() and torch.equal(q, got[0]) and torch.equal(k, got[1])


def test_rotary_strides(cuda):
    """Heads in front of tokens, odd offsets, positions shared by the batch."""
    g = gen(21)
    B, L, H, D = 3, 11, 4, 64
    freq = 500.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    pos = torch.randint(0, 999, (2, 1, L), generator=g).cuda().expand(2, B, L)
    for T in TYPES.values():
        for x in (normal(g, B, H, L, D, t=T).transpose(1, 2), normal(g, B, L, H, D + 1, t=T)[..., 1:],
                  normal(g, L, B, H, 2 * D, t=T).transpose(0, 1)[..., 8:8 + D]):
            y, _ = ppdl.rotary(x, None, pos, freq, (20, 12))
            want, tol = rot_want(x, pos, freq, (20, 12), False, False)
            close(y, want, tol)
            keep = x.clone()
            ppdl.rotary(x, None, pos, freq, (20, 12), inplace=True)
            assert torch.equal(x, y)
            ppdl.rotary(x, None, pos, freq, (20, 12), inplace=True, inverse=True)
            _, back = rot_want(want.to(T), pos, freq, (20, 12), False, True)
            # there and back: the first rounding turns with its pair, the second adds its own
            size = 1.5 * half(T) * (keep.double().abs() + keep.double().roll(D // 2, -1).abs()) + 2 * tol.amax()
            close(x, keep.double(), size + back)


# ---- together ------------------------------------------------------------------------------------

def test_attention_block(cuda):
    """norm -> 8-bit q|k|v projection -> rotary on the views q and k -> the
    attention core -> 8-bit projection with the residual -> norm, as a program
    runs it, each step against 64 bits on what the step was given; then the
    whole captured once and replayed on new data, and run on another stream."""
    B, T, H = 2, 300, 8
    D = H * 32
    g = gen(1)
    h = normal(g, B, T, D)
    w1, b1 = normal(g, D, shift=1.0, scale=0.2), normal(g, D, scale=0.2)
    wqkv, sqkv = ppdl.quantize_rows(normal(g, 3 * D, D, scale=D ** -0.5))
    wo, so = ppdl.quantize_rows(normal(g, D, D, scale=D ** -0.5))
    bq = normal(g, 3 * D, scale=0.1)
    gy, gx = torch.meshgrid(torch.arange(20), torch.arange(15), indexing="ij")
    pos = torch.stack((gy.flatten(), gx.flatten())).cuda()[:, None].expand(2, B, T)
    freq = 100.0 ** (-torch.arange(16, dtype=torch.float64, device="cuda") / 16)
    L = ppdl.lib()

    def block(h):
        n = ppdl.layernorm(h, w1, b1)
        qkv = ppdl.linear_i8(n, wqkv, sqkv, bias=bq).view(B, T, 3, H, 32)
        before = qkv.clone()
        q, k = ppdl.rotary(qkv[:, :, 0], qkv[:, :, 1], pos, freq, (8, 8), inplace=True)
        L.ppdl_attention_f32.argtypes = ([C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_longlong, C.c_int,
                                         C.c_longlong, C.c_float, C.c_void_p])
        v = qkv[:, :, 2].contiguous()
        o = torch.empty((B, T, D), device="cuda")
        ppdl.check(L.ppdl_attention_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, T, H,
                                        3 * D, T * 3 * D, D, T * D, 32 ** -0.5,
                                        torch.cuda.current_stream().cuda_stream))
        out = ppdl.linear_i8(o, wo, so, residual=h)
        y, mean, rstd = ppdl.layernorm(out, w1, b1, return_stats=True)
        return n, before, qkv, o, out, y

    n, before, qkv, o, out, y = block(h)
    want = ln_want(h, w1, b1, 1e-5)
    close(n, want[0], want[4])
    nq, ns = q_want(n)
    want, tol = lin_want(nq.view(-1, D), ns.view(-1), wqkv, sqkv, bq, "none", None, torch.float32)
    close(before.view(-1, 3 * D), want, tol)
    for i in range(2):
        want, tol = rot_want(before[:, :, i], pos, freq, (8, 8), False, False)
        close(qkv[:, :, i], want, tol)
    q, k, v = (qkv[:, :, i].double().transpose(1, 2) for i in range(3))
    want = (torch.softmax(q @ k.transpose(-1, -2) * 32 ** -0.5, -1) @ v).transpose(1, 2).reshape(B, T, D)
    assert float((o.double() - want).abs().max()) <= 2e-6 * float(v.abs().max())
    oq, os_ = q_want(o)
    want, tol = lin_want(oq.view(-1, D), os_.view(-1), wo, so, None, "none", h.view(-1, D), torch.float32)
    close(out.view(-1, D), want, tol)
    want = ln_want(out, w1, b1, 1e-5)
    close(y, want[0], want[4])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(block(h)[-1], y)
    torch.cuda.current_stream().wait_stream(side)
    still = h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block(still)[-1]
    graph.replay()
    assert torch.equal(captured, y)
    h2 = normal(g, B, T, D)
    still.copy_(h2)
    graph.replay()
    assert torch.equal(captured, block(h2)[-1])


def test_training_step_captured(cuda):
    """Forward and backward of a residual norm, captured twice; the graphs run
    one after the other on their own workspaces."""
    g = gen(2)
    x, r, dy, ds = (normal(g, 700, 512, t=torch.bfloat16) for _ in range(4))
    w, b = normal(g, 512), normal(g, 512)

    def step():
        y, s, mean, rstd = ppdl.layernorm(x, w, b, residual=r, return_sum=True, return_stats=True)
        return (y,) + ppdl.layernorm_backward(dy, s, w, mean, rstd, dsum=ds)

    want = step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for graph, got in graphs * 2:
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_two_streams_at_once(cuda):
    g = gen(4)
    x = [normal(g, 2000, 1024, t=torch.bfloat16) for _ in range(2)]
    wq, ws = ppdl.quantize_rows(normal(g, 1024, 1024))
    want = [ppdl.linear_i8(v, wq, ws) for v in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ppdl.linear_i8(x[i], wq, ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(v, want[i]) for v in got[i])


FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, ppdl
x, w = torch.randn(300, 2048, device="cuda").bfloat16(), torch.randn(2048, device="cuda")
wq, ws = torch.randint(-127, 128, (512, 2048), device="cuda").to(torch.int8), torch.rand(512, device="cuda")
pos, freq = torch.arange(300, device="cuda").view(1, 1, 300), torch.ones(64, dtype=torch.float64, device="cuda")
def step():
    y, s, mean, rstd = ppdl.layernorm(x, w, w, residual=x, return_sum=True, return_stats=True)
    return (y, *ppdl.layernorm_backward(x, s, w, mean, rstd), ppdl.linear_i8(x, wq, ws), ppdl.linear_i8(x[:1], wq, ws),
            ppdl.rotary(x.view(1, 300, 16, 128), None, pos, freq, (64,))[0])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
assert ppdl.lib().ppdl_op_device_error() == 0
"""


def test_first_calls_inside_a_capture(cuda):
    """A process whose first call of each operator is a captured one."""
    import os
    import subprocess
    import sys
    subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(ppdl.__file__)], check=True, timeout=300)


def test_tensors_of_another_device(cuda, monkeypatch):
    """Tensors of a GPU that is not the current one: the call is made with
    theirs current (shown on one GPU, by a current device that claims to be
    another until it is set)."""
    x, w = torch.randn(5, 64, device="cuda"), torch.ones(64, device="cuda")
    wq, ws = ppdl.quantize_rows(torch.randn(8, 64, device="cuda"))
    h, pos = x.view(1, 5, 1, 64), torch.arange(5, device="cuda").view(1, 1, 5)
    freq = torch.ones(32, dtype=torch.float64, device="cuda")
    _, mean, rstd = ppdl.layernorm(x, w, return_stats=True)
    calls = [lambda: ppdl.layernorm(x, w, w), lambda: ppdl.layernorm_backward(x, x, w, mean, rstd),
             lambda: ppdl.quantize_rows(x), lambda: ppdl.linear_i8(x, wq, ws),
             lambda: ppdl.rotary(h, h, pos, freq, (32,))]
    want = [f() for f in calls]
    entered = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *a):
            pass

    for f, expected in zip(calls, want):
        n = len(entered)
        monkeypatch.setitem(ppdl._tt, "device", Device)
        monkeypatch.setitem(ppdl._tt, "current", lambda: 0 if len(entered) > n else 7)
        got = f()
        assert entered[n:] == [0]
        pairs = zip(got, expected) if isinstance(got, tuple) else [(got, expected)]
        assert all(torch.equal(a, b) for a, b in pairs)


def test_no_kernel_gave_up(cuda):
    torch.cuda.synchronize()
    assert ppdl.lib().ppdl_op_device_error() == 0
