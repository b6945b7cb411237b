"""Calls of the transformer-block operators at the edges of what they take:
infinities, NaNs and far scales in the data, overlapping views, widths next
to 2^31.  Tolerances count roundings as in test_block_ops_gpu."""
import ctypes
import threading

import pytest
import torch

import ppdl
from test_block_ops_gpu import TYPES, U, bwd_want, close, gen, half, ln_want, normal, q_want, rot_want

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


WIDEST = 2 ** 31 - 1


def guarded(n, t, fill):
    """n values with 4096 of `fill` in front and behind, all of that value."""
    room = torch.full((n + 8192,), fill, device="cuda", dtype=t)
    return room, room[4096:4096 + n]


def test_widest_row_quantised(cuda):
    """The last step over a row of 2^31 - 1 values passes 2^31."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    x[-1] = 0.5
    room, q = guarded(2 ** 31, torch.int8, 55)
    scale = torch.zeros(1, device="cuda")
    ppdl.check(ppdl.lib().ppdl_quantize_rows_i8(x.data_ptr(), WIDEST, 1, 1, WIDEST, q.data_ptr(), 2 ** 31,
                                                scale.data_ptr(), torch.cuda.current_stream().cuda_stream))
    step = (torch.ones((), dtype=torch.float64) / 127).float()
    assert scale[0] == step
    assert (q[0:WIDEST - 1:2] == 127).all() and (q[1:WIDEST:2] == -127).all()
    assert q[WIDEST - 1] == round(0.5 / step.item())
    assert (room[:4096] == 55).all() and (room[4096 + WIDEST:] == 55).all()


def test_widest_row_normalised(cuda):
    """Values +-1 in turn: 512 threads add one sign each, 2^22 times, which is
    exact; the mean is 2^-31, the variance 1."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    room, y = guarded(WIDEST, torch.bfloat16, 7.0)
    ppdl.check(ppdl.lib().ppdl_layernorm(x.data_ptr(), WIDEST, None, 0, None, None, 1, 1, 1, WIDEST, 1e-5, y.data_ptr(),
                                         WIDEST, None, 0, None, None, torch.cuda.current_stream().cuda_stream))
    want = torch.tensor((1 + 1e-5) ** -0.5, dtype=torch.bfloat16).item()
    assert (y[::2] == want).all() and (y[1::2] == -want).all()
    assert (room[:4096] == 7).all() and (room[4096 + WIDEST:] == 7).all()


def test_widest_row_backward(cuda):
    """x = + - + - and dy = + + - - in turn: exact sums of 0 and 1 over the row,
    so that dx is dy to within 2^-31, at mean 0 and rstd 1."""
    x = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    x[1::2] = -1
    dy = torch.ones(WIDEST, device="cuda", dtype=torch.bfloat16)
    dy[2::4] = -1
    dy[3::4] = -1
    room, dx = guarded(WIDEST, torch.bfloat16, 7.0)
    mean, rstd = torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")
    ppdl.check(ppdl.lib().ppdl_layernorm_backward(
        dy.data_ptr(), WIDEST, x.data_ptr(), WIDEST, None, mean.data_ptr(), rstd.data_ptr(), None, 0, 1, 1, 1, WIDEST,
        dx.data_ptr(), WIDEST, None, None, None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(dx, dy)
    assert (room[:4096] == 7).all() and (room[4096 + WIDEST:] == 7).all()


@pytest.mark.parametrize("act", ppdl.ACTS)
@pytest.mark.parametrize("M,K,N", [(1, 512, 200), (2, 300, 200), (16, 512, 1000), (5, 2047, 260), (40, 256, 96),
                                   (300, 256, 1024), (2400, 256, 256), (5003, 200, 2100), (20, 4096, 4097),
                                   (100, 4096, 641), (2049, 513, 1025), (2570, 1024, 1537)])
def test_bad_tokens_stay_bad(cuda, M, K, N, act):
    """A token with a NaN or an infinity is a row of NaNs behind every
    activation, in every form of the product; so is a channel whose scale or
    bias is a NaN.  Nothing else changes."""
    g = gen(M + K + N)
    for T in TYPES.values():
        x, res = normal(g, M, K, t=T), normal(g, M, N, t=T)
        wq, ws = ppdl.quantize_rows(normal(g, N, K, scale=K ** -0.5))
        bias = normal(g, N)
        for r in (None, res):
            clean = ppdl.linear_i8(x, wq, ws, bias=bias, act=act, residual=r)
            bad, bs, bb = x.clone(), ws.clone(), bias.clone()
            rows, cols = {M - 1, M // 2}, {N - 1, N // 3}
            bad[M - 1, K - 1], bad[M // 2, 0] = NAN, -INF
            bs[N - 1], bb[N // 3] = NAN, NAN
            y = ppdl.linear_i8(bad, wq, bs, bias=bb, act=act, residual=r)
            keep_r = [i for i in range(M) if i not in rows]
            keep_c = [i for i in range(N) if i not in cols]
            assert y[list(rows)].isnan().all() and y[:, list(cols)].isnan().all()
            assert torch.equal(y[keep_r][:, keep_c], clean[keep_r][:, keep_c])


# rows that fill no block of any form; by value, groups, rings and two readings
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 3), (5, 31), (33, 51), (3, 101), (13, 257), (7, 333), (5, 641), (9, 1001),
                                    (5, 1153), (3, 2501), (3, 4097), (2, 16383), (2, 20001), (64001, 79), (17001, 257),
                                    (3651, 1153), (5, 8), (5, 64), (33, 256), (13, 1000), (5, 4096), (3, 8192),
                                    (3, 16384), (2, 32768)])
def test_backward_infinite_gradient_of_the_last_row(cuda, rows, D, t):
    """An infinity in the last row's gradient spoils its own row of dx and its
    own columns of dweight and dbias: their sums are infinite, not NaN."""
    T = TYPES[t]
    g = gen(rows + D)
    x, dy, w = normal(g, rows, D, t=T), normal(g, rows, D, t=T), normal(g, D, t=T, shift=1.0, scale=0.2)
    _, mean, rstd = ppdl.layernorm(x, w, None, return_stats=True)
    up, down = D - 1, D // 2
    xh = (x[-1].double() - mean[-1].double()) * rstd[-1].double()
    dy[-1, up], dy[-1, down] = INF, -INF
    dx, dw, db = ppdl.layernorm_backward(dy, x, w, mean, rstd)
    assert db[up] == INF and db[down] == -INF
    assert dw[up] == INF * float(xh[up].sign()) and dw[down] == -INF * float(xh[down].sign())
    finite = dy.clone()
    finite[-1, up] = finite[-1, down] = 0
    want, tol = bwd_want(finite, x, w, mean, rstd)
    keep = [c for c in range(D) if c not in (up, down)]
    close(dw[keep], want[1][keep], tol[1][keep])
    close(db[keep], want[2][keep], tol[2][keep])
    close(dx[:-1], want[0][:-1], tol[0][:-1])


FORMS = [(5, 31), (5, 64), (3, 100), (7, 257), (6, 333), (5, 641), (8, 1001), (5, 1153), (3, 2501), (3, 4097),
         (2, 9999), (2, 16383), (2, 20001), (5, 256), (8, 1000), (5, 4096), (3, 8192), (3, 12000), (2, 16384), (2, 32768)]


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", FORMS)
def test_backward_common_offset(cuda, rows, D, t):
    """Rows whose values share a large offset: (x - mean) is taken first, one
    rounding of a small difference, and its product with rstd another, in
    every form; a product of the offset and rstd would be rounded to far more."""
    T = TYPES[t]
    g = gen(rows * 3 + D)
    x = normal(g, rows, D, scale=1.0 if t == "f32" else 128.0, shift=2.0 ** 14, t=T)
    mean = x.double().mean(-1).float()
    rstd = (x.double().var(-1, unbiased=False) + 1e-5).rsqrt().float()
    w = normal(g, D, shift=1.0, scale=0.2)
    mm, r = mean.double()[:, None], rstd.double()[:, None]
    xh = (x.double() - mm) * r
    dy = (xh.float() / xh.abs().max().float() + 0.1 * normal(g, rows, D)).to(T)
    gg = dy.double() * w.double()
    m1, m2 = gg.mean(-1, keepdim=True), (gg * xh).mean(-1, keepdim=True)
    want = r * (gg - m1 - xh * m2)
    k = D / 32 + 24
    size = gg.abs() + gg.abs().mean(-1, keepdim=True) + xh.abs() * (gg * xh).abs().mean(-1, keepdim=True)
    # xh: 2 u; with it in two products and the two sums
    tol = r * ((k + 8) * U * size) + (half(T) + U) * want.abs() + 1e-38
    dx, dw, db = ppdl.layernorm_backward(dy, x, w, mean, rstd)
    close(dx, want, tol)
    # at most 8 rows: 8 additions, the product and xh's 2 u
    p = dy.double() * xh
    close(dw, p.sum(0), 12 * U * p.abs().sum(0) + 2 * U * p.sum(0).abs() + 1e-38)
    close(db, dy.double().sum(0), 10 * U * dy.double().abs().sum(0) + 1e-38)


@pytest.mark.parametrize("rows,D", FORMS + [(64001, 79), (17001, 257), (3651, 1153)])
def test_backward_constant_rows_of_large_values(cuda, rows, D):
    """x = mean = 2^90 and rstd = 2^50 (a constant row with a small eps): xh is
    zero, although the product of mean and rstd passes FP32's range, in the
    places past the row's end as well."""
    for T in (torch.float32, torch.bfloat16):
        x = torch.full((rows, D), 2.0 ** 90, device="cuda", dtype=T)
        mean, rstd = torch.full((rows,), 2.0 ** 90, device="cuda"), torch.full((rows,), 2.0 ** 50, device="cuda")
        dy = normal(gen(D), rows, D, t=T)
        dx, dw, db = ppdl.layernorm_backward(dy, x, None, mean, rstd)
        want, tol = bwd_want(dy, x * 0, None, mean * 0, rstd)
        close(dx, want[0], tol[0])
        assert (dw == 0).all()
        close(db, want[2], tol[2])


LIN = [(1, 512, 200), (2, 300, 200), (16, 512, 1000), (5, 2047, 260), (40, 256, 96), (300, 256, 1024), (2400, 256, 256),
       (5003, 200, 2100), (20, 4096, 4097), (100, 4096, 641), (2049, 513, 1025), (2570, 1024, 1537)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", LIN)
def test_linear_far_scales(cuda, M, K, N, t):
    """Scales whose product leaves FP32's normal range, with results inside
    it: no digits lost, no NaN where a sum is zero; ordinary tokens and
    channels beside them keep their bits."""
    T = TYPES[t]
    g = gen(M + K + N)
    q = torch.randint(-127, 128, (M, (K + 15) // 16 * 16), generator=g).to(torch.int8).cuda()[:, :K]
    w = torch.randint(-127, 128, (N, (K + 15) // 16 * 16), generator=g).to(torch.int8).cuda()[:, :K]
    qs, ws = 1e-3 * (1 + torch.rand(M, generator=g)).cuda(), 1e-3 * (1 + torch.rand(N, generator=g)).cuda()
    w[N // 2] = 0
    clean = ppdl.linear_i8(q, w, ws, x_scale=qs, out_dtype=T)
    acc = q.double() @ w.double().t()
    for rows, cols in (((0, M - 1, M // 3), ()), ((), (0, N - 1, N // 2, N // 3)), ((M // 2, M - 1), (1, N // 2, N - 2))):
        far_q, far_w = qs.clone(), ws.clone()
        for i, r in enumerate(rows):
            far_q[r] = (1e-37, 1e34, 1e-36)[i] if not cols else (1e-20, 1e24)[i % 2]
        for i, c in enumerate(cols):
            far_w[c] = (1e-37, 1e35, 1e37, 1e-36)[i] if not rows else (1e-20, 1e33, 1e-25)[i]
        for act in ("none", "relu"):
            y = ppdl.linear_i8(q, w, far_w, x_scale=far_q, act=act, out_dtype=T)
            want = acc * far_q.double()[:, None] * far_w.double()
            want = want.clamp_min(0) if act == "relu" else want
            # a result past the type's range is an infinity of its sign, next to its end either
            end = torch.finfo(T).max
            tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[T]
            inside = want.abs() < 0.99 * end
            tol = (half(T) + 5 * U) * want.abs() + tiny
            assert (y.isfinite() | ~inside).all()
            close(torch.where(inside, y.double(), 0.0), torch.where(inside, want, 0.0), tol)
            past = want.abs() > 1.01 * end
            assert torch.equal(y[past].double(), want[past].sign() * INF)
            if act == "none":
                kr = [i for i in range(M) if i not in rows]
                kc = [i for i in range(N) if i not in cols]
                assert torch.equal(y[kr][:, kc], clean[kr][:, kc])


def test_linear_tiny_tokens(cuda):
    """Tokens of 1e-35 through weights of 1/16: results of 1e-34, normal
    numbers, to a few roundings."""
    g = gen(77)
    for M in (1, 2, 40, 600):
        x, (wq, ws) = normal(g, M, 256, scale=1e-35), ppdl.quantize_rows(normal(g, 96, 256, scale=1 / 16))
        xq, xs = q_want(x)
        want = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
        close(ppdl.linear_i8(x, wq, ws), want, 5 * U * want.abs() + 2.0 ** -149)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_overlapping_inputs(cuda, interleaved, t):
    """Windows of one buffer and expanded views as queries and keys: the
    results are tensors of their own."""
    g = gen(31)
    T, B, L, H, D = TYPES[t], 2, 5, 3, 8
    base = normal(g, 400, t=T)
    pos, freq = torch.arange(B * L, device="cuda").view(1, B, L), torch.rand(D // 2, generator=g).double().cuda()
    for strides in ((100, 30, 1, 1), (100, 1, 8, 1), (1, 50, 8, 1), (24, 1, 8, 1), (0, 8, 16, 1), (100, 0, 8, 1),
                    (100, 24, 0, 1), (0, 0, 0, 1), (120, 24, 8, 1), (100, 3, 12, 1)):
        x = base.as_strided((B, L, H, D), strides)
        want, tol = rot_want(x, pos, freq, (D // 2,), interleaved, False)
        for y in ppdl.rotary(x, x, pos, freq, (D // 2,), interleaved=interleaved):
            close(y, want, tol)


@pytest.mark.parametrize("t,rows,D", [("bf16", 2200000, 1024), ("f16", 1900001, 1153), ("bf16", 560000, 4001),
                                      ("f32", 140000, 16384)])
def test_norm_offsets_past_31_bits(cuda, t, rows, D):
    """More than 2^31 values: the first and last rows against the definition,
    the weights' gradients by gradients that are zero elsewhere."""
    T = TYPES[t]
    assert rows * D > 2 ** 31
    x = torch.empty((rows, D), device="cuda", dtype=T)
    x[:] = normal(gen(1), 1, D, t=T)
    ends = [slice(0, 300), slice(rows - 300, rows)]
    for i, e in enumerate(ends):
        x[e] = normal(gen(2 + i), 300, D, t=T)
    w, b = normal(gen(5), D, shift=1.0, scale=0.3), normal(gen(6), D)
    y, mean, rstd = ppdl.layernorm(x, w, b, return_stats=True)
    for e in ends:
        want = ln_want(x[e], w, b, 1e-5)
        close(y[e], want[0], want[4])
    q, scale = ppdl.quantize_rows(x)
    for e in ends:
        wq, ws = q_want(x[e])
        assert torch.equal(q[e], wq) and torch.equal(scale[e], ws)
    del q, scale
    y.zero_()
    for i, e in enumerate(ends):
        y[e] = normal(gen(7 + i), 300, D, t=T)
    dx, dw, db = ppdl.layernorm_backward(y, x, w, mean, rstd)
    both = torch.cat([torch.arange(rows, device="cuda")[e] for e in ends])
    want, tol = bwd_want(y[both], x[both], w, mean[both], rstd[both])
    # a column's sum takes in rows / 128 + 320 terms in a row at most, all but 600 zeros
    for got, a, c in zip((dx[both], dw, db), want, tol):
        close(got, a, c)
    assert (dx[300:rows - 300] == 0).all()


def test_linear_offsets_past_31_bits(cuda):
    M, K, N = 1100000, 2000, 2100
    q = torch.zeros((M, K), device="cuda", dtype=torch.int8)
    ends = [slice(0, 300), slice(M - 300, M)]
    g = gen(9)
    for e in ends:
        q[e] = torch.randint(-128, 128, (300, K), generator=g).to(torch.int8).cuda()
    w = torch.randint(-128, 128, (N, K), generator=g).to(torch.int8).cuda()
    y = ppdl.linear_i8(q, w, torch.ones(N, device="cuda"), x_scale=torch.ones(M, device="cuda"))
    assert y.numel() > 2 ** 31 and q.numel() > 2 ** 31
    for e in ends:
        want = q[e].double() @ w.double().t()
        assert float(want.abs().max()) < 2 ** 24 and torch.equal(y[e].double(), want)
    assert (y[300:M - 300] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [128, 126])
def test_rotary_offsets_past_31_bits(cuda, dim, interleaved):
    B, L, H = 2, 540000, 16
    qk = torch.empty((B, L, H, dim), device="cuda", dtype=torch.bfloat16)
    assert qk.numel() > 2 ** 31
    qk[:] = normal(gen(3), 1, 1, H, dim, t=torch.bfloat16)
    pos = torch.arange(L, device="cuda").view(1, 1, L).expand(1, B, L)
    freq = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device="cuda") / 64)
    y, _ = ppdl.rotary(qk, None, pos, freq, (dim // 2,), interleaved=interleaved)
    for e in (slice(0, 200), slice(L - 200, L)):
        want, tol = rot_want(qk[:, e], pos[:, :, e], freq, (dim // 2,), interleaved, False)
        close(y[:, e], want, tol)


def test_first_call_of_a_new_thread(cuda):
    """A host thread that has not used the GPU before: its first call may be
    any of the operators, those that make tensor maps among them."""
    g = gen(41)
    x, few = normal(g, 300, 512), normal(g, 2, 512)
    wq, ws = ppdl.quantize_rows(normal(g, 96, 512))
    q, s = ppdl.quantize_rows(x)
    heads, pos = x.view(1, 300, 8, 64), torch.arange(300, device="cuda").view(1, 1, 300)
    freq = torch.rand(32, generator=g).double().cuda()
    _, mean, rstd = ppdl.layernorm(x, return_stats=True)
    a, b = normal(g, 256, 128), normal(g, 64, 128)
    L = ppdl.lib()

    def gemm():
        ws_, out = torch.empty(2 * 64 * 128, device="cuda"), torch.empty((256, 64), device="cuda")
        P, LL = ctypes.c_void_p, ctypes.c_longlong
        ppdl.check(L.ppdl_gemm_tf32x3(256, 64, 128, 1, P(a.data_ptr()), 0, LL(128), LL(256 * 128), P(b.data_ptr()),
                                      P(ws_.data_ptr()), P(out.data_ptr()), LL(64), LL(1), LL(256 * 64),
                                      P(torch.cuda.current_stream().cuda_stream)))
        return out

    calls = [lambda: ppdl.linear_i8(few, wq, ws), lambda: ppdl.linear_i8(few[:1], wq, ws),
             lambda: ppdl.linear_i8(q, wq, ws, x_scale=s), lambda: ppdl.linear_i8(x, wq, ws), gemm,
             lambda: ppdl.quantize_rows(x)[0], lambda: ppdl.layernorm(x),
             lambda: ppdl.layernorm_backward(x, x, None, mean, rstd)[1],
             lambda: ppdl.rotary(heads, None, pos, freq, (32,))[0]]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    for f, w in zip(calls, want):
        got = []

        def run():
            try:
                got.append(f())
            except Exception as e:
                got.append(e)

        t = threading.Thread(target=run)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert torch.is_tensor(got[0]), got[0]
        assert torch.equal(got[0], w)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(3000, 2000), (1501, 4096), (1301, 8192), (9001, 513), (2100, 2049)])
def test_norm_in_place_through_shared_memory(cuda, rows, D, t):
    """Results over inputs where several rows are on their way at once: y over
    x and the sum over the residual, and the other way round; x as its own
    residual."""
    g = gen(rows)
    T, code, stream = TYPES[t], {"bf16": 1, "f16": 2}[t], torch.cuda.current_stream().cuda_stream
    x, r, w = normal(g, rows, D, t=T), normal(g, rows, D, t=T), normal(g, D, t=T)
    y, s = ppdl.layernorm(x, w, w, residual=r, return_sum=True)

    def run(a, b, out, total):
        ppdl.check(ppdl.lib().ppdl_layernorm(
            a.data_ptr(), D, b.data_ptr(), D, w.data_ptr(), w.data_ptr(), code, code, rows, D, 1e-5, out.data_ptr(), D,
            total.data_ptr() if total is not None else None, D, None, None, stream))

    a, b = x.clone(), r.clone()
    run(a, b, a, b)
    assert torch.equal(a, y) and torch.equal(b, s)
    a, b = x.clone(), r.clone()
    run(a, b, b, a)
    assert torch.equal(b, y) and torch.equal(a, s)
    want = ppdl.layernorm(x, w, w, residual=x)
    run(x, x, x, None)
    assert torch.equal(x, want)
