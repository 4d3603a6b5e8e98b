"""K12 (RMS norm of a residual sum) and K13 (gated feed-forward block), forward, in 8 bits and backward, against their
definitions in 64 bits on the same inputs.

Tolerances, element by element.  u = finfo(type).eps / 2 is the relative error of one rounding to the type; every kernel
rounds each output once, from 32-bit arithmetic whose own errors are bounded by the usual  n 2^-24 sum|terms|  for a sum of
n terms.  Where a half-precision result is subnormal the rounding is absolute (2^-25).  The gradient of K13 rounds dg and du
to the type between its two steps: each counts u |dg| in every sum that takes it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from framepack_amd import ops  # noqa: E402

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
E32 = 2.0 ** -24
EPS = 1e-6


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def tiny_of(dtype):
    return 2.0 ** -25 if dtype == HF else 0.0


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got - want)[bad][:4].tolist(), want[bad][:4].tolist(),
                           torch.as_tensor(tol, device=got.device).expand_as(want)[bad][:4].tolist())


def rel_l2(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


def embed(t, left, right, fill=float("nan")):
    """t as a row-strided view into a wider buffer of another value; returns (view, buffer)."""
    big = torch.full((t.shape[0], left + t.shape[1] + right), fill, dtype=torch.float32, device=t.device).to(t.dtype)
    big[:, left:left + t.shape[1]] = t
    return big[:, left:left + t.shape[1]], big


# ---- K12 ---------------------------------------------------------------------------------------------------------

def norm64(x, resid, w, eps=EPS):
    h = x.double() if resid is None else x.double() + resid.double()
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()


def norm_tol(y, dtype, cols):
    # sum of squares: relative error cols 2^-24 of a positive sum, halved by the root; four more roundings
    return y.abs() * (u_of(dtype) + (cols / 2 + 8) * E32) + tiny_of(dtype)


NORM_SHAPES = [(1, 1), (3, 7), (1, 64), (5, 72), (300, 128), (4, 1000), (7, 1001), (33, 1152), (1, 4096), (257, 4096), (3, 5003),
               (2, 8192), (9, 8200), (2, 20000), (1, 40001), (2, 70000)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm(rows, cols, dtype):
    x, r = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, scale=3.0, dtype=dtype)
    w = (1 + randn(cols, seed=3, scale=0.3)).to(dtype)
    y, h = ops.rmsnorm_residual(x, w, r)
    h64, y64 = norm64(x, r, w)
    within(h, h64, h64.abs() * (u_of(dtype) + 2 * E32) + tiny_of(dtype), "h")
    within(y, y64, norm_tol(y64, dtype, cols), "y")
    y1, h1 = ops.rmsnorm_residual(x, w)
    assert h1 is x
    _, y64 = norm64(x, None, w)
    within(y1, y64, norm_tol(y64, dtype, cols), "y without a residual")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cols", [64, 1000, 1001])
def test_norm_of_strided_rows_leaves_the_gaps(cols, dtype):
    rows = 37
    x, r = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, dtype=dtype)
    w = (1 + randn(cols, seed=3, scale=0.3)).to(dtype)
    want, want_h = ops.rmsnorm_residual(x, w, r)
    for left, right in ((8, 16), (3, 2)):                  # aligned for wide loads or not
        xv, _ = embed(x, left, right)
        rv, _ = embed(r, left, right)
        ov, obuf = embed(torch.zeros_like(x), left, right, fill=7.0)
        hv, hbuf = embed(torch.zeros_like(x), left, right, fill=7.0)
        y, h = ops.rmsnorm_residual(xv, w, rv, out=ov, resid_out=hv)
        assert y.data_ptr() == ov.data_ptr() and h.data_ptr() == hv.data_ptr()
        within(y, want, want.double().abs() * (2 * u_of(dtype)) + 2 * tiny_of(dtype))
        assert torch.equal(h, want_h)
        for buf in (obuf, hbuf):
            assert (buf[:, :left] == 7).all() and (buf[:, left + cols:] == 7).all()
    y, h = ops.rmsnorm_residual(x[:1].expand(rows, cols), w, r)             # one row of x for all
    h64, y64 = norm64(x[:1].expand(rows, cols), r, w)
    within(y, y64, norm_tol(y64, dtype, cols))


@pytest.mark.parametrize("cols", [64, 1001, 4096, 20000, 70000])
def test_norm_in_place(cols):
    x, r, w = randn(9, cols, seed=1, dtype=BF), randn(9, cols, seed=2, dtype=BF), randn(cols, seed=3, dtype=BF)
    y0, h0 = ops.rmsnorm_residual(x, w, r)
    for swap in (False, True):
        a, b = x.clone(), r.clone()
        y, h = ops.rmsnorm_residual(a, w, b, out=b if swap else a, resid_out=a if swap else b)
        assert torch.equal(y, y0) and torch.equal(h, h0)
        assert torch.equal(a, h0 if swap else y0) and torch.equal(b, y0 if swap else h0)


def test_norm_of_rows_of_zeros_infinities_and_nan_keeps_to_the_row():
    cols = 1024
    x, w = randn(8, cols, seed=1, dtype=BF), randn(cols, seed=3, dtype=BF)
    r = randn(8, cols, seed=2, dtype=BF)
    y0, h0 = ops.rmsnorm_residual(x, w, r)
    q0, s0, _ = ops.rmsnorm_residual_fp8(x, w, r)
    x[1], r[1] = 0, 0
    x[3, 5] = float("nan")
    x[5, 7] = float("inf")
    y, h = ops.rmsnorm_residual(x, w, r)
    q, s, hq = ops.rmsnorm_residual_fp8(x, w, r)
    keep = [0, 2, 4, 6, 7]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(h[keep], h0[keep])
    assert torch.equal(q[keep].view(torch.uint8), q0[keep].view(torch.uint8)) and torch.equal(s[keep], s0[keep])
    assert (y[1] == 0).all() and (h[1] == 0).all() and s[1].item() == 1.0 and (q[1].float() == 0).all()
    assert y[3].isnan().all() and q[3].float().isnan().all() and h[3].isnan().sum() == 1
    # inf: the mean is inf, the finite values go to 0 and inf * 0 is NaN - as in torch
    f = x[5].float() + r[5].float()
    want = f * torch.rsqrt(f.square().mean() + EPS) * w.float()
    assert torch.equal(y[5].isnan(), want.isnan()) and (y[5][~want.isnan()] == 0).all() and h[5, 7].item() == float("inf")
    assert torch.equal(hq.isnan(), h.isnan())


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm_to_8_bits(rows, cols):
    x, r = randn(rows, cols, seed=1, dtype=BF), randn(rows, cols, seed=2, scale=3.0, dtype=BF)
    x[0, 0] = 90.0                                          # an outlier: only its row loses resolution
    w = (1 + randn(cols, seed=3, scale=0.3)).to(BF)
    q, s, h = ops.rmsnorm_residual_fp8(x, w, r)
    h64, y64 = norm64(x, r, w)
    within(h, h64, h64.abs() * (u_of(BF) + 2 * E32), "h")
    amax = y64.abs().amax(1)
    fp = (cols / 2 + 10) * E32
    within(s, amax / 448, amax / 448 * fp, "scale")
    deq = q.double() * s.double()[:, None]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normal range
    within(deq, y64, (y64.abs() * 2.0 ** -4).clamp_min(0) * (1 + 4 * fp) + s.double()[:, None] * 2.0 ** -10 + y64.abs() * fp, "q")
    assert not q.float().isnan().any()
    # nearly always the nearest of all e4m3 values
    ref = (y64 / (amax / 448)[:, None]).float().to(ops.FP8).float()
    assert (q.float() != ref).double().mean().item() <= 1e-3 + 2 / (rows * cols)
    ov, obuf = embed(torch.zeros(rows, cols, device=DEV), 5, 6, fill=1.0)
    o8 = obuf.to(ops.FP8)
    q2, s2, _ = ops.rmsnorm_residual_fp8(x, w, r, out=o8[:, 5:5 + cols])
    within(q2.double() * s2.double()[:, None], deq, deq.abs() * 2.0 ** -3 * (1 + 4 * fp) + s.double()[:, None] * 2.0 ** -9)
    assert (o8[:, :5].float() == 1).all() and (o8[:, 5 + cols:].float() == 1).all()


def norm_grad64(dy, h, w, dh, eps=EPS):
    dy, h, w = dy.double(), h.double(), w.double()
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    n, dn = h * r, dy * w
    k = (dn * n).mean(1, keepdim=True)
    dx = r * (dn - n * k) + (0 if dh is None else dh.double())
    terms = r * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True)) + (0 if dh is None else dh.double().abs())
    return dx, (dy * n).sum(0), terms, (dy * n).abs().sum(0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(700, 64), (1500, 520), (2049, 136)])
def test_norm_gradient(rows, cols, dtype):
    dy, h = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, scale=2.0, dtype=dtype)
    dh, w = randn(rows, cols, seed=4, dtype=dtype), (1 + randn(cols, seed=3, scale=0.3)).to(dtype)
    h[rows // 2] = 0                                        # a row of padding
    dy[rows // 2] = 0
    for up in (dh, None):
        dx, dw = ops.rmsnorm_residual_backward(dy, h, w, dh=up)
        dx64, dw64, tx, tw = norm_grad64(dy, h, w, up)
        within(dx, dx64, dx64.abs() * u_of(dtype) + tx * (cols + 16) * E32 * 2 + tiny_of(dtype), "dx")
        within(dw, dw64, dw64.abs() * u_of(dtype) + tw * (rows + cols / 2 + 16) * E32 * 2 + tiny_of(dtype), "dweight")
    again = ops.rmsnorm_residual_backward(dy, h, w)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)          # a fixed order
    inplace = dh.clone()
    got, _ = ops.rmsnorm_residual_backward(dy, h, w, dh=inplace, dx=inplace)
    assert got.data_ptr() == inplace.data_ptr()
    assert torch.equal(got, ops.rmsnorm_residual_backward(dy, h, w, dh=dh)[0])


def test_norm_gradient_of_strided_and_broadcast_rows():
    rows, cols = 40, 264
    dy, h, dh = (randn(rows, cols, seed=i, dtype=BF) for i in (1, 2, 3))
    w = randn(cols, seed=4, dtype=BF)
    want = ops.rmsnorm_residual_backward(dy, h, w, dh=dh)
    for left, right in ((8, 8), (1, 4)):
        dxv, buf = embed(torch.zeros_like(h), left, right, fill=5.0)
        got = ops.rmsnorm_residual_backward(embed(dy, left, right)[0], embed(h, left, right)[0], w, dh=embed(dh, left, right)[0],
                                            dx=dxv)
        within(got[0], want[0], want[0].double().abs() * 2 * u_of(BF) + 1e-5)
        within(got[1], want[1], want[1].double().abs() * 2 * u_of(BF) + 1e-4)
        assert (buf[:, :left] == 5).all() and (buf[:, left + cols:] == 5).all()
    one = dy[:1].expand(rows, cols)
    assert torch.equal(ops.rmsnorm_residual_backward(one, h, w)[0], ops.rmsnorm_residual_backward(one.contiguous(), h, w)[0])


def test_norm_gradient_against_differences():
    rows, cols = 6, 96
    h, w, dy = randn(rows, cols, seed=1, dtype=BF), randn(cols, seed=2, dtype=BF), randn(rows, cols, seed=3, dtype=BF)
    dx, dw = ops.rmsnorm_residual_backward(dy, h, w)

    def loss(h_, w_):
        return (dy.double() * (h_ / torch.sqrt((h_ * h_).mean(1, keepdim=True) + EPS) * w_)).sum()

    v, z, d = randn(rows, cols, seed=5).double(), randn(cols, seed=6).double(), 1e-5
    num = (loss(h.double() + d * v, w.double()) - loss(h.double() - d * v, w.double())) / (2 * d)
    assert abs((dx.double() * v).sum() - num) <= u_of(BF) * (dx.double() * v).abs().sum() + 1e-5 * (dx.double() * v).abs().sum()
    num = (loss(h.double(), w.double() + d * z) - loss(h.double(), w.double() - d * z)) / (2 * d)
    assert abs((dw.double() * z).sum() - num) <= u_of(BF) * (dw.double() * z).abs().sum() + 1e-5 * (dw.double() * z).abs().sum()


# ---- K13 ---------------------------------------------------------------------------------------------------------

def act64(v, act):
    """act(v), act'(v) for finite v."""
    if act == ops.ACT_SILU:
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)


def ff64(x, wg, wu, bg, bu, act):
    """h, g, u and the bounds of the 32-bit sums' errors of g and u."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    n = 2 * (x.shape[1] + 4) * E32
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = n * (x.abs() @ wg.abs().t()), n * (x.abs() @ wu.abs().t())
    if bg is not None:
        g, u = g + bg.double(), u + bu.double()
        eg, eu = eg + 2 * E32 * bg.double().abs(), eu + 2 * E32 * bu.double().abs()
    return act64(g, act)[0] * u, g, u, eg, eu


def ff_tol(h, g, u, eg, eu, act, dtype):
    # |act'| < 1.13; the sigmoid's exponential has a relative error of about 2 |z| 2^-24, |z| < 88 where it is not 0
    return h.abs() * (u_of(dtype) + 400 * E32) + 1.13 * eg * u.abs() + eu * act64(g, act)[0].abs() + 1.13 * eg * eu + tiny_of(dtype)


FF_SHAPES = [(1, 1, 1), (1, 8, 64), (1, 130, 100), (2, 7, 40), (5, 64, 64), (16, 72, 128), (17, 136, 192), (33, 264, 520), (64, 520, 64),
             (65, 129, 72), (129, 256, 128), (257, 264, 256), (300, 1000, 1001), (513, 24, 320), (1, 4096, 1024), (7, 2056, 576),
             (8, 8200, 72), (9, 8201, 64), (30, 8192, 130), (48, 8209, 200), (70, 8195, 128), (600, 8193, 192), (66, 7, 5),
             (1, 24, 8192), (20, 130, 4100), (40, 17, 2048), (49, 65, 1600), (300, 129, 2050), (513, 64, 6400)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act", [ops.ACT_SILU, ops.ACT_GELU])
@pytest.mark.parametrize("M,F,K", FF_SHAPES)
def test_gated_ff(M, F, K, act, dtype):
    x = randn(M, K, seed=1, dtype=dtype)
    wg, wu = randn(F, K, seed=2, scale=2 * K ** -0.5, dtype=dtype), randn(F, K, seed=3, scale=K ** -0.5, dtype=dtype)
    bg, bu = randn(F, seed=4, dtype=dtype), randn(F, seed=5, dtype=dtype)
    for b in ((None, None), (bg, bu)):
        h64, g, u, eg, eu = ff64(x, wg, wu, *b, act)
        h = ops.gated_ff(x, wg, wu, *b, act=act)
        within(h, h64, ff_tol(h64, g, u, eg, eu, act, dtype), "h")
        h2, gate, up = ops.gated_ff(x, wg, wu, *b, act=act, keep=True)
        assert torch.equal(h, h2)
        within(gate, g, g.abs() * u_of(dtype) + 2 * eg + tiny_of(dtype), "gate")
        within(up, u, u.abs() * u_of(dtype) + 2 * eu + tiny_of(dtype), "up")


@pytest.mark.parametrize("M,F,K", [(3, 64, 128), (70, 136, 192), (300, 264, 64)])
@pytest.mark.parametrize("left,right", [(8, 24), (3, 2)])
def test_gated_ff_of_strided_operands_leaves_the_gaps(M, F, K, left, right):
    x, w = randn(M, K, seed=1, dtype=BF), randn(2 * F, K, seed=2, scale=K ** -0.5, dtype=BF)
    wv, _ = embed(w, left, right)
    xv, _ = embed(x, left, right)
    ov, buf = embed(torch.zeros(M, F, dtype=BF, device=DEV), left, right, fill=7.0)
    h = ops.gated_ff(xv, wv[:F], wv[F:], out=ov)
    h64, g, u, eg, eu = ff64(x, w[:F], w[F:], None, None, ops.ACT_SILU)
    assert h.data_ptr() == ov.data_ptr()
    within(h, h64, ff_tol(h64, g, u, eg, eu, ops.ACT_SILU, BF))
    assert (buf[:, :left] == 7).all() and (buf[:, left + F:] == 7).all()
    one = x[:1].expand(M, K)                                # one row for all
    got = ops.gated_ff(one, w[:F], w[F:])
    assert torch.equal(got, ops.gated_ff(one.contiguous(), w[:F], w[F:]))
    # two weights of different strides
    got = ops.gated_ff(x, wv[:F], w[F:].contiguous())
    within(got, h64, ff_tol(h64, g, u, eg, eu, ops.ACT_SILU, BF))


@pytest.mark.parametrize("M", [1, 20, 70, 260])
def test_gated_ff_keeps_infinities_and_nan_to_their_rows(M):
    F, K = 136, 128
    x, wg, wu = randn(M, K, seed=1, dtype=BF), randn(F, K, seed=2, dtype=BF), randn(F, K, seed=3, dtype=BF)
    clean = ops.gated_ff(x, wg, wu)
    x[0, 3] = float("nan")
    if M > 1:
        x[M - 1, 4] = float("inf")
    h = ops.gated_ff(x, wg, wu)
    assert h[0].isnan().all()
    assert torch.equal(h[1:M - 1], clean[1:M - 1])
    if M > 1:
        ref = x[M - 1:].float()
        g, u = ref @ wg.float().t(), ref @ wu.float().t()
        want = torch.nn.functional.silu(g) * u
        assert torch.equal(h[M - 1:].isnan(), want.isnan()) and torch.equal(h[M - 1:].isinf(), want.isinf())


def quantised(t):
    return ops.quantize_weight_fp8(t)


@pytest.mark.parametrize("act", [ops.ACT_SILU, ops.ACT_GELU])
@pytest.mark.parametrize("M,F,K", [(1, 8, 128), (1, 1040, 256), (3, 72, 128), (16, 136, 384), (17, 520, 128), (33, 64, 256), (65, 136, 512),
                                   (130, 264, 128), (257, 128, 256), (300, 1000, 1152), (2, 8200, 256), (20, 8192, 128), (64, 8216, 384), (1, 24, 8192),
                                   (20, 136, 8320), (48, 8, 8192), (49, 72, 3200), (300, 136, 4096)])
def test_gated_ff_in_8_bits(M, F, K, act):
    x, xs = ops.quantize_rows_fp8(randn(M, K, seed=1, dtype=BF))
    wg, gs = quantised(randn(F, K, seed=2, scale=2 * K ** -0.5))
    wu, us = quantised(randn(F, K, seed=3, scale=K ** -0.5))
    bg, bu = randn(F, seed=4, dtype=BF), randn(F, seed=5, dtype=BF)
    deq = [q.double() * s.double()[:, None] for q, s in ((x, xs), (wg, gs), (wu, us))]
    for b in ((None, None), (bg, bu)):
        h = ops.gated_ff_fp8(x, xs, wg, gs, wu, us, *b, act=act)
        h64, g, u, eg, eu = ff64(*deq, *b, act)
        within(h, h64, ff_tol(h64, g, u, eg + 4 * E32 * g.abs(), eu + 4 * E32 * u.abs(), act, BF))
    ov, buf = embed(torch.zeros(M, F, dtype=BF, device=DEV), 8, 16, fill=7.0)
    assert torch.equal(ops.gated_ff_fp8(x, xs, wg, gs, wu, us, bg, bu, act=act, out=ov), h)
    assert (buf[:, :8] == 7).all() and (buf[:, 8 + F:] == 7).all()


def ff_grad64(dh, x, wg, wu, g, u, act):
    dh, x, wg, wu, g, u = (t.double() for t in (dh, x, wg, wu, g, u))
    a, da = act64(g, act)
    return dh * u * da, dh * a, x, wg, wu


def check_ff_grad(got, dh, x, wg, wu, g, u, act, dtype):
    dx, dwg, dwu, dbg, dbu = got
    M, F, K = dh.shape[0], dh.shape[1], x.shape[1]
    dg, du, x, wg, wu = ff_grad64(dh, x, wg, wu, g, u, act)
    # dg and du: 32-bit arithmetic, then one rounding.  act' = s + v s (1 - s) z' cancels near its zeros (|act'| can be
    # far below its terms, which stay below 1.13 + |v z'| s (1 - s) < 3): an absolute part of 3 |dh u| times the 32-bit errors
    ug = u_of(dtype) * dg.abs() + 3 * 400 * E32 * dh.double().abs() * u.double().abs() + tiny_of(dtype)
    uu = (u_of(dtype) + 400 * E32) * du.abs() + tiny_of(dtype)
    n = 2 * (2 * F + 8) * E32
    want = dg @ wg + du @ wu
    within(dx, want, want.abs() * u_of(dtype) + (ug + n * dg.abs()) @ wg.abs() + (uu + n * du.abs()) @ wu.abs() + tiny_of(dtype), "dx")
    n = 2 * (M + 8) * E32
    for d, e, o, b, name in ((dg, ug, dwg, dbg, "gate"), (du, uu, dwu, dbu, "up")):
        want = d.t() @ x
        within(o, want, want.abs() * u_of(dtype) + (e + n * d.abs()).t() @ x.abs() + tiny_of(dtype), "dw_" + name)
        if b is not None:
            within(b, d.sum(0), d.sum(0).abs() * u_of(dtype) + (e + n * d.abs()).sum(0) + tiny_of(dtype), "db_" + name)


FF_GRAD_SHAPES = [(1, 1, 1), (1, 64, 64), (2, 7, 40), (5, 130, 100), (16, 72, 128), (65, 129, 72), (64, 128, 64), (129, 256, 128),
                  (257, 264, 256), (300, 1000, 1001), (513, 24, 320), (1000, 136, 64), (200, 2056, 576)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act", [ops.ACT_SILU, ops.ACT_GELU])
@pytest.mark.parametrize("M,F,K", FF_GRAD_SHAPES)
def test_gated_ff_gradient(M, F, K, act, dtype):
    dh, x = randn(M, F, seed=1, dtype=dtype), randn(M, K, seed=2, dtype=dtype)
    wg, wu = randn(F, K, seed=3, scale=K ** -0.5, dtype=dtype), randn(F, K, seed=4, scale=K ** -0.5, dtype=dtype)
    g, u = randn(M, F, seed=5, scale=2.0, dtype=dtype), randn(M, F, seed=6, dtype=dtype)
    for bias in (True, False):
        got = ops.gated_ff_backward(dh, x, wg, wu, g, u, act=act, bias=bias)
        assert (got[3] is not None) == bias and (got[4] is not None) == bias
        check_ff_grad(got, dh, x, wg, wu, g, u, act, dtype)
    again = ops.gated_ff_backward(dh, x, wg, wu, g, u, act=act)
    assert all(torch.equal(a, b) for a, b in zip(again[:3], got[:3]))
    if M * F * K > 1 << 20:                                # two roundings of relative rms at most u / sqrt(3) each
        d = ff_grad64(dh, x, wg, wu, g, u, act)
        assert rel_l2(got[0], d[0] @ d[3] + d[1] @ d[4]) < 1.0 * u_of(dtype)
        assert rel_l2(got[1], d[0].t() @ d[2]) < 1.0 * u_of(dtype)


@pytest.mark.parametrize("left,right", [(8, 24), (3, 2)])
def test_gated_ff_gradient_of_strided_operands(left, right):
    M, F, K = 70, 136, 192
    t = [randn(M, F, seed=1, dtype=BF), randn(M, K, seed=2, dtype=BF), randn(F, K, seed=3, dtype=BF), randn(F, K, seed=4, dtype=BF),
         randn(M, F, seed=5, dtype=BF), randn(M, F, seed=6, dtype=BF)]
    got = ops.gated_ff_backward(*[embed(v, left, right)[0] for v in t], bias=True)
    check_ff_grad(got, *t, ops.ACT_SILU, BF)
    t[0] = t[0][:1].expand(M, F)                           # one gradient for all rows, as of a sum over them
    check_ff_grad(ops.gated_ff_backward(*t, bias=True), *t, ops.ACT_SILU, BF)


def test_gated_ff_gradient_far_from_zero_is_finite():
    M, F, K = 4, 64, 64
    g = torch.tensor([-300.0, -90.0, 90.0, 300.0], device=DEV).to(BF)[:, None].expand(M, F).contiguous()
    dh, u, x = torch.ones(M, F, device=DEV, dtype=BF), torch.ones(M, F, device=DEV, dtype=BF), randn(M, K, seed=1, dtype=BF)
    wg, wu = randn(F, K, seed=2, dtype=BF), randn(F, K, seed=3, dtype=BF)
    for act in (ops.ACT_SILU, ops.ACT_GELU):
        check_ff_grad(ops.gated_ff_backward(dh, x, wg, wu, g, u, act=act, bias=True), dh, x, wg, wu, g, u, act, BF)


def test_gated_ff_gradient_against_differences():
    M, F, K = 9, 40, 64
    x, wg, wu = randn(M, K, seed=1, dtype=HF), randn(F, K, seed=2, scale=0.125, dtype=HF), randn(F, K, seed=3, scale=0.125, dtype=HF)
    bg, bu, dh = randn(F, seed=4, dtype=HF), randn(F, seed=5, dtype=HF), randn(M, F, seed=6, dtype=HF)
    for act in (ops.ACT_SILU, ops.ACT_GELU):
        _, g, u = ops.gated_ff(x, wg, wu, bg, bu, act=act, keep=True)
        got = ops.gated_ff_backward(dh, x, wg, wu, g, u, act=act, bias=True)
        at = [t.double() for t in (x, wg, wu, bg, bu)]

        def loss(p):
            return (dh.double() * act64(p[0] @ p[1].t() + p[3], act)[0] * (p[0] @ p[2].t() + p[4])).sum()

        for i, grad in enumerate(got):
            v, d = randn(*grad.shape, seed=10 + i).double(), 1e-5
            num = (loss([t + d * v if j == i else t for j, t in enumerate(at)]) -
                   loss([t - d * v if j == i else t for j, t in enumerate(at)])) / (2 * d)
            # g and u are rounded where they are kept, dg and du where they are handed on, the result at the end: each
            # moves a term by at most a few u of its size; the terms add up to at most sum|dh| (|act'| |u| + |act|) |..|
            a, da = act64(g.double(), act)
            size = (dh.double().abs() * (da.abs() * u.double().abs() + a.abs())).sum() * 3
            assert abs((grad.double() * v).sum() - num) <= 4 * u_of(HF) * size, (act, i)


# ---- together, and the ways they are called -----------------------------------------------------------------------

def layer_inputs(M, D, F, dtype=BF):
    x, r = randn(M, D, seed=1, dtype=dtype), randn(M, D, seed=2, dtype=dtype)
    w = (1 + randn(D, seed=3, scale=0.2)).to(dtype)
    wg, wu, wd = (randn(a, b, seed=s, scale=b ** -0.5, dtype=dtype) for a, b, s in ((F, D, 4), (F, D, 5), (D, F, 6)))
    return x, r, w, wg, wu, wd


@pytest.mark.parametrize("M", [1, 19, 260])
def test_a_block_of_norm_gated_ff_and_residual_linear(M):
    D, F = 256, 640
    x, r, w, wg, wu, wd = layer_inputs(M, D, F)
    n, h = ops.rmsnorm_residual(x, w, r)
    a, gate, up = ops.gated_ff(n, wg, wu, keep=True)
    y = ops.gemm(a, wd, None, epilogue=ops.EPI_RESIDUAL, resid=h)
    h64, n64 = norm64(x, r, w)
    a64 = ff64(n64, wg, wu, None, None, ops.ACT_SILU)[0]
    y64 = a64 @ wd.double().t() + h64
    # n, a, h and y are rounded once each: rms at most u / sqrt(3) relative, the first three through maps of size about one
    assert rel_l2(y, y64) < 2 * u_of(BF)
    # in 8 bits: e4m3 values are within 2^-4, of relative rms at most 2^-4 / sqrt(3) = 3.6 %, in x, the weights and a:
    # three linears' worth of two roundings each, of which the residual takes a part
    q, s, h8 = ops.rmsnorm_residual_fp8(x, w, r)
    assert torch.equal(h8, h)
    a8 = ops.gated_ff_fp8(q, s, *quantised(wg.float()), *quantised(wu.float()))
    aq, as_ = ops.quantize_rows_fp8(a8)
    wq, ws = quantised(wd.float())
    y8 = ops.gemm_fp8(aq, as_, wq, ws, None, epilogue=ops.EPI_RESIDUAL, resid=h)
    assert rel_l2(y8, y64) < 3 * math.sqrt(2) * 0.036
    # and back: the whole block's gradient against differences of its definition in 64 bits
    dy = randn(M, D, seed=9, dtype=BF)
    da = ops.gemm(dy, wd.t().contiguous(), None)
    dn, dwg, dwu, _, _ = ops.gated_ff_backward(da, n, wg, wu, gate, up)
    dx, dw = ops.rmsnorm_residual_backward(dn, h, w, dh=dy)

    def loss(x_, w_):
        h_ = r.double() + x_
        n_ = h_ / torch.sqrt((h_ * h_).mean(1, keepdim=True) + EPS) * w_
        return (dy.double() * (h_ + (act64(n_ @ wg.double().t(), 0)[0] * (n_ @ wu.double().t())) @ wd.double().t())).sum()

    with torch.enable_grad():                              # (other test modules switch it off for the process)
        p = x.double().requires_grad_(), w.double().requires_grad_()
        want = torch.autograd.grad(loss(*p), p)
    # seven roundings between the loss and dx (n, gate and up, da, dg and du, dn, h, dx), of relative rms at most u / sqrt(3)
    assert rel_l2(dx, want[0]) < math.sqrt(9 / 3) * 2 * u_of(BF)
    assert rel_l2(dw, want[1]) < math.sqrt(9 / 3) * 2 * u_of(BF)


@pytest.mark.parametrize("M", [1, 19, 300])
def test_captured_replayed_and_on_another_stream(M):
    D, F = 256, 264
    x, r, w, wg, wu, _ = layer_inputs(M, D, F)
    dh = randn(M, F, seed=8, dtype=BF)
    q8, s8 = ops.quantize_rows_fp8(x)
    w8 = (*quantised(wg.float()), *quantised(wu.float()))

    def step():
        n, h = ops.rmsnorm_residual(x, w, r)
        q, s, _ = ops.rmsnorm_residual_fp8(x, w, r)
        a, g, u = ops.gated_ff(n, wg, wu, keep=True)
        dn, dwg, dwu, dbg, dbu = ops.gated_ff_backward(dh, n, wg, wu, g, u, bias=True)
        dx, dw = ops.rmsnorm_residual_backward(dn, h, w)
        return [n, h, q.view(torch.uint8), s, a, g, u, dn, dwg, dwu, dbg, dbu, dx, dw, ops.gated_ff_fp8(q8, s8, *w8)]

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs, outs = [], []
    for _ in range(2):                                     # two graphs alive at once, captured one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    x0 = x.clone()
    for k in range(3):
        x.copy_(x0 * (1 + k))
        for o in outs:
            for t in o:
                t.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, o)), k


def test_empty_batches():
    x, w, wg = torch.empty(0, 64, dtype=BF, device=DEV), torch.ones(64, dtype=BF, device=DEV), randn(16, 64, dtype=BF)
    y, h = ops.rmsnorm_residual(x, w, x)
    assert y.shape == (0, 64) and h.shape == (0, 64)
    q, s, h = ops.rmsnorm_residual_fp8(x, w, x)
    assert q.shape == (0, 64) and s.shape == (0,)
    dx, dw = ops.rmsnorm_residual_backward(x, x, w)
    assert dx.shape == (0, 64) and (dw == 0).all()
    assert [t.shape[0] for t in ops.gated_ff(x, wg, wg, keep=True)] == [0, 0, 0]
    e = torch.empty(0, 16, dtype=BF, device=DEV)
    dx, dwg, dwu, dbg, dbu = ops.gated_ff_backward(e, x, wg, wg, e, e, bias=True)
    assert dx.shape == (0, 64) and all((t == 0).all() for t in (dwg, dwu, dbg, dbu)) and dwg.shape == (16, 64)


def test_matrices_past_four_gigabytes():
    rows, cols = 140000, 16384                             # 4.6 GB a matrix: byte offsets past 2^32, elements past 2^31
    x = torch.randn(64, cols, device=DEV).to(BF).repeat(rows // 64 + 1, 1)[:rows]
    w = randn(cols, seed=1, dtype=BF)
    y, h = ops.rmsnorm_residual(x, w, x)
    want, _ = ops.rmsnorm_residual(x[:64].contiguous(), w, x[:64].contiguous())
    assert torch.equal(y[rows // 64 * 64 - 64:rows // 64 * 64], want) and torch.equal(y[:64], want)
    dx, _ = ops.rmsnorm_residual_backward(y, x, w, dh=x)
    want, _ = ops.rmsnorm_residual_backward(y[:64], x[:64], w, dh=x[:64])
    assert torch.equal(dx[rows // 64 * 64 - 64:rows // 64 * 64], want)
    del y, h, dx
    wg = randn(64, cols, seed=2, scale=cols ** -0.5, dtype=BF)
    a = ops.gated_ff(x, wg, wg)
    k = rows // 256 * 256
    h64, g, u, eg, eu = ff64(x[:64], wg, wg, None, None, ops.ACT_SILU)      # (fewer rows may be cut into other parts of K)
    for at in (0, k - 64):
        within(a[at:at + 64], h64, ff_tol(h64, g, u, eg, eu, ops.ACT_SILU, BF))
    dh = a[:64].repeat(rows // 64 + 1, 1)[:rows]
    dx, _, _, _, _ = ops.gated_ff_backward(dh, x, wg, wg, a, a)
    want, _, _, _, _ = ops.gated_ff_backward(dh[:256], x[:256], wg, wg, a[:256], a[:256])
    # (a product of another size may be cut into other parts of K: the same sums in another order, rounded once)
    within(dx[k - 256:k], want, want.double().abs() * 2 * u_of(BF) + 1e-3 * want.double().abs().max())


def test_norm_of_more_rows_than_a_launch_takes():
    rows = (1 << 22) + 77
    x = torch.randn(rows, 8, device=DEV).to(BF)
    w = randn(8, seed=1, dtype=BF)
    y, h = ops.rmsnorm_residual(x, w, x)
    h64, y64 = norm64(x, x, w)
    within(y, y64, norm_tol(y64, BF, 8))
    within(h, h64, h64.abs() * (u_of(BF) + 2 * E32))
    q, s, _ = ops.rmsnorm_residual_fp8(x, w, x)
    within(s, y64.abs().amax(1) / 448, y64.abs().amax(1) / 448 * 16 * E32)
    within(q.double() * s.double()[:, None], y64, y64.abs() * 2.0 ** -4 * 1.001 + s.double()[:, None] * 2.0 ** -10)


def test_norm_without_eps_and_of_sums_past_the_types_range():
    x, r = randn(5, 520, seed=1, dtype=HF), randn(5, 520, seed=2, dtype=HF)
    w = randn(520, seed=3, dtype=HF)
    h64, y64 = norm64(x, r, w, eps=0.0)
    y, _ = ops.rmsnorm_residual(x, w, r, eps=0.0)
    within(y, y64, norm_tol(y64, HF, 520))
    x[2], r[2] = x[2] * 0 + 60000, r[2] * 0 + 60000          # h is inf in 16 bits; the norm is taken of the 32-bit sum
    h64, y64 = norm64(x, r, w)
    y, h = ops.rmsnorm_residual(x, w, r)
    assert torch.isinf(h[2]).all() and torch.isfinite(h[[0, 1, 3, 4]]).all()
    within(y, y64, norm_tol(y64, HF, 520))
    z = torch.zeros(3, 520, dtype=HF, device=DEV)            # 0 / 0: NaN, as the formula has it, and only there
    z[1] = x[0]
    y, _ = ops.rmsnorm_residual(z, w, eps=0.0)
    assert torch.isnan(y[0]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[1]).all()


@pytest.mark.parametrize("M,F,K", [(70, 136, 192), (64, 130, 100)])
def test_gated_ff_gradient_of_a_fused_weight_and_of_repeated_rows(M, F, K):
    dh, w = randn(M, F, seed=1, dtype=BF), randn(2 * F, K, seed=2, scale=K ** -0.5, dtype=BF)
    g, u = randn(M, F, seed=3, dtype=BF), randn(M, F, seed=4, dtype=BF)
    x = randn(1, K, seed=5, dtype=BF).expand(M, K)           # one row for all: the gradient of each copy
    gu = torch.cat([g, u], 1)                                # the two projections side by side, as one product leaves them
    got = ops.gated_ff_backward(dh, x, w[:F], w[F:], gu[:, :F], gu[:, F:], bias=True)
    check_ff_grad(got, dh, x, w[:F], w[F:], g, u, ops.ACT_SILU, BF)
    # the same matrix for two arguments, and the same row of it in every place
    got = ops.gated_ff_backward(g, x, w[:F], w[:F], g, g)
    check_ff_grad(got, g, x, w[:F], w[:F], g, g, ops.ACT_SILU, BF)


@pytest.mark.parametrize("M", [3, 130])
def test_calls_that_overlap_on_two_streams(M):
    D, F = 1024, 520                                         # (forward in parts of K, both products of the gradient too)
    sets = []
    for k in range(2):
        x, r, w, wg, wu, _ = layer_inputs(M, D, F)
        sets.append(((x * (k + 1)).contiguous(), r, w, wg, wu, randn(M, F, seed=20 + k, dtype=BF)))

    def step(x, r, w, wg, wu, dh):
        n, h = ops.rmsnorm_residual(x, w, r)
        a, g, u = ops.gated_ff(n, wg, wu, keep=True)
        dn, dwg, dwu, dbg, dbu = ops.gated_ff_backward(dh, n, wg, wu, g, u, bias=True)
        return [n, h, a, g, u, dn, dwg, dwu, dbg, dbu, *ops.rmsnorm_residual_backward(dn, h, w, dh=h)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):                                       # in turn, so that both streams' calls are in flight together
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for o in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(o, want[k]))


def test_leading_dimensions_of_one_and_batches():
    x, r = randn(2, 3, 64, seed=1, dtype=BF), randn(2, 3, 64, seed=2, dtype=BF)
    w, wg = randn(64, seed=3, dtype=BF), randn(24, 64, seed=4, scale=0.125, dtype=BF)
    y, h = ops.rmsnorm_residual(x, w, r)                     # [.., rows, cols] in, [rows, cols] out, as the other norms
    y2, h2 = ops.rmsnorm_residual(x.reshape(6, 64), w, r.reshape(6, 64))
    assert torch.equal(y, y2) and torch.equal(h, h2)
    assert torch.equal(ops.gated_ff(x, wg, wg), ops.gated_ff(x.reshape(6, 64), wg, wg))
    a, g, u = ops.gated_ff(x[:1], wg, wg, keep=True)
    got = ops.gated_ff_backward(a[None], x[:1], wg, wg, g, u)
    assert all(torch.equal(p, q) for p, q in zip(got[:3], ops.gated_ff_backward(a, x[0], wg, wg, g, u)[:3]))


def test_the_widest_blocks():
    F = (1 << 22) + 24                                       # row strides of the output past 2^22
    x, wg = randn(50, 8, seed=1, dtype=BF), randn(F, 8, seed=2, dtype=BF)
    for M in (3, 50):
        h64, g, u, eg, eu = ff64(x[:M], wg, wg, None, None, ops.ACT_SILU)
        within(ops.gated_ff(x[:M], wg, wg), h64, ff_tol(h64, g, u, eg, eu, ops.ACT_SILU, BF))
    cols = (1 << 24) + 9                                     # 32-bit column offsets in the long rows' kernels
    x, w = randn(2, cols, seed=3, dtype=BF), randn(cols, seed=4, dtype=BF)
    h64, y64 = norm64(x, x, w)
    y, h = ops.rmsnorm_residual(x, w, x)
    within(h, h64, h64.abs() * (u_of(BF) + 2 * E32))
    # each lane adds 65537 squares up, then the lanes' sums: half of (65537 + 8) 2^-24 relative, by the root
    within(y, y64, y64.abs() * (u_of(BF) + (65545 / 2 + 8) * E32))


# both products in one launch with dw whole / in parts of K; two launches, dx in parts of K / whole 256 x 128 / 256 x 256 tiles
@pytest.mark.parametrize("M,F,K", [(700, 1400, 392), (2100, 136, 264), (130, 4104, 4096), (1300, 4104, 4096), (2100, 4104, 4096)])
def test_gated_ff_gradient_each_way_its_products_are_cut(M, F, K):
    dh, x = randn(M, F, seed=1, dtype=BF), randn(M, K, seed=2, dtype=BF)
    wg, wu = randn(F, K, seed=3, scale=K ** -0.5, dtype=BF), randn(F, K, seed=4, scale=K ** -0.5, dtype=BF)
    g, u = randn(M, F, seed=5, scale=2.0, dtype=BF), randn(M, F, seed=6, dtype=BF)
    got = ops.gated_ff_backward(dh, x, wg, wu, g, u, bias=True)
    check_ff_grad(got, dh, x, wg, wu, g, u, ops.ACT_SILU, BF)
    again = ops.gated_ff_backward(dh, x, wg, wu, g, u, bias=True)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("cols", [1000, 520])
def test_norm_of_many_short_rows(cols):
    rows = 2050                                              # four rows a workgroup from 2048 rows on, two chunks a lane
    x, r, w = randn(rows, cols, seed=1, dtype=BF), randn(rows, cols, seed=2, dtype=BF), randn(cols, seed=3, dtype=BF)
    h64, y64 = norm64(x, r, w)
    y, h = ops.rmsnorm_residual(x, w, r)
    within(y, y64, norm_tol(y64, BF, cols))
    within(h, h64, h64.abs() * (u_of(BF) + 2 * E32))
    q, s, _ = ops.rmsnorm_residual_fp8(x, w, r)
    amax = y64.abs().amax(1)
    within(s, amax / 448, amax / 448 * (cols / 2 + 10) * E32)
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normal range
    within(q.double() * s.double()[:, None], y64, y64.abs() * (2.0 ** -4 + 2 * (cols / 2 + 10) * E32) + s.double()[:, None] * 2.0 ** -10)


# one launch for both products with several tiles a workgroup, of whole and of ragged tiles, dw whole and in parts
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,F,K", [(512, 4096, 1024), (729, 4304, 1152), (8192, 512, 512), (7777, 520, 392)])
def test_gated_ff_gradient_of_several_tiles_a_workgroup(M, F, K, dtype):
    dh, x = randn(M, F, seed=1, dtype=dtype), randn(M, K, seed=2, dtype=dtype)
    wg, wu = randn(F, K, seed=3, scale=K ** -0.5, dtype=dtype), randn(F, K, seed=4, scale=K ** -0.5, dtype=dtype)
    g, u = randn(M, F, seed=5, scale=2.0, dtype=dtype), randn(M, F, seed=6, dtype=dtype)
    want = ops.gated_ff_backward(dh, x, wg, wu, g, u, act=ops.ACT_GELU)
    check_ff_grad(want, dh, x, wg, wu, g, u, ops.ACT_GELU, dtype)
    for _ in range(4):
        got = ops.gated_ff_backward(dh, x, wg, wu, g, u, act=ops.ACT_GELU)
        assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))


# more tiles than workgroups, in either order of the tiles
@pytest.mark.parametrize("M,F,K", [(3000, 4104, 256), (2816, 3968, 128), (12300, 776, 128)])
def test_gated_ff_of_several_tiles_a_workgroup(M, F, K):
    w = [randn(F, K, seed=s, scale=K ** -0.5) for s in (2, 3)]
    bg, bu = randn(F, seed=4), randn(F, seed=5)
    for dtype in (BF, HF):
        x, wg, wu = randn(M, K, seed=1, dtype=dtype), w[0].to(dtype), w[1].to(dtype)
        b = (bg.to(dtype), bu.to(dtype))
        h64, g, u, eg, eu = ff64(x, wg, wu, *b, ops.ACT_GELU)
        h, gate, up = ops.gated_ff(x, wg, wu, *b, act=ops.ACT_GELU, keep=True)
        within(h, h64, ff_tol(h64, g, u, eg, eu, ops.ACT_GELU, dtype), "h")
        within(gate, g, g.abs() * u_of(dtype) + 2 * eg + tiny_of(dtype), "gate")
        within(up, u, u.abs() * u_of(dtype) + 2 * eu + tiny_of(dtype), "up")
        for _ in range(4):
            assert torch.equal(ops.gated_ff(x, wg, wu, *b, act=ops.ACT_GELU), h)
    x, xs = ops.quantize_rows_fp8(randn(M, K, seed=1, dtype=BF))
    (wg, gs), (wu, us) = quantised(w[0]), quantised(w[1])
    deq = [q.double() * s.double()[:, None] for q, s in ((x, xs), (wg, gs), (wu, us))]
    h64, g, u, eg, eu = ff64(*deq, None, None, ops.ACT_SILU)
    h = ops.gated_ff_fp8(x, xs, wg, gs, wu, us)
    within(h, h64, ff_tol(h64, g, u, eg + 4 * E32 * g.abs(), eu + 4 * E32 * u.abs(), ops.ACT_SILU, BF), "e4m3")
    for _ in range(4):
        assert torch.equal(ops.gated_ff_fp8(x, xs, wg, gs, wu, us), h)


def test_gated_ff_gradient_of_more_weights_than_a_launch_adds_up():
    M, F, K = 2, 1 << 17, 16385                              # dw: 2^32 values and more, in 32-bit parts (an odd width)
    dh, x = randn(M, F, seed=1, dtype=BF), randn(M, K, seed=2, dtype=BF)
    g, u = randn(M, F, seed=5, scale=2.0, dtype=BF), randn(M, F, seed=6, dtype=BF)
    gen = torch.Generator(DEV).manual_seed(3)
    wg, wu = (torch.empty(F, K, dtype=BF, device=DEV).normal_(generator=gen) for _ in range(2))
    dx, dwg, dwu, _, _ = ops.gated_ff_backward(dh, x, wg, wu, g, u)
    dg, du = ff_grad64(dh, x, wg[:1], wu[:1], g, u, ops.ACT_SILU)[:2]
    ug = u_of(BF) * dg.abs() + 3 * 400 * E32 * dh.double().abs() * u.double().abs()
    uu = (u_of(BF) + 400 * E32) * du.abs()
    n = 2 * (M + 8) * E32
    for d, e, o in ((dg, ug, dwg), (du, uu, dwu)):
        for at in (slice(0, 200), slice(F - 300, F)):
            want = d[:, at].t() @ x.double()
            within(o[at], want, want.abs() * u_of(BF) + (e + n * d.abs())[:, at].t() @ x.double().abs(), "dw")
    n = 2 * (2 * F + 8) * E32
    for at in (slice(0, 40), slice(K - 40, K)):
        a, b = wg[:, at].double(), wu[:, at].double()
        want = dg @ a + du @ b
        within(dx[:, at], want, want.abs() * u_of(BF) + (ug + n * dg.abs()) @ a.abs() + (uu + n * du.abs()) @ b.abs(), "dx")


def test_norm_gradient_of_more_wide_rows_than_a_launch_takes():
    rows, cols, step = (1 << 21) + 5, 16392, 8             # dx 69 GB; the inputs' rows overlap each other, 8 values apart
    g = torch.Generator(DEV).manual_seed(1)
    one, two = (torch.randn(rows * step + cols, generator=g, device=DEV).to(BF) for _ in range(2))
    two[step << 21:] *= 1000                               # the rows behind the first launch's count
    h, dy = (t.as_strided((rows, cols), (step, 1)) for t in (one, two))
    w = (1 + randn(cols, seed=3, scale=0.3)).to(BF)
    dx, dw = ops.rmsnorm_residual_backward(dy, h, w)
    for a in (0, (1 << 21) - 4, rows - 7):
        s = slice(a, a + 7)
        dx64, _, tx, _ = norm_grad64(dy[s], h[s], w, None)
        within(dx[s], dx64, dx64.abs() * u_of(BF) + tx * (cols + 16) * E32 * 2, "dx")
    del dx
    sq = torch.cat([torch.zeros(1, device=DEV, dtype=torch.float64), one.double().square().cumsum(0)])
    r = 1 / torch.sqrt((sq[cols::step][:rows] - sq[:-cols:step][:rows]) / cols + EPS)
    at = torch.arange(0, 40, device=DEV)                   # columns in which only the last rows see the factor
    want = (torch.stack([two[c:c + rows * step:step].double() * one[c:c + rows * step:step].double() for c in at.tolist()], 1) * r[:, None]).sum(0)
    # 32-bit sums of 2^15 terms a part err by far less than the last rounding does
    assert rel_l2(dw[at], want) < 1.0 * u_of(BF)


# widths whose partial last chunk begins a wave, so that another wave owns (and in place overwrites) the values in front of it
@pytest.mark.parametrize("cols", [1537, 2561, 8705, 16897, 33281])
def test_ragged_rows_in_place(cols):
    rows = 4100 if cols < 10000 else 300                    # several rows a workgroup in the gradient
    x, r, dy = (randn(rows, cols, seed=i, dtype=BF) for i in (1, 2, 3))
    w = (1 + randn(cols, seed=4, scale=0.3)).to(BF)
    y, h = ops.rmsnorm_residual(x, w, r)
    dx, dw = ops.rmsnorm_residual_backward(dy, h, w, dh=r)
    for _ in range(3):
        a, b = x.clone(), r.clone()
        ops.rmsnorm_residual(a, w, b, out=a, resid_out=b)
        assert torch.equal(a, y) and torch.equal(b, h)
        a, b = x.clone(), r.clone()
        ops.rmsnorm_residual(a, w, b, out=b, resid_out=a)
        assert torch.equal(b, y) and torch.equal(a, h)
        d = r.clone()
        assert torch.equal(ops.rmsnorm_residual_backward(dy, h, w, dh=d, dx=d)[1], dw) and torch.equal(d, dx)
    for at in (0, rows - 20):
        s = slice(at, at + 20)
        h64, y64 = norm64(x[s], r[s], w)
        within(y[s], y64, norm_tol(y64, BF, cols))
        dx64, _, tx, _ = norm_grad64(dy[s], h[s], w, r[s])
        within(dx[s], dx64, dx64.abs() * u_of(BF) + tx * (cols + 16) * E32 * 2, "dx")


# weights of more than 2^31 values: copied into rows (an odd width), and read as they lie but for the last 24 rows.  dx rounds twice
# (dg and du, then itself), each of relative rms at most u / sqrt(3); its 32-bit sums err by far less.
@pytest.mark.parametrize("K", [16385, 16384])
def test_gated_ff_gradient_reads_weights_past_two_to_the_31(K):
    M, F = 2, (1 << 17) + 24
    dh, x = randn(M, F, seed=1, dtype=BF), randn(M, K, seed=2, dtype=BF)
    g, u = randn(M, F, seed=5, scale=2.0, dtype=BF), randn(M, F, seed=6, dtype=BF)
    gen = torch.Generator(DEV).manual_seed(3)
    wg, wu = (torch.empty(F, K, dtype=BF, device=DEV).normal_(generator=gen) for _ in range(2))
    dx, dwg, dwu, _, _ = ops.gated_ff_backward(dh, x, wg, wu, g, u)
    dg, du = ff_grad64(dh, x, wg[:1], wu[:1], g, u, ops.ACT_SILU)[:2]
    at = torch.cat([torch.arange(0, 40), torch.arange(K // 2, K // 2 + 40), torch.arange(K - 40, K)]).to(DEV)
    a, b = wg[:, at].double(), wu[:, at].double()
    want = dg @ a + du @ b
    assert rel_l2(dx[:, at], want) < 1.0 * u_of(BF)
    # the bound sees any of these: nothing at all, one projection alone, a last K tile of 24 rows left out
    for wrong in (0 * want, dg @ a, du @ b, want - dg[:, -24:] @ a[-24:], want - du[:, -24:] @ b[-24:]):
        assert rel_l2(wrong, want) > 1.5 * u_of(BF)
    for d, o in ((dg, dwg), (du, dwu)):
        for rows in (slice(0, 200), slice(F // 2, F // 2 + 200), slice(F - 200, F)):
            assert rel_l2(o[rows], d[:, rows].t() @ x.double()) < 1.0 * u_of(BF)


def test_sums_over_rows_past_four_gigabytes():
    rows, cols, F, far = 140000, 16384, 64, 131072          # row `far` begins 2^31 elements, 2^32 bytes behind the first
    base, grad = randn(64, cols, seed=1, dtype=BF), randn(64, cols, seed=2, dtype=BF)
    x = base.repeat(rows // 64 + 1, 1)[:rows]
    dy = grad.repeat(rows // 64 + 1, 1)[:rows]
    x[far:] *= 4                                           # (the rows repeat every 64: these would not be told apart)
    dy[far:] *= 4
    w = (1 + randn(cols, seed=3, scale=0.3)).to(BF)
    _, dw = ops.rmsnorm_residual_backward(dy, x, w)
    n = torch.stack([((t := f * base.double()) / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)) * f for f in (1.0, 4.0)])
    per = torch.bincount(torch.arange(rows, device=DEV) % 64 + (torch.arange(rows, device=DEV) >= far) * 64).double().view(2, 64, 1)
    want = (n * per * grad.double()).sum((0, 1))
    # parts of 547 rows are added up in 32 bits: 547 2^-24 of the sum of |terms|, six times the sum; then one rounding
    assert rel_l2(dw, want) < 1.0 * u_of(BF)
    assert rel_l2((n[:1] * per[:1] * grad.double()).sum((0, 1)), want) > 10 * u_of(BF)          # (the far rows count)
    del dy
    dh, g, u = randn(rows, F, seed=4, dtype=BF), randn(rows, F, seed=5, dtype=BF), randn(rows, F, seed=6, dtype=BF)
    wg = randn(F, cols, seed=7, scale=cols ** -0.5, dtype=BF)
    _, dwg, dwu, dbg, dbu = ops.gated_ff_backward(dh, x, wg, wg, g, u, bias=True)
    dg, du = ff_grad64(dh, x[:1], wg, wg, g, u, ops.ACT_SILU)[:2]
    for at in (slice(0, 128), slice(cols - 128, cols)):
        xs = x[:, at].double()
        for d, o in ((dg, dwg), (du, dwu)):
            want = d.t() @ xs
            assert rel_l2(o[:, at], want) < 1.0 * u_of(BF)
            assert rel_l2(d[:far].t() @ xs[:far], want) > 10 * u_of(BF)
    for d, o in ((dg, dbg), (du, dbu)):
        assert rel_l2(o, d.sum(0)) < 1.0 * u_of(BF)


@pytest.mark.parametrize("rows,cols", [(5, 72), (33, 1152), (7, 1001), (257, 4096), (3, 5003), (2, 20000), (2, 70000)])
def test_norm_to_8_bits_into_strided_rows_gives_the_same_bytes(rows, cols):
    x, r, w = randn(rows, cols, seed=1, dtype=BF), randn(rows, cols, seed=2, dtype=BF), randn(cols, seed=3, dtype=BF)
    q, s, h = ops.rmsnorm_residual_fp8(x, w, r)
    for left, right in ((16, 16), (5, 6)):
        out = torch.zeros(rows, left + cols + right, dtype=torch.uint8, device=DEV).view(ops.FP8)[:, left:left + cols]
        q2, s2, h2 = ops.rmsnorm_residual_fp8(embed(x, left, right)[0], w, embed(r, left, right)[0], out=out)
        assert q2.data_ptr() == out.data_ptr() and torch.equal(q2.contiguous().view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(s2, s) and torch.equal(h2, h)


# One rounding of relative rms at most u / sqrt(3), and sums that err by a hundredth of that or less: a bound in norm, and one on
# how many values are not the type's nearest.  An error of e before the rounding moves a value to its neighbour with probability
# 2 e / ulp, ulp >= u of the value.  e: 32-bit sums of K / 32 steps and the activation's exponential, 2^-21 of a value of ordinary
# size (K <= 4096); the matrix instructions for e4m3 drop what lies 2^13 below the largest of eight products, 2^-15 of such a
# value; ten times as much for the values that are small by cancellation.
def off_nearest(got, want, dtype):
    return (got != want.to(dtype)).double().mean().item()


FF_NORM_SHAPES = [(1, 4096, 1024), (16, 1040, 512), (33, 264, 520), (40, 72, 2048), (48, 8208, 256), (64, 520, 256), (129, 256, 640),
                  (300, 136, 4096), (300, 1000, 1152), (600, 8192, 256)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,F,K", FF_NORM_SHAPES)
def test_gated_ff_in_norm(M, F, K, dtype):
    x, wg, wu = randn(M, K, seed=1, dtype=dtype), randn(F, K, seed=2, scale=2 * K ** -0.5, dtype=dtype), randn(F, K, seed=3, scale=K ** -0.5, dtype=dtype)
    for act in (ops.ACT_SILU, ops.ACT_GELU):
        h64, g, u, _, _ = ff64(x, wg, wu, None, None, act)
        got = ops.gated_ff(x, wg, wu, act=act, keep=True)
        for o, want in zip(got, (h64, g, u)):
            assert rel_l2(o, want) < 0.6 * u_of(dtype)
            assert off_nearest(o, want, dtype) < 10 * 2 * 2.0 ** -21 / u_of(dtype)


@pytest.mark.parametrize("M,F,K", [(m, f, k) for m, f, k in FF_NORM_SHAPES if k % 128 == 0])
def test_gated_ff_in_8_bits_in_norm(M, F, K):
    x, xs = ops.quantize_rows_fp8(randn(M, K, seed=1, dtype=BF))
    (wg, gs), (wu, us) = quantised(randn(F, K, seed=2, scale=2 * K ** -0.5)), quantised(randn(F, K, seed=3, scale=K ** -0.5))
    deq = [q.double() * s.double()[:, None] for q, s in ((x, xs), (wg, gs), (wu, us))]
    for act in (ops.ACT_SILU, ops.ACT_GELU):
        h64 = ff64(*deq, None, None, act)[0]
        h = ops.gated_ff_fp8(x, xs, wg, gs, wu, us, act=act)
        assert rel_l2(h, h64) < 0.6 * u_of(BF)
        assert off_nearest(h, h64, BF) < 10 * 2 * 2.0 ** -15 / u_of(BF)


# e4m3 products are cut, towards zero, at 2^-13 of the binade of the largest of eight neighbours (k = 8 i .. 8 i + 7): an error of
# up to 7 2^-13 of it for every eight, beside the 32-bit sums'
@pytest.mark.parametrize("M", [3, 40, 70])
def test_gated_ff_in_8_bits_of_products_that_cancel(M):
    K, F = 1024, 8
    big = torch.arange(K, device=DEV) % 8 == 0
    x = torch.where(big, 16.0, 0.234375).expand(M, K).contiguous()
    wu = torch.where(big, 16.0 - 32.0 * (torch.arange(K, device=DEV) // 8 % 2), 0.234375).expand(F, K).contiguous()
    wg = torch.zeros(F, K, device=DEV)
    wg[:, 0] = 4.0                                         # g = 64: act(g) = 64 in 32 bits
    h64, _, u, _, eu = ff64(x, wg, wu, None, None, ops.ACT_SILU)
    cut = 7 * 2.0 ** -13 * 256 * (K / 8)
    one = torch.ones(max(M, F), device=DEV)
    h = ops.gated_ff_fp8(x.to(ops.FP8), one[:M], wg.to(ops.FP8), one[:F], wu.to(ops.FP8), one[:F])
    within(h, h64, h64.abs() * u_of(BF) + 64 * (cut + eu) * (1 + u_of(BF)))
    assert cut < u.min()                                   # (the sum of what is small is seen)


# ---- at the limits that the entry points document ------------------------------------------------------------------

def test_norm_of_the_most_columns():
    cols = 1 << 28
    g = torch.Generator(DEV).manual_seed(1)
    x, w = torch.randn(1, cols, generator=g, device=DEV).to(BF), torch.randn(cols, generator=g, device=DEV).to(BF)
    y, h = ops.rmsnorm_residual(x, w, x)
    r = 1 / math.sqrt(sum((2 * v.double()).square().sum().item() for v in x[0].split(1 << 24)) / cols + EPS)
    for at in (slice(0, 1000), slice(cols // 2 - 500, cols // 2 + 500), slice(cols - 1000, cols)):
        assert torch.equal(h[0, at], 2 * x[0, at])
        # 2^20 squares a lane: their sum's roundings stay far below the output's
        assert rel_l2(y[0, at], 2 * x[0, at].double() * r * w[at].double()) < 1.0 * u_of(BF)
    q, s, _ = ops.rmsnorm_residual_fp8(x, w, x)
    for at in (slice(0, 1000), slice(cols - 1000, cols)):
        # half a step of e4m3, 2^-4 of a value (2^-10 of the scale below the normal range)
        want = 2 * x[0, at].double() * r * w[at].double()
        within(q[0, at].double() * s.double(), want, want.abs() * (2.0 ** -4 + 1e-3) + s.double() * 2.0 ** -10)
    dx, dw = ops.rmsnorm_residual_backward(y, h, w)
    dot = sum((a.double() * b.double() * c.double()).sum().item() for a, b, c in zip(y[0].split(1 << 24), w.split(1 << 24), h[0].split(1 << 24)))
    for at in (slice(0, 1000), slice(cols - 1000, cols)):
        hs, ys, ws = h[0, at].double(), y[0, at].double(), w[at].double()
        assert rel_l2(dw[at], ys * hs * r) < 1.0 * u_of(BF)
        assert rel_l2(dx[0, at], r * (ys * ws - hs * r * r * dot / cols)) < 1.0 * u_of(BF)


@pytest.mark.parametrize("M,F,K", [(1, 1 << 27, 8), (3, 40, (1 << 24) + 24), (49, 40, (1 << 20) - 64), (49, 24, (1 << 20) - 65), ((1 << 20) + 1, 16, 64)])
def test_gated_ff_at_its_limits(M, F, K):
    g = torch.Generator(DEV).manual_seed(1)
    x, wg, wu = (torch.randn(r, K, generator=g, device=DEV).mul_(K ** -0.5 if i else 1).to(BF) for i, r in enumerate((M, F, F)))
    h = ops.gated_ff(x, wg, wu)
    rows, cols = sorted({0, M // 2, M - 1}), torch.tensor(sorted({0, min(F - 1, 7), F // 2, F - 2, F - 1}), device=DEV)
    h64, gt, up, eg, eu = ff64(x[rows], wg[cols], wu[cols], None, None, ops.ACT_SILU)
    # (K roundings of a sum's terms grow as their root: 2^-24 sqrt(K) of the sum of |terms| is a hundred times what is met)
    few = min(1.0, 16 * K ** -0.5)
    within(h[rows][:, cols], h64, ff_tol(h64, gt, up, eg * few, eu * few, ops.ACT_SILU, BF))


@pytest.mark.parametrize("M,F,K", [((1 << 20) - 64, 16, 64), ((1 << 20) - 65, 24, 40), (3, (1 << 20) - 64, 64), (3, 24, (1 << 20) - 64)])
def test_gated_ff_gradient_at_its_limits(M, F, K):
    gen = torch.Generator(DEV).manual_seed(1)
    dh, g, u = (torch.randn(M, F, generator=gen, device=DEV).to(BF) for _ in range(3))
    x = torch.randn(M, K, generator=gen, device=DEV).to(BF)
    wg, wu = (torch.randn(F, K, generator=gen, device=DEV).to(BF) for _ in range(2))
    dx, dwg, dwu, dbg, dbu = ops.gated_ff_backward(dh, x, wg, wu, g, u, bias=True)
    dg, du = ff_grad64(dh, x[:1], wg[:1], wu[:1], g, u, ops.ACT_SILU)[:2]
    rows = torch.cat([torch.arange(0, min(M, 200)), torch.arange(max(0, M - 200), M)]).unique().to(DEV)
    cols = torch.cat([torch.arange(0, min(K, 200)), torch.arange(max(0, K - 200), K)]).unique().to(DEV)
    want = dg[rows] @ wg[:, cols].double() + du[rows] @ wu[:, cols].double()
    assert rel_l2(dx[rows][:, cols], want) < 1.0 * u_of(BF)
    inner = torch.cat([torch.arange(0, min(F, 200)), torch.arange(max(0, F - 200), F)]).unique().to(DEV)
    for d, o, b in ((dg, dwg, dbg), (du, dwu, dbu)):
        assert rel_l2(o[inner][:, cols], d[:, inner].t() @ x[:, cols].double()) < 1.0 * u_of(BF)
        assert rel_l2(b, d.sum(0)) < 1.0 * u_of(BF)


def test_gated_ff_of_rows_far_apart_and_of_rows_that_overlap():
    M, F, K = 64, 24, 64
    x, w = randn(M, K, seed=1, dtype=BF), randn(2 * F, K, seed=2, scale=K ** -0.5, dtype=BF)
    far = torch.zeros(2 * F, (1 << 22) + 16, dtype=BF, device=DEV)           # a stride that the wide reads' offsets do not hold
    far[:, :K] = w
    wv = far[:, :K]
    near = randn(M * 8 + K, seed=3, dtype=BF).as_strided((M, K), (8, 1))
    dh, g, u = (randn(M, F, seed=i, dtype=BF) for i in (4, 5, 6))
    for rows in (3, M):
        for a in (x[:rows], near[:rows]):
            h64, gt, up, eg, eu = ff64(a, w[:F], w[F:], None, None, ops.ACT_SILU)
            within(ops.gated_ff(a, wv[:F], wv[F:]), h64, ff_tol(h64, gt, up, eg, eu, ops.ACT_SILU, BF))
            t = (dh[:rows], a, wv[:F], wv[F:], g[:rows], u[:rows])
            check_ff_grad(ops.gated_ff_backward(*t, bias=True), *t, ops.ACT_SILU, BF)


@pytest.mark.parametrize("cols", [64, 1537, 4096, 20000, 70000])
def test_norm_to_8_bits_with_the_sum_in_place(cols):
    x, r, w = randn(9, cols, seed=1, dtype=BF), randn(9, cols, seed=2, dtype=BF), randn(cols, seed=3, dtype=BF)
    q, s, h = ops.rmsnorm_residual_fp8(x, w, r)
    for into in (0, 1):
        a = [x.clone(), r.clone()]
        q2, s2, h2 = ops.rmsnorm_residual_fp8(a[0], w, a[1], resid_out=a[into])
        assert h2 is a[into] and torch.equal(h2, h) and torch.equal(s2, s) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))
