"""The training operators on the GPU against float64 restatements of their
formulas: layer norm and its gradient, the vocabulary cross entropy and its
gradient, the orthogonalised update, alone and as a training step uses them.

Tolerances are elementwise bounds from the arithmetic, computed in float64
beside each reference value (u = 2^-24, a rounding to type t is off by at most
finfo(t).eps / 2 of the value):

* norm: sums of a row take at most 16 serial and 10 tree additions, the
  variance and the reciprocal root a few more operations: 32 u of the summed
  magnitudes;
* tensor-core sums add by truncation, at most 2 u of the running magnitude per
  16-k step, so (steps + 2) 2 u of sum |a||b|; two-piece float32 operands are
  2^-22 off each and drop a product below 2^-22;
* exponentials: 2^-22 of the value and the error of the argument;
* the orthogonalised update: a step's relative error passes to the next with a
  factor of at most 2 near 1 (x p'(x) / p(x)) and 1 for small singular values,
  cancellation in the polynomial multiplies a product's error by at most 14:
  about 100 times the 2^-21 of a product, 5e-5."""

import pytest
import torch

import model_b200 as mb
from model_b200 import _lib as L

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half of the smallest subnormal: what rounding a tiny result may lose."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    nan = torch.isnan(want)
    assert torch.isfinite(torch.as_tensor(tol, device=want.device).expand(want.shape)[~nan]).all(), what
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaNs differ"
    bad = ((got - want).abs() > tol) & ~nan
    assert not bad.any(), f"{what}: {int(bad.sum())} entries off, worst {float(((got - want).abs() / tol)[bad].max())} bounds"


# ---- layer norm -----------------------------------------------------------------------
def norm_ref(x, scale, bias, eps):
    v = x.double()
    mean = v.mean(-1, keepdim=True)
    rstd = ((v - mean) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    xhat = (v - mean) * rstd
    lead = 32 * U * (1 + v.abs().mean(-1, keepdim=True) * rstd)     # error of the centred, scaled value
    y = xhat * scale.double() + bias.double()
    tol = scale.double().abs() * (lead + 32 * U * xhat.abs()) + 4 * U * bias.double().abs()
    return y, tol, xhat, rstd, lead


def norm_case(M, d, t, seed=0, spread=True):
    g = gen(seed)
    x = torch.randn(M, d, device="cuda", generator=g)
    if spread:
        x = x * (0.1 + 3 * torch.rand(M, 1, device="cuda", generator=g)) + 2 * torch.randn(M, 1, device="cuda", generator=g)
    r, dy, dr = (torch.randn(M, d, device="cuda", generator=g) for _ in range(3))
    scale, bias = 1 + 0.3 * torch.randn(d, device="cuda", generator=g), 0.2 * torch.randn(d, device="cuda", generator=g)
    return x.to(t), r.to(t), scale, bias, dy.to(t), dr.to(t)


def check_norm_backward(dx, dp, dy, x, scale, dr, eps, t):
    _, _, xhat, rstd, lead = norm_ref(x, scale, scale, eps)
    g, d = dy.double(), x.shape[-1]
    gy = g * scale.double()
    c1, c2 = gy.mean(-1, keepdim=True), (gy * xhat).mean(-1, keepdim=True)
    want = rstd * (gy - c1 - xhat * c2)
    mag = rstd * (gy.abs() + gy.abs().mean(-1, keepdim=True)
                  + xhat.abs() * (gy * xhat).abs().mean(-1, keepdim=True))
    # xhat's own error enters c2 and the last term
    tol = 64 * U * mag + rstd * lead * (c2.abs() + xhat.abs() * gy.abs().mean(-1, keepdim=True))
    if dr is not None:
        want = want + dr.double()
    within(dx, want, tol + half_step(t) * want.abs() + tiny(t) + 2 * U * want.abs(), "dx")
    M = x.reshape(-1, d).shape[0]
    flat = lambda a: a.reshape(-1, d)  # noqa: E731
    within(dp["bias"], flat(g).sum(0), (M + 64) * U * flat(g).abs().sum(0), "dbias")
    ph = flat(g * xhat)
    within(dp["scale"], ph.sum(0), (M + 96) * U * ph.abs().sum(0) + (flat(g.abs() * lead)).sum(0), "dscale")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,d", [(1, 1), (1, 7), (3, 2), (5, 33), (2, 64), (257, 100), (64, 256), (1000, 520), (31, 1000),
                                 (129, 1024), (7, 4096), (3, 5001), (2, 16384)])
def test_norm_forward_and_backward(M, d, t):
    x, r, scale, bias, dy, dr = norm_case(M, d, t, seed=M + d)
    y = mb.layer_norm(x, scale, bias)
    want, tol, *_ = norm_ref(x, scale, bias, 1e-6)
    within(y, want, tol + half_step(t) * want.abs() + tiny(t), "y")
    y2, s = mb.layer_norm(x, scale, bias, residual=r, eps=1e-5)
    assert torch.equal(s, (x.float() + r.float()).to(t))
    want, tol, *_ = norm_ref(s, scale, bias, 1e-5)
    within(y2, want, tol + half_step(t) * want.abs() + tiny(t), "y of the sum")
    dx, dp = mb.layer_norm_backward(dy, s, scale, eps=1e-5)
    check_norm_backward(dx, dp, dy, s, scale, None, 1e-5, t)
    dx, dp = mb.layer_norm_backward(dy, s, scale, dresidual=dr, eps=1e-5)
    check_norm_backward(dx, dp, dy, s, scale, dr, 1e-5, t)


# packed rows that begin inside of a 16-byte vector: fewer and more of them than blocks, one or several vectors a thread
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,d", [(1, 513), (2, 515), (9, 516), (3001, 514), (2003, 1001), (1501, 2047), (1200, 2498), (700, 4097),
                                 (310, 8201), (5, 9001), (3, 16381), (2, 16383)])
def test_norm_rows_between_vectors(M, d, t):
    x, r, scale, bias, dy, dr = norm_case(M, d, t, seed=M + d)
    y, s = mb.layer_norm(x, scale, bias, residual=r, eps=1e-5)
    assert torch.equal(s, (x.float() + r.float()).to(t))
    want, tol, *_ = norm_ref(s, scale, bias, 1e-5)
    within(y, want, tol + half_step(t) * want.abs() + tiny(t), "y")
    within(mb.layer_norm(s, scale, bias, eps=1e-5), want, tol + half_step(t) * want.abs() + tiny(t), "y alone")
    dx, dp = mb.layer_norm_backward(dy, s, scale, dresidual=dr, eps=1e-5, check=True)
    check_norm_backward(dx, dp, dy, s, scale, dr, 1e-5, t)
    dx, dp = mb.layer_norm_backward(dy, s, scale, eps=1e-5)
    check_norm_backward(dx, dp, dy, s, scale, None, 1e-5, t)


@pytest.mark.parametrize("t", TYPES)
def test_norm_rows_between_vectors_keep_to_themselves(t):
    M, d = 1500, 1003
    x, _, scale, bias, dy, _ = norm_case(M, d, t, seed=21)
    clean, (cdx, _) = mb.layer_norm(x, scale, bias), mb.layer_norm_backward(dy, x, scale)
    bad = list(range(1, M, 7))
    x[bad, 0], x[bad, d - 1], dy[bad, d - 1] = float("nan"), float("inf"), float("nan")
    y, (dx, _) = mb.layer_norm(x, scale, bias), mb.layer_norm_backward(dy, x, scale)
    keep = [i for i in range(M) if i % 7 != 1]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cdx[keep])
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).all()
    # what is around the rows stays as it was
    room = torch.full((M * d + 64,), 7.0, device="cuda").to(t)
    inner = room[32:32 + M * d].view(M, d)
    inner.copy_(cdx)
    before = room.clone()
    assert torch.equal(mb.layer_norm(inner, scale, bias), mb.layer_norm(cdx, scale, bias)) and torch.equal(room, before)


@pytest.mark.parametrize("t", TYPES)
def test_norm_many_rows(t):
    x, _, scale, bias, dy, _ = norm_case(20011, 48, t, seed=5)
    dx, dp = mb.layer_norm_backward(dy, x, scale)
    check_norm_backward(dx, dp, dy, x, scale, None, 1e-6, t)


@pytest.mark.parametrize("t", TYPES)
def test_norm_strided_and_shifted_rows(t):
    x, r, scale, bias, dy, dr = norm_case(65, 96, t, seed=3)
    wide = torch.empty(65, 3 * 96 + 1, dtype=t, device="cuda")
    wide[:, 1:97], wide[:, 97:193], wide[:, 193:289] = x, dy, dr
    xs, gs, ds = wide[:, 1:97], wide[:, 97:193], wide[:, 193:289]       # odd stride and odd offset
    # single elements instead of 16 bytes a thread: another order of the row's sums
    want, tol, *_ = norm_ref(x, scale, bias, 1e-6)
    within(mb.layer_norm(xs, scale, bias), want, tol + half_step(t) * want.abs() + tiny(t), "y")
    dx, dp = mb.layer_norm_backward(gs, xs, scale, dresidual=ds)
    check_norm_backward(dx, dp, dy, x, scale, dr, 1e-6, t)
    x3 = x.reshape(5, 13, 96)
    assert torch.equal(mb.layer_norm(x3, scale, bias), mb.layer_norm(x, scale, bias).reshape(5, 13, 96))
    xt = x3.transpose(0, 1)                                               # a layout that has to be copied
    assert torch.equal(mb.layer_norm(xt, scale, bias), mb.layer_norm(x, scale, bias).reshape(5, 13, 96).transpose(0, 1))


def test_norm_constant_rows_and_large_means():
    # a constant row: xhat is 0, y the bias, and its gradient cancels
    x = torch.full((4, 256), 3.0, device="cuda")
    scale, bias = torch.rand(256, device="cuda") + 0.5, torch.randn(256, device="cuda")
    assert torch.equal(mb.layer_norm(x, scale, bias), bias.expand(4, 256))
    one = torch.ones(3, 1, device="cuda")
    dx, dp = mb.layer_norm_backward(torch.randn(3, 1, device="cuda"), one, torch.full((1,), 1.3, device="cuda"))
    assert torch.equal(dx, torch.zeros_like(dx)) and float(dp["scale"]) == 0.0
    # a mean 10^4 times the spread leaves the centred variance its digits
    g = gen(9)
    x = 1e4 + torch.randn(16, 512, device="cuda", generator=g)
    one, zero = torch.ones(512, device="cuda"), torch.zeros(512, device="cuda")
    want, tol, *_ = norm_ref(x, one, zero, 1e-6)
    within(mb.layer_norm(x, one, zero), want, tol + U * want.abs(), "y")


def test_norm_nan_and_infinity_stay_in_their_rows():
    x, _, scale, bias, dy, _ = norm_case(40, 200, F32, seed=8)
    clean = mb.layer_norm(x, scale, bias)
    x[3, 5], x[17, 199] = float("nan"), float("inf")
    y = mb.layer_norm(x, scale, bias)
    keep = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all() and torch.isnan(y[17]).all()


def test_norm_empty():
    s = torch.ones(16, device="cuda")
    e = torch.empty(0, 16, device="cuda")
    assert mb.layer_norm(e, s, s).shape == (0, 16)
    dx, dp = mb.layer_norm_backward(e, e, s)
    assert dx.shape == (0, 16) and torch.equal(dp["scale"], torch.zeros_like(s)) and not dp["bias"].any()


def test_norm_gradient_against_differences():
    # sum(dy * y) along a direction: the third derivative of a normalised row
    # along a unit step is below 100 (|d xhat| grows with rstd <= 2 here), so
    # the central difference is off by at most 100 h^2 / 6 |dy| |scale|, plus
    # the roundings of two float32 sums over 2 h
    x, _, scale, bias, dy, _ = norm_case(6, 64, F32, seed=21, spread=False)
    v = torch.randn(6, 64, device="cuda", generator=gen(4)) / 8
    h = 1e-2
    f = lambda z: float((dy.double() * mb.layer_norm(z, scale, bias).double()).sum())  # noqa: E731
    got = (f(x + h * v) - f(x - h * v)) / (2 * h)
    dx, dp = mb.layer_norm_backward(dy, x, scale)
    mag = float((dy.abs() * scale.abs()).sum())
    assert abs(got - float((dx.double() * v.double()).sum())) <= 100 * h * h / 6 * mag + 64 * U * 4 * mag / h


def test_norm_offsets_beyond_32_bits():
    rows, d = (1 << 20) + 3, 2056                       # 2^31 + 8.4e6 entries
    x = torch.empty(rows, d, dtype=BF16, device="cuda")
    x[-300:] = torch.randn(300, d, device="cuda", generator=gen(2)).to(BF16)
    x[:-300] = 0
    scale, bias = torch.rand(d, device="cuda") + 0.5, torch.randn(d, device="cuda")
    y = mb.layer_norm(x, scale, bias)
    assert torch.equal(y[-300:], mb.layer_norm(x[-300:].clone(), scale, bias))
    del y
    dx, dp = mb.layer_norm_backward(x, x, scale)
    dx1, dp1 = mb.layer_norm_backward(x[-300:].clone(), x[-300:].clone(), scale)
    assert torch.equal(dx[-300:], dx1)
    # the zero rows add nothing: only the order of the sums differs
    g = x[-300:].double()
    xh = norm_ref(x[-300:], scale, bias, 1e-6)[2]
    within(dp["scale"], dp1["scale"].double(), 700 * U * (g * xh).abs().sum(0), "dscale")


# ---- cross entropy ----------------------------------------------------------------------
def loss_case(T, d, V, t, seed=0, gap=0):
    g = gen(seed)
    w = (torch.randn(V, d, device="cuda", generator=g) * (2.0 / d ** 0.5)).to(t)
    h = torch.randn(T, d, device="cuda", generator=g).to(t)
    y = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    if gap:
        y[::gap] = -100
    dl = (0.2 + torch.rand(T, device="cuda", generator=g)) / max(T, 1)
    return h, w, y, dl


class LossRef:
    """float64 values and elementwise bounds."""

    def __init__(self, h, w, y, dl=None, dlse=None, ignore=-100):
        t, (T, d), V = h.dtype, h.shape, w.shape[0]
        f32 = t == F32
        H, W = h.double(), w.double()
        z, zm = H @ W.T, H.abs() @ W.abs().T
        steps = (3 if f32 else 1) * ((d + 15) // 16) + 2
        dz = zm * (steps * 2 * U + (3 * 2.0 ** -22 if f32 else 0))       # error of a logit
        if f32:   # entries far below their matrix's largest have an absolute error instead
            dz = dz + 2.0 ** -38 * (h.double().abs().max() * W.abs().sum(1)[None] + w.double().abs().max()
                                    * H.abs().sum(1)[:, None])
        self.lse = torch.logsumexp(z, 1)
        p = (z - self.lse[:, None]).exp()
        # argument roundings, 2^-22 an exponential, and the order of the sum
        arg = 4 * U * (z.abs() + self.lse.abs()[:, None]) + 2.0 ** -21
        self.lse_tol = (p * (dz + arg)).sum(1) + (V / 32 + 64) * U + 6 * U * self.lse.abs() + dz.max(1).values * 2.0 ** -10
        on = y != ignore
        at = y.long().clamp(0, V - 1)[:, None]
        zt = z.gather(1, at)[:, 0]
        self.loss = torch.where(on, self.lse - zt, torch.zeros_like(zt))
        self.loss_tol = self.lse_tol + dz.gather(1, at)[:, 0] + 4 * U * (self.lse.abs() + zt.abs())
        if dl is None:
            return
        g = torch.where(on, dl.double(), torch.zeros_like(zt))
        q = g + (dlse.double() if dlse is not None else 0)
        one = torch.zeros_like(p).scatter_(1, at, on.double()[:, None])
        grad = p * q[:, None] - one * g[:, None]
        mag = p * q.abs()[:, None] + one * g.abs()[:, None]
        et = 2.0 ** -21 if f32 or T <= 128 and t == F16 else 2.0 ** -16 if T <= 128 else half_step(t)
        dg = p * q.abs()[:, None] * (dz + self.lse_tol[:, None] + arg) + mag * (et + 4 * U)
        if t != BF16:
            dg = dg + 2.0 ** -38 * torch.stack([q.abs().max(), g.abs().max()]).max()
        self.dh, self.dw = grad @ W, grad.T @ H
        k = lambda n: (((3 if f32 else 1) * ((n + 15) // 16)) + 8) * 2 * U + (2.0 ** -20 if f32 else 0)  # noqa: E731
        self.dh_tol = dg @ W.abs() + k(V) * (mag @ W.abs()) + half_step(t) * self.dh.abs() + tiny(t)
        self.dw_tol = dg.T @ H.abs() + k(T) * (mag.T @ H.abs()) + half_step(t) * self.dw.abs() + tiny(t)
        if f32:
            self.dh_tol = self.dh_tol + 2.0 ** -38 * w.double().abs().max() * mag.sum(1)[:, None]
            self.dw_tol = self.dw_tol + 2.0 ** -38 * h.double().abs().max() * mag.sum(0)[:, None]

    def check(self, loss, lse, dh=None, dw=None):
        within(lse, self.lse, self.lse_tol, "lse")
        within(loss, self.loss, self.loss_tol, "loss")
        if dh is not None:
            within(dh, self.dh, self.dh_tol, "dh")
            within(dw, self.dw, self.dw_tol, "dw")


def run_loss(h, w, y, dl, dlse=None, ignore=-100, check=False):
    loss, lse = mb.linear_cross_entropy(h, w, y, ignore_index=ignore, check=check)
    dh, dw = mb.linear_cross_entropy_backward(h, w, y, lse, dl, dlse=dlse, ignore_index=ignore, check=check)
    return loss, lse, dh, dw


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,d,V", [(1, 1, 1), (1, 64, 2), (2, 8, 300), (7, 33, 129), (128, 64, 256), (129, 72, 257),
                                   (300, 100, 1000), (257, 256, 511), (256, 130, 1024), (40, 640, 2003), (513, 65, 4099)])
def test_loss_and_gradient(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + d + V, gap=5 if T > 4 else 0)
    LossRef(h, w, y, dl).check(*run_loss(h, w, y, dl, check=True))


@pytest.mark.parametrize("T", [1, 3, 16, 17, 24, 25])
@pytest.mark.parametrize("d,V", [(4, 127), (36, 128), (100, 129), (256, 1000), (1500, 300)])
def test_loss_of_few_float32_tokens(T, d, V):
    h, w, y, dl = loss_case(T, d, V, F32, seed=T + d, gap=4 if T > 4 else 0)
    LossRef(h, w, y).check(*mb.linear_cross_entropy(h, w, y, check=True))
    wide = torch.zeros(V, d + 8, device="cuda")                   # rows 16 bytes apart, and rows that are not
    wide[:, 4:d + 4] = w
    LossRef(h, w, y).check(*mb.linear_cross_entropy(h, wide[:, 4:d + 4], y, check=True))
    wide[:, 3:d + 3] = w
    LossRef(h, w, y).check(*mb.linear_cross_entropy(h, wide[:, 3:d + 3], y, check=True))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T", [1, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("d,V", [(1, 1), (7, 63), (36, 65), (513, 129), (1024, 300), (1025, 130), (50, 21001)])
def test_loss_gradient_of_few_tokens(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + d, gap=3 if T > 4 else 0)
    dlse = 0.1 * torch.randn(T, device="cuda", generator=gen(2))
    LossRef(h, w, y, dl, dlse).check(*run_loss(h, w, y, dl, dlse))
    wide = torch.zeros(V, d + 3, dtype=t, device="cuda")                    # rows from odd addresses
    wide[:, 1:d + 1] = w
    LossRef(h, w, y, dl).check(*run_loss(h, wide[:, 1:d + 1], y, dl))


@pytest.mark.parametrize("t", TYPES)
def test_loss_gradient_of_few_tokens_special(t):
    h, w, y, dl = loss_case(6, 40, 500, t, seed=3)
    _, lse = mb.linear_cross_entropy(h, w, y)
    dh, dw = mb.linear_cross_entropy_backward(h, w, y, lse, dl)
    z = y.clone()
    z[2] = -100                                                             # its dloss and lse are not read
    nan = torch.full_like(dl, float("nan"))
    a = mb.linear_cross_entropy_backward(h, w, z, torch.where(z < 0, nan, lse), torch.where(z < 0, nan, dl))
    b = mb.linear_cross_entropy_backward(h, w, y, lse, torch.where(z < 0, torch.zeros_like(dl), dl))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[0][2].any()
    z[2] = 500                                                              # out of range: loud, no gradient
    c = mb.linear_cross_entropy_backward(h, w, z, lse, dl)
    assert torch.equal(c[0], a[0]) and torch.equal(c[1], a[1])
    with pytest.raises(L.DeviceError, match="27"):
        mb.linear_cross_entropy_backward(h, w, z, lse, dl, check=True)
    z[:] = 7                                                                # one entry for all
    _, ls = mb.linear_cross_entropy(h, w, z)
    d2, w2 = mb.linear_cross_entropy_backward(h, w, z, ls, dl)
    LossRef(h, w, z, dl).check(*mb.linear_cross_entropy(h, w, z), d2, w2)
    bad = h.clone()
    bad[1, 3] = float("nan")                                                # stays in its token's dh; dW of all entries
    _, ls = mb.linear_cross_entropy(bad, w, y)
    d3, w3 = mb.linear_cross_entropy_backward(bad, w, y, ls, dl)
    keep = [0, 2, 3, 4, 5]
    assert torch.equal(d3[keep], dh[keep]) and torch.isnan(d3[1]).all() and torch.isnan(w3).all()


@pytest.mark.parametrize("t", TYPES)
def test_loss_gradient_of_lse_and_weighted_tokens(t):
    h, w, y, dl = loss_case(200, 96, 700, t, seed=4, gap=3)
    dl = dl * torch.randint(-1, 2, (200,), device="cuda")        # zero and negative weights
    dlse = 0.01 * torch.randn(200, device="cuda", generator=gen(1))
    LossRef(h, w, y, dl, dlse).check(*run_loss(h, w, y, dl, dlse))


@pytest.mark.parametrize("t", TYPES)
def test_loss_strided_operands(t):
    h, w, y, dl = loss_case(150, 80, 400, t, seed=6)
    hw = torch.zeros(150, 200, dtype=t, device="cuda")
    ww = torch.zeros(400, 163, dtype=t, device="cuda")           # rows TMA cannot address
    hw[:, 8:88], ww[:, 3:83] = h, w
    hv, wv = hw[:, 8:88], ww[:, 3:83]
    ref = LossRef(h, w, y, dl)
    ref.check(*run_loss(hv, wv, y.to(torch.int64), dl))
    h3 = h.reshape(3, 50, 80)
    loss, lse = mb.linear_cross_entropy(h3, w, y.reshape(3, 50))
    assert loss.shape == (3, 50)
    dh, dw = mb.linear_cross_entropy_backward(h3, w, y.reshape(3, 50), lse, dl.reshape(3, 50))
    assert dh.shape == (3, 50, 80)
    ref.check(loss.reshape(-1), lse.reshape(-1), dh.reshape(150, 80), dw)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T", [5, 300])
def test_loss_every_token_ignored(T, t):
    h, w, y, dl = loss_case(T, 48, 333, t, seed=2)
    y.fill_(-100)
    dl.fill_(float("nan"))                                        # not read
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    assert not loss.any() and not dh.any() and not dw.any()
    within(lse, LossRef(h, w, y).lse, LossRef(h, w, y).lse_tol, "lse")


@pytest.mark.parametrize("ignore", [-1, 7, 2 ** 31 - 1, -2 ** 31])
def test_loss_other_ignored_values(ignore):
    h, w, y, dl = loss_case(64, 32, 50, F32, seed=3)
    y[::4] = ignore
    LossRef(h, w, y, dl, ignore=ignore).check(*run_loss(h, w, y, dl, ignore=ignore, check=True))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T", [20, 200])
def test_loss_bad_targets_are_loud_and_harmless(T, t):
    h, w, y, dl = loss_case(T, 40, 100, t, seed=5)
    bad = y.clone()
    bad[3], bad[11] = 100, -7
    loss, lse, dh, dw = run_loss(h, w, bad, dl)
    assert torch.isnan(loss[[3, 11]]).all() and not dh[[3, 11]].any()
    y[3], y[11] = -100, -100                                       # the others as if these were ignored
    ref = LossRef(h, w, y, dl)
    keep = [i for i in range(T) if i not in (3, 11)]
    within(loss[keep], ref.loss[keep], ref.loss_tol[keep], "loss")
    within(dh, ref.dh, ref.dh_tol, "dh")
    within(dw, ref.dw, ref.dw_tol, "dw")
    with pytest.raises(L.DeviceError, match="27"):
        mb.linear_cross_entropy(h, w, bad, check=True)
    with pytest.raises(L.DeviceError, match="27"):
        mb.linear_cross_entropy_backward(h, w, bad, lse, dl, check=True)
    with pytest.raises(L.DeviceError, match="27"):
        mb.linear_cross_entropy(h, w, bad.to(torch.int64) + 2 ** 32, check=True)   # not 3 again


@pytest.mark.parametrize("t", TYPES)
def test_loss_nan_stays_in_its_token(t):
    h, w, y, dl = loss_case(70, 64, 90, t, seed=7)
    clean = mb.linear_cross_entropy(h, w, y)[0]
    h[13, 2] = float("nan")
    loss = mb.linear_cross_entropy(h, w, y)[0]
    keep = [i for i in range(70) if i != 13]
    assert torch.isnan(loss[13]) and torch.equal(loss[keep], clean[keep])


@pytest.mark.parametrize("t", TYPES)
def test_loss_peaked_and_flat_rows(t):
    # logits of a few hundred: one entry has all the probability; and none at all
    h, w, y, dl = loss_case(130, 64, 1000, t, seed=11)
    h[:40] *= 60
    h[40:80] = 0
    LossRef(h, w, y, dl).check(*run_loss(h, w, y, dl))


def test_loss_tiny_and_huge_float32_operands():
    for a, b in ((1e-30, 1e30), (1e18, 1e-18), (1e-20, 1e-20), (1e-38, 1.0)):
        h, w, y, dl = loss_case(33, 24, 77, F32, seed=12)
        h, w = h * a, w * b
        LossRef(h, w, y, dl).check(*run_loss(h, w, y, dl))
    h, w, y, dl = loss_case(33, 24, 77, F32, seed=12)
    LossRef(torch.zeros_like(h), w, y, dl).check(*run_loss(torch.zeros_like(h), w, y, dl))


def test_loss_empty():
    h = torch.empty(0, 16, dtype=BF16, device="cuda")
    w = torch.randn(40, 16, device="cuda").to(BF16)
    y = torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse, dh, dw = run_loss(h, w, y, torch.empty(0, device="cuda"), check=True)
    assert loss.shape == lse.shape == (0,) and dh.shape == (0, 16) and not dw.any()


@pytest.mark.parametrize("t,T,d,V", [(BF16, 3000, 64, 60000), (F32, 2500, 40, 40000)])
def test_loss_several_vocabulary_pieces(t, T, d, V):
    # dz of the whole vocabulary is 360 and 400 MB: two pieces
    h, w, y, dl = loss_case(T, d, V, t, seed=15, gap=9)
    loss, lse, dh, dw = run_loss(h, w, y, dl)
    rows = torch.arange(0, T, 97, device="cuda")
    ref = LossRef(h[rows], w, y[rows], dl[rows])
    within(loss[rows], ref.loss, ref.loss_tol, "loss")
    # 26 tokens take the exact dz of short calls in the bounds above; here each
    # entry is rounded once to the type
    extra = 0 if t == F32 else half_step(t) * ((ref.dh.abs() * 0 + 1) * (dl[rows].double()[:, None] * w.double().abs().max() * 3))
    within(dh[rows], ref.dh, ref.dh_tol + extra, "dh")
    p = torch.exp(h.double() @ w[-70:].double().T - lse.double()[:, None])
    g = torch.where(y != -100, dl, torch.zeros_like(dl)).double()
    one = (y[:, None] == torch.arange(V - 70, V, device="cuda")[None]).double()
    dz = (p - one) * g[:, None]
    want, mag = dz.T @ h.double(), ((p + one) * g[:, None]).T @ h.double().abs()
    within(dw[-70:], want, mag * ((2e-5 if t == F32 else 2 * half_step(t)) + 2 * U * T) + half_step(t) * want.abs(), "dw")


def test_loss_offsets_beyond_32_bits():
    V, d = (1 << 21) + 5, 1032                                     # 2^31 + 1.7e7 entries of the weight
    g = gen(3)
    w = torch.empty(V, d, dtype=BF16, device="cuda")
    for i in range(0, V, 1 << 18):
        w[i:i + (1 << 18)] = torch.randn(min(1 << 18, V - i), d, device="cuda", generator=g).to(BF16) * 0.05
    h = torch.randn(3, d, device="cuda", generator=g).to(BF16)
    y = torch.tensor([V - 1, 0, V // 2], dtype=torch.int32, device="cuda")
    dl = torch.full((3,), 1 / 3, device="cuda")
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    z = torch.cat([h.double() @ w[i:i + (1 << 17)].double().T for i in range(0, V, 1 << 17)], 1)
    want = torch.logsumexp(z, 1)
    tol = (d / 16 + V / 32 / 148 + 64) * 2 * U * 40
    within(lse, want, tol, "lse")
    within(loss, want - z[torch.arange(3), y.long()], 2 * tol, "loss")
    p = (z - want[:, None]).exp()
    p[torch.arange(3), y.long()] -= 1
    for at in (0, V // 2, V - 40):
        a = p[:, at:at + 40].T @ h.double() / 3
        within(dw[at:at + 40], a, half_step(BF16) * a.abs() + (2.0 ** -15 + tol) * (p[:, at:at + 40].abs().T @ h.double().abs()) / 3, "dw")


def test_loss_gradient_against_differences():
    h, w, y, dl = loss_case(9, 32, 120, F32, seed=31)
    v, vw = torch.randn(9, 32, device="cuda", generator=gen(5)), torch.randn(120, 32, device="cuda", generator=gen(6)) * 0.1
    e = 2e-3
    f = lambda a, b: float((dl.double() * mb.linear_cross_entropy(a, b, y)[0].double()).sum())  # noqa: E731
    _, lse = mb.linear_cross_entropy(h, w, y)
    dh, dw = mb.linear_cross_entropy_backward(h, w, y, lse, dl)
    # the third derivative of log sum exp along s is at most 2 max |s|^3; the
    # values' own error enters over the step
    ref = LossRef(h, w, y)
    noise = float((dl.double() * ref.loss_tol).sum()) / e
    for dirs, got in (((v, 0 * w), (dh.double() * v.double()).sum()), ((0 * h, vw), (dw.double() * vw.double()).sum())):
        diff = (f(h + e * dirs[0], w + e * dirs[1]) - f(h - e * dirs[0], w - e * dirs[1])) / (2 * e)
        s = (dirs[0].double() @ w.double().T + h.double() @ dirs[1].double().T).abs().max(1).values
        assert abs(diff - float(got)) <= float((dl.double() * 2 * s ** 3).sum()) * e * e / 6 + noise + 1e-5 * abs(float(got))


# ---- orthogonalised update -----------------------------------------------------------------
def orth_ref(u, steps, coef, eps):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        p = x @ x.mT
        x = coef[0] * x + (coef[1] * p + coef[2] * p @ p) @ x
    return x.mT if tall else x


def orth_within(got, want, t, factor=1.0):
    got, want = got.double(), want.double()
    n = torch.linalg.matrix_norm
    bound = (5e-5 * factor + half_step(t)) * n(want) + tiny(t) * want.shape[-1] ** 0.5 * want.shape[-2] ** 0.5
    off = n(got - want)
    assert (off <= bound).all(), float((off / bound).max())


MUON = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (2, 3), (33, 32), (64, 64), (100, 257), (257, 100), (128, 1000),
                                   (1000, 128), (513, 512), (3, 40, 24), (2, 2, 130, 70), (5, 256, 256)])
def test_orthogonalize(shape, t):
    u = (1e-3 * torch.randn(*shape, device="cuda", generator=gen(sum(shape)))).to(t)
    x = mb.orthogonalize(u)
    assert x.dtype == t and x.shape == u.shape
    orth_within(x, orth_ref(u, 5, MUON, 1e-7), t)


# one to eight CTAs a matrix, the last one's columns partly or all past the end; and the first sizes beyond
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(16, 128, 256), (3, 128, 257), (3, 257, 65), (64, 512), (2, 65, 513), (513, 64), (2, 127, 1025),
                                   (1030, 128), (128, 2048), (2048, 17), (3, 2047), (40, 8, 1100), (128, 2049), (2049, 64),
                                   (129, 130), (2, 200, 129), (130, 1000)])
def test_orthogonalize_small_sides(shape, t):
    u = (1e-3 * torch.randn(*shape, device="cuda", generator=gen(sum(shape)))).to(t)
    x = mb.orthogonalize(u, check=True)
    assert x.dtype == t and x.shape == u.shape
    orth_within(x, orth_ref(u, 5, MUON, 1e-7), t)
    assert torch.equal(mb.orthogonalize(u), x)


@pytest.mark.parametrize("steps,coef", [(1, MUON), (12, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375))])
def test_orthogonalize_other_iterations(steps, coef):
    u = torch.randn(96, 160, device="cuda", generator=gen(1))
    # converging iterations contract errors in the end; every step adds its own
    orth_within(mb.orthogonalize(u, steps=steps, coefficients=coef), orth_ref(u, steps, coef, 1e-7), F32, max(1, steps / 5))


def test_orthogonalize_brings_singular_values_near_one():
    u = torch.randn(200, 512, device="cuda", generator=gen(2)) + 3 * torch.randn(200, 1, device="cuda", generator=gen(3))
    s = torch.linalg.svdvals(mb.orthogonalize(u).double())
    # the map's fixed band for singular values that start above 0.01
    assert 0.6 < float(s.min()) and float(s.max()) < 1.22


@pytest.mark.parametrize("shape", [(100, 200), (60, 700), (700, 60), (128, 2048)])
def test_orthogonalize_special_values_of_small_sides(shape):
    u = torch.randn(*shape, device="cuda", generator=gen(7))
    a = mb.orthogonalize(u, eps=0.0)
    for s in (2.0 ** 70, 2.0 ** -70):                                      # as below
        assert torch.equal(mb.orthogonalize(u * s, eps=0.0), a)
    assert not mb.orthogonalize(torch.zeros(2, *shape, device="cuda")).any()
    b = torch.stack([u, u, u, u])
    b[1, shape[0] - 1, shape[1] - 1], b[2, 0, 0] = float("nan"), float("inf")
    x = mb.orthogonalize(b, eps=0.0)
    assert torch.equal(x[0], a) and torch.equal(x[3], a) and torch.isnan(x[1:3]).all()
    for off in (1, 4):                                                     # 4- and 16-byte aligned
        shifted = torch.empty(u.numel() + off, device="cuda")[off:].view(*shape)
        shifted.copy_(u)
        assert torch.equal(mb.orthogonalize(shifted, eps=0.0), a)
    # what is around the result stays as it was
    room = torch.full((u.numel() + 64,), 3.0, device="cuda")
    cfg = L.MemlayerOrthConfig(1, *shape, L.F32, 5, 3.4445, -4.7750, 2.0315, 0.0)
    ws = torch.empty(512, dtype=torch.uint8, device="cuda")
    assert L.lib().memlayer_orthogonalize(cfg, u.data_ptr(), room[32:].data_ptr(), ws.data_ptr(), 512,
                                          torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(room[32:-32].view(*shape), a) and (room[:32] == 3).all() and (room[-32:] == 3).all()


def test_small_updates_beside_other_calls():
    us = [torch.randn(*s, device="cuda", generator=gen(i)) for i, s in enumerate([(30, 64, 64), (9, 128, 700), (2, 300, 300),
                                                                                  (4, 1500, 100)])]
    h, w = torch.randn(700, 256, device="cuda", generator=gen(8)), torch.randn(3000, 256, device="cuda", generator=gen(9)) * 0.1
    y = torch.randint(0, 3000, (700,), device="cuda", generator=gen(10))
    want, loss = [mb.orthogonalize(u) for u in us], mb.linear_cross_entropy(h, w, y)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(5)]
    got = []
    for _ in range(20):
        got.append([mb.orthogonalize(u, stream=s) for u, s in zip(us, streams)]
                   + [mb.linear_cross_entropy(h, w, y, stream=streams[4])[0]])
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want + [loss]))


def test_small_update_captured_and_replayed():
    u = torch.randn(3, 100, 900, device="cuda", generator=gen(11))
    mb.orthogonalize(u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = mb.orthogonalize(u)
        z = mb.orthogonalize(x, steps=2)
    for i in range(3):
        u.copy_(torch.randn(3, 100, 900, device="cuda", generator=gen(20 + i)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, mb.orthogonalize(u)) and torch.equal(z, mb.orthogonalize(x, steps=2))


def test_orthogonalize_scales_and_special_values():
    u = torch.randn(40, 56, device="cuda", generator=gen(4))
    a = mb.orthogonalize(u, eps=0.0)
    # powers of two change no bit; squares of these leave float32's range
    for s in (2.0 ** 70, 2.0 ** -70):
        assert torch.equal(mb.orthogonalize(u * s, eps=0.0), a)
    assert not mb.orthogonalize(torch.zeros(3, 20, 30, device="cuda")).any()
    b = torch.stack([u, u, u])
    b[1, 3, 4] = float("nan")
    x = mb.orthogonalize(b, eps=0.0)
    assert torch.equal(x[0], a) and torch.equal(x[2], a) and torch.isnan(x[1]).all()
    assert mb.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    ut = torch.randn(56, 40, device="cuda", generator=gen(5)).t()          # a layout that has to be copied
    assert torch.equal(mb.orthogonalize(ut), mb.orthogonalize(ut.contiguous()))
    shifted = torch.empty(40 * 56 + 1, device="cuda")[1:].view(40, 56)     # not 16-byte aligned
    shifted.copy_(u)
    assert torch.equal(mb.orthogonalize(shifted, eps=0.0), a)


# ---- refusals of the entry points --------------------------------------------------------------
def test_entry_points_refuse_mismatched_tensors():
    x, s = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    y = torch.zeros(4, dtype=torch.int32, device="cuda")
    w = torch.randn(16, 8, device="cuda")
    v = torch.zeros(4, device="cuda")
    for error, call in [
            (ValueError, lambda: mb.layer_norm(x, s[:7], s)), (TypeError, lambda: mb.layer_norm(x.double(), s, s)),
            (TypeError, lambda: mb.layer_norm(x, s.cpu(), s)), (ValueError, lambda: mb.layer_norm(x, s, s, residual=x[:2])),
            (TypeError, lambda: mb.layer_norm(x, s, s, residual=x.half())),
            (L.MemlayerError, lambda: mb.layer_norm(x, s, s, eps=0.0)),
            (L.MemlayerError, lambda: mb.layer_norm(torch.zeros(2, 16385, device="cuda"), torch.ones(16385, device="cuda"),
                                                    torch.ones(16385, device="cuda"))),
            (ValueError, lambda: mb.layer_norm_backward(x, x[:3], s)), (TypeError, lambda: mb.layer_norm_backward(x, x.half(), s)),
            (TypeError, lambda: mb.linear_cross_entropy(x, w.half(), y)), (ValueError, lambda: mb.linear_cross_entropy(x, w[:, :7], y)),
            (ValueError, lambda: mb.linear_cross_entropy(x, w, y[:3])), (ValueError, lambda: mb.linear_cross_entropy(x, w, v)),
            (TypeError, lambda: mb.linear_cross_entropy(x, w, y.cpu())),
            (ValueError, lambda: mb.linear_cross_entropy(x, w, y, ignore_index=2 ** 31)),
            (ValueError, lambda: mb.linear_cross_entropy_backward(x, w, y, v[:2], v)),
            (ValueError, lambda: mb.linear_cross_entropy_backward(x, w, y, v, v, dlse=v[:1])),
            (ValueError, lambda: mb.orthogonalize(v)), (TypeError, lambda: mb.orthogonalize(y[None])),
            (L.MemlayerError, lambda: mb.orthogonalize(w, coefficients=(9.0, 0.0, 0.0))),
            (L.MemlayerError, lambda: mb.orthogonalize(w, steps=0))]:
        with pytest.raises(error):
            call()


# ---- as a program uses them ---------------------------------------------------------------------
def all_of_them(t=BF16):
    """One pass through every operator on fixed inputs."""
    h, w, y, dl = loss_case(400, 128, 1500, t, seed=40, gap=6)
    x, r, scale, bias, _, dr = norm_case(400, 128, t, seed=41)
    u = torch.randn(2, 96, 128, device="cuda", generator=gen(42)).to(t)

    def run():
        n, s = mb.layer_norm(x, scale, bias, residual=r)
        loss, lse = mb.linear_cross_entropy(n, w, y)
        dn, dw = mb.linear_cross_entropy_backward(n, w, y, lse, dl)
        dx, dp = mb.layer_norm_backward(dn, s, scale, dresidual=dr)
        return [n, s, loss, lse, dn, dw, dx, dp["scale"], dp["bias"], mb.orthogonalize(u)]
    return run


@pytest.mark.parametrize("t", TYPES)
def test_equal_calls_give_equal_bits(t):
    run = all_of_them(t)
    a, b = run(), run()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_calls_on_two_streams_at_once():
    run = all_of_them()
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want))


def test_stream_argument():
    h, w, y, dl = loss_case(300, 64, 500, F32, seed=43)
    x, _, scale, bias, dy, _ = norm_case(300, 64, F32, seed=44)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    a = mb.linear_cross_entropy(h, w, y, stream=s)
    b = mb.linear_cross_entropy_backward(h, w, y, a[1], dl, stream=s)
    c = mb.layer_norm_backward(dy, x, scale, stream=s)
    d = mb.orthogonalize(w, stream=s)
    s.synchronize()
    assert torch.equal(a[0], mb.linear_cross_entropy(h, w, y)[0])
    assert torch.equal(b[1], mb.linear_cross_entropy_backward(h, w, y, a[1], dl)[1])
    assert torch.equal(c[0], mb.layer_norm_backward(dy, x, scale)[0])
    assert torch.equal(d, mb.orthogonalize(w))


@pytest.mark.parametrize("t", TYPES)
def test_extension_and_general_way_agree(t):
    from model_b200 import train_ops
    fast, here = train_ops._fast, torch.cuda.current_stream()          # with a stream: the general way
    x, r, scale, bias, dy, dr = norm_case(90, 70, t, seed=51)
    h, w, y, dl = loss_case(90, 70, 300, t, seed=52)
    u = torch.randn(2, 90, 40, device="cuda", generator=gen(53)).to(t)
    x3 = x.view(9, 10, 70)
    pairs = [
        (fast.layer_norm(x, scale, bias, r, 1e-5), mb.layer_norm(x, scale, bias, residual=r, eps=1e-5, stream=here)),
        ((fast.layer_norm(x3, scale, bias, None, 1e-6),), (mb.layer_norm(x3, scale, bias, stream=here),)),
        ((fast.orthogonalize(u, 4, 3.4445, -4.775, 2.0315, 1e-7),), (mb.orthogonalize(u, steps=4, stream=here),)),
        (fast.linear_cross_entropy(h, w, y, -100), mb.linear_cross_entropy(h, w, y, stream=here))]
    lse = pairs[-1][1][1]
    pairs.append((fast.linear_cross_entropy_backward(h, w, y, lse, dl, dl, -100),
                  mb.linear_cross_entropy_backward(h, w, y, lse, dl, dlse=dl, stream=here)))
    dx, dp = mb.layer_norm_backward(dy, x, scale, dresidual=dr, stream=here)
    pairs.append((fast.layer_norm_backward(dy, x, scale, dr, 1e-6), (dx, dp["scale"], dp["bias"])))
    for got, want in pairs:
        assert len(got) == len(want)
        for p, q in zip(got, want):
            assert torch.equal(p, q) and p.shape == q.shape and p.dtype == q.dtype and p.is_contiguous()
            assert not p.requires_grad and p.device == q.device
    # parameters and tensors that carry gradients are taken, their results carry none
    p = torch.nn.Parameter(scale.clone())
    z = fast.layer_norm(x.float().requires_grad_(), p, bias, None, 1e-6)
    assert z is not None and not z.requires_grad
    assert fast.layer_norm(torch.empty(0, 70, device="cuda", dtype=t), scale, bias, None, 1e-6).shape == (0, 70)


def test_extension_leaves_the_rest_to_the_general_way():
    from model_b200 import train_ops
    fast = train_ops._fast
    x, _, scale, bias, dy, _ = norm_case(12, 32, F32, seed=54)
    h, w, y, dl = loss_case(12, 32, 50, F32, seed=55)
    class Sub(torch.Tensor):
        pass
    other = torch.zeros(12, 32)                                          # on the CPU
    for args in ((x[:, ::2], scale[:16], bias[:16]), (x.t(), scale[:12], bias[:12]), (x.double(), scale, bias),
                 (x, scale.half(), bias), (x, scale[:31], bias), (x, scale, bias.cpu()), (x.as_subclass(Sub), scale, bias),
                 (torch.tensor(1.0, device="cuda"), scale, bias), (torch.empty(3, 0, device="cuda"), scale[:0], bias[:0])):
        assert fast.layer_norm(*args, None, 1e-6) is None
    assert fast.layer_norm(x, scale, bias, other, 1e-6) is None and fast.layer_norm(x, scale, bias, x[:3], 1e-6) is None
    assert fast.layer_norm(x, scale, bias, None, -1.0) is None and fast.layer_norm(x, scale, bias, None, "1") is None
    assert fast.layer_norm_backward(dy, x.half(), scale, None, 1e-6) is None
    assert fast.linear_cross_entropy(h, w, y.long(), -100) is None and fast.linear_cross_entropy(h, w, y[:5], -100) is None
    assert fast.linear_cross_entropy(h, w, y, 2 ** 31) is None and fast.linear_cross_entropy(h, w.half(), y, -100) is None
    assert fast.linear_cross_entropy_backward(h, w, y, dl[:3], dl, None, -100) is None
    assert fast.orthogonalize(h, 5, 30.0, 1.0, 1.0, 1e-7) is None and fast.orthogonalize(h[0], 5, 1., 1., 1., 1e-7) is None
    # the public functions take or refuse them as before
    assert torch.equal(mb.layer_norm(x.t(), scale[:12], bias[:12]), mb.layer_norm(x.t().contiguous(), scale[:12], bias[:12]))
    assert torch.equal(mb.linear_cross_entropy(h, w, y.long())[0], mb.linear_cross_entropy(h, w, y)[0])
    with pytest.raises(TypeError):
        mb.layer_norm(x.double(), scale, bias)
    with pytest.raises(L.MemlayerError):
        mb.layer_norm(x, scale, bias, eps=-1.0)


def test_captured_and_replayed():
    run = all_of_them()
    want = run()
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for _ in range(2):                       # two graphs that share their workspaces' memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(run())
        graphs.append(g)
    for k in (0, 1, 0):
        graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs[k], want))
        eager = run()
        assert all(torch.equal(p, q) for p, q in zip(eager, want))


def test_training_step_around_the_memory_layer():
    """Norm -> memory layer -> residual -> norm -> loss, and back: the hidden
    state's gradient along a direction against differences of the loss, then
    an orthogonalised update of the Dense kernels that lowers the loss's
    linear model."""
    from model_b200 import MemoryLayer, MemoryPool
    dm, V, M = 64, 300, 96
    layer = MemoryLayer(MemoryPool(n_sub_keys=16, heads=2, d_key=32, d_value=64, top_k=4), d_model=dm, layer=1)
    params = layer.init(3)
    g = gen(50)
    x = torch.randn(M, dm, device="cuda", generator=g)
    emb = torch.randn(V, dm, device="cuda", generator=g) * 0.2
    y = torch.randint(0, V, (M,), device="cuda", generator=g, dtype=torch.int32)
    one, zero = torch.ones(dm, device="cuda"), torch.zeros(dm, device="cuda")

    def forward(out_kernel):
        p = dict(params, mem_out_1={"kernel": out_kernel, "bias": params["mem_out_1"]["bias"]})
        a = mb.layer_norm(x, one, zero)
        upd, _, _, ctx = layer.apply_train(p, a)
        n, s = mb.layer_norm(upd, one, zero, residual=x)
        loss, lse = mb.linear_cross_entropy(n, emb, y)
        return a, ctx, n, s, loss, lse

    k = params["mem_out_1"]["kernel"]
    a, ctx, n, s, loss, lse = forward(k)
    dl = torch.full((M,), 1.0 / M, device="cuda")
    dn, demb = mb.linear_cross_entropy_backward(n, emb, y, lse, dl)
    ds, dp = mb.layer_norm_backward(dn, s, one)
    grads = layer.backward(ctx, ds)
    da = grads["h"]
    dx, _ = mb.layer_norm_backward(da, x, one, dresidual=ds)
    assert dx.shape == x.shape and torch.isfinite(dx).all()
    gk = grads["mem_out_1"]["kernel"]
    step = mb.orthogonalize(gk)
    inner = float((gk.double() * step.double()).sum())
    assert inner > 0                          # a descent direction: <G, orth G> is G's weighted nuclear norm
    e = 1e-2
    mean = lambda kk: float(forward(kk)[4].double().mean())  # noqa: E731
    diff = (mean(k + e * step) - mean(k - e * step)) / (2 * e)
    # the output kernel reaches the loss through a norm and log sum exp only
    # (the routing does not depend on it); the read and the update are O(1), so
    # the third-derivative term is below 100 e^2, the float32 noise 1e-6 / e
    assert abs(diff - inner) <= 100 * e * e * max(1.0, inner) / 6 + 2e-4


def test_model_loss_matches_its_logits():
    from model_b200 import MemoryPoolLM, ModelConfig
    cfg = ModelConfig(vocab_size=512, max_len=64, d_model=128, n_layers=2, n_heads=2, ffn_mult=2, memory_layers=(1,),
                      n_sub_keys=32, pool_heads=2, d_key=64, d_value=128, top_k=8)
    m = MemoryPoolLM(cfg)
    p = m.init(1)
    prep = m.prepare(p)
    tok = torch.randint(0, 512, (4, 64), device="cuda", generator=gen(60))
    tgt = torch.randint(0, 512, (4, 64), device="cuda", generator=gen(61))
    tgt[:, -1] = -100
    logits, _ = m.apply(prep, tok, check=True)
    loss, lse = m.loss(prep, tok, tgt, check=True)
    z = logits.double()
    want = torch.logsumexp(z, -1)
    zt = z.gather(-1, tgt.clamp(min=0)[..., None])[..., 0]
    # the logits come from another float32 GEMM and a norm with E[x^2] - E[x]^2:
    # each within 1e-5 of the largest logit
    tol = 4e-5 * float(z.abs().max())
    within(lse, want, tol, "lse")
    within(loss, torch.where(tgt == -100, 0.0, want - zt), 2 * tol, "loss")
    loss2, grads = m.loss_and_head_grads(prep, tok, tgt)
    assert torch.equal(loss, loss2)
    assert grads["hidden"].shape == (4, 64, 128) and grads["embed"]["embedding"].shape == (512, 128)
    # the same through float64 autograd from the residual stream
    x = prep.hidden(tok).double().requires_grad_()
    sc, bi = (p["ln_final"][k].double().requires_grad_() for k in ("scale", "bias"))
    E = p["embed"]["embedding"].double().requires_grad_()
    c = x - x.mean(-1, keepdim=True)
    h = c / (c.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * sc + bi
    z = h @ E.T
    nll = torch.logsumexp(z, -1) - z.gather(-1, tgt.clamp(min=0)[..., None])[..., 0]
    (nll * (tgt != -100)).sum().div((tgt != -100).sum()).backward()
    for got, ref in ((grads["hidden"], x.grad), (grads["ln_final"]["scale"], sc.grad),
                     (grads["ln_final"]["bias"], bi.grad), (grads["embed"]["embedding"], E.grad)):
        # logits of |z| <= 60 with 2^-20 of sum |h||e| each: 2e-4 of a probability
        assert float((got.double() - ref).abs().max()) <= 5e-4 * float(ref.abs().max())
    assert torch.equal(m.apply(prep, tok)[0], logits)
