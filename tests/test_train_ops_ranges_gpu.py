"""The training operators where several of their parts meet: calls whose
clusters work on both gradients, sums cut into slices, rows and tokens of very
different magnitudes, padding with anything in it.  References, bounds and
their derivation: test_train_ops_gpu.py."""

import ctypes as C

import pytest
import torch

import model_b200 as mb
from model_b200 import _lib as L
from test_train_ops_gpu import (BF16, F16, F32, TYPES, U, LossRef, check_norm_backward, gen, half_step, loss_case,
                                norm_case, norm_ref, run_loss, tiny, within)

pytestmark = pytest.mark.gpu


# ---- loss: clusters with tiles of dh and of dW ------------------------------------------
# dh is summed from float32 partials and dW written in 16 bits by the same warps (60 to 81 of the clusters)
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("T,d,V", [(64, 768, 50257), (128, 1024, 32768), (32, 512, 65536), (64, 512, 65536), (1024, 768, 50257)])
def test_loss_gradients_that_share_a_cluster(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + V, gap=7)
    got = run_loss(h, w, y, dl, check=True)
    LossRef(h, w, y, dl).check(*got)
    for _ in range(5):
        again = run_loss(h, w, y, dl)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_loss_dh_of_a_vocabulary_beyond_32_bits():
    V, d = (1 << 21) + 5, 1032
    g = gen(3)
    w = torch.empty(V, d, dtype=BF16, device="cuda")
    for i in range(0, V, 1 << 18):
        w[i:i + (1 << 18)] = torch.randn(min(1 << 18, V - i), d, device="cuda", generator=g).to(BF16) * 0.05
    h = torch.randn(3, d, device="cuda", generator=g).to(BF16)
    y = torch.tensor([V - 1, 0, V // 2], dtype=torch.int32, device="cuda")
    dl = torch.full((3,), 1 / 3, device="cuda")
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    z = torch.cat([h.double() @ w[i:i + (1 << 17)].double().T for i in range(0, V, 1 << 17)], 1)
    p = (z - torch.logsumexp(z, 1, keepdim=True)).exp() / 3
    mag = p.clone()
    at = torch.arange(3), y.long()
    p[at] -= 1 / 3
    mag[at] += 1 / 3
    want, size = torch.zeros(3, d, dtype=torch.float64, device="cuda"), torch.zeros(3, d, dtype=torch.float64, device="cuda")
    for i in range(0, V, 1 << 17):
        block = w[i:i + (1 << 17)].double()
        want += p[:, i:i + (1 << 17)] @ block
        size += mag[:, i:i + (1 << 17)] @ block.abs()
    # dz in two bf16 pieces 2^-16 of it, a logit of |z| <= 40 2^-15; truncating sums of at most V / 16 steps
    tol = size * (2.0 ** -16 + 2.0 ** -15 + (V / 16 + 64) * 2 * U) + half_step(BF16) * want.abs()
    within(dh, want, tol, "dh")


# dh for TMA, dweight two bytes beside a 16-byte boundary: one goes out by bulk stores, the other entry by entry
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("T,d,V", [(64, 768, 5000), (600, 256, 3000)])
def test_loss_gradients_stored_both_ways(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + V)
    _, lse = mb.linear_cross_entropy(h, w, y)
    dh, dw = mb.linear_cross_entropy_backward(h, w, y, lse, dl)
    code = {BF16: L.BF16, F16: L.F16}[t]
    cfg, nb = L.MemlayerLossConfig(T, d, V, code, -100), C.c_size_t()
    L.check(L.lib().memlayer_cross_entropy_workspace_size(cfg, 1, nb), "size")
    ws = torch.empty(nb.value, dtype=torch.uint8, device="cuda")
    for off_h, off_w in ((0, 1), (1, 0), (1, 1)):
        oh, ow = (torch.full((n + 16,), 5.0, device="cuda").to(t) for n in (T * d, V * d))
        a = L.MemlayerLossArgs(h.data_ptr(), d, w.data_ptr(), d, y.data_ptr(), None, None)
        g = L.MemlayerLossGrads(lse.data_ptr(), dl.data_ptr(), None, oh[off_h:].data_ptr(), ow[off_w:].data_ptr())
        L.check(L.lib().memlayer_cross_entropy_backward(cfg, a, g, ws.data_ptr(), nb.value,
                                                        torch.cuda.current_stream().cuda_stream), "backward")
        assert torch.equal(oh[off_h:off_h + T * d].view(T, d), dh) and torch.equal(ow[off_w:off_w + V * d].view(V, d), dw)
        assert (oh[:off_h] == 5).all() and (oh[off_h + T * d:] == 5).all()
        assert (ow[:off_w] == 5).all() and (ow[off_w + V * d:] == 5).all()


# the last tokens fill one warp's rows or part of them: the warps behind have nothing to store
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("T,d,V", [(545, 64, 9000), (769, 128, 5000), (1999, 96, 6007), (1057, 256, 4096)])
def test_loss_gradient_of_a_partly_filled_row_tile(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T, gap=11)
    got = run_loss(h, w, y, dl, check=True)
    LossRef(h, w, y, dl).check(*got)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(got, run_loss(h, w, y, dl)))


@pytest.mark.parametrize("it", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.uint32, torch.int64])
def test_loss_targets_of_any_integer_type(it):
    h, w, y, dl = loss_case(40, 32, 120, F32, seed=9)
    want = run_loss(h, w, y, dl)
    got = run_loss(h, w, y.to(it), dl, check=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_model_head_with_targets_of_any_integer_type():
    from model_b200 import MemoryPoolLM, ModelConfig
    cfg = ModelConfig(vocab_size=200, max_len=32, d_model=64, n_layers=1, n_heads=2, ffn_mult=2, memory_layers=(),
                      n_sub_keys=16, pool_heads=2, d_key=32, d_value=64, top_k=4)
    m = MemoryPoolLM(cfg)
    prep = m.prepare(m.init(1))
    tok = torch.randint(0, 200, (2, 32), device="cuda", generator=gen(60))
    tgt = torch.randint(0, 200, (2, 32), device="cuda", generator=gen(61))
    tgt[0, :8] = 156                         # -100 in eight bits
    loss, grads = m.loss_and_head_grads(prep, tok, tgt)
    for it in (torch.uint8, torch.int16, torch.int32):
        l2, g2 = m.loss_and_head_grads(prep, tok, tgt.to(it))
        assert torch.equal(loss, l2) and torch.equal(grads["hidden"], g2["hidden"])
        assert torch.equal(grads["embed"]["embedding"], g2["embed"]["embedding"])


# ---- loss: large logits -----------------------------------------------------------------
# the largest logit's own term is exp(0) whatever its size; one entry has all the probability
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("T,d,V", [(1, 64, 300), (16, 64, 1000), (24, 36, 500), (40, 130, 700), (200, 64, 3000), (300, 640, 300)])
def test_loss_of_large_logits(T, d, V, size, t):
    h, w, y, dl = loss_case(T, d, V, F32, seed=T + d)
    at = (h.double() @ w.double().T).argmax(1)
    y[::2] = at[::2].int()
    if t == F16:
        size = min(size, 1e8)                     # its range
    a = (size / 3) ** 0.5
    h, w = (h * a).to(t), (w * a).to(t)
    ref = LossRef(h, w, y, dl)
    # an exponential below the smallest normal float is 0, and bf16 holds what is left of it beside such
    # logits: 2^-126 of every term on top of the bounds (dw of entries of a probability of 1e-40 is 1e-40)
    none = 2.0 ** -126 * dl.double()[:, None].expand(T, V)
    ref.dh_tol, ref.dw_tol = ref.dh_tol + none @ w.double().abs(), ref.dw_tol + none.T @ h.double().abs()
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    ref.check(loss, lse, dh, dw)
    z = h.double() @ w.double().T
    top = z.max(1).values
    clear = (z < top[:, None] - 100).sum(1) == V - 1       # nothing else counts: lse is the logit itself
    assert size < 1e3 or clear.any()
    hit = clear & (y == z.argmax(1))
    assert not loss[hit].any()
    if T > 24:                                    # the gradient finds the forward's logits again: p is 1, dz 0
        assert not dh[hit].any()


# ---- loss: tokens of very different magnitudes -------------------------------------------
# float32 states run as two 16-bit pieces: each token's have to keep their digits whatever the others hold
@pytest.mark.parametrize("huge", [1e6, 1e10, 1e30])
@pytest.mark.parametrize("T,d,V", [(40, 24, 300), (200, 64, 700), (300, 1100, 400), (600, 130, 1001), (530, 256, 6000)])
def test_loss_of_tokens_beside_a_huge_one(T, d, V, huge):
    h, w, y, dl = loss_case(T, d, V, F32, seed=T + d)
    y[3], y[T - 1] = -100, -100
    h[3] *= huge                                  # padding with something in it
    h[T - 1] = huge
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    keep = torch.tensor([i for i in range(T) if i not in (3, T - 1)], device="cuda")
    ref = LossRef(h[keep], w, y[keep], dl[keep])
    ref.check(loss[keep], lse[keep], dh[keep], dw)         # ignored tokens add nothing to dW
    assert not loss[[3, T - 1]].any() and not dh[[3, T - 1]].any()
    # live ones: the others' loss, lse and dh are theirs; dW's sums keep their digits beside its largest term
    y[3] = 5
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    ref.check(loss[keep], lse[keep], dh[keep], ref.dw)
    LossRef(h[3:4], w, y[3:4], dl[3:4]).check(loss[3:4], lse[3:4], dh[3:4], LossRef(h[3:4], w, y[3:4], dl[3:4]).dw)
    live = torch.cat([keep, torch.tensor([3], device="cuda")])
    all_ = LossRef(h[live], w, y[live], dl[live])
    within(dw, all_.dw, all_.dw_tol, "dw")


def test_loss_of_tokens_beside_tiny_ones():
    h, w, y, dl = loss_case(150, 48, 500, F32, seed=8, gap=4)
    scale = 10.0 ** (torch.arange(150, device="cuda") % 30 - 25).double()
    h = (h.double() * scale[:, None]).float()
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    for e in range(30):
        at = torch.arange(e, 150, 30, device="cuda")
        ref = LossRef(h[at], w, y[at], dl[at])
        within(lse[at], ref.lse, ref.lse_tol, "lse")
        within(loss[at], ref.loss, ref.loss_tol, "loss")
        within(dh[at], ref.dh, ref.dh_tol, "dh")
    ref = LossRef(h, w, y, dl)
    within(dw, ref.dw, ref.dw_tol, "dw")


# loss weights over many orders of magnitude: every token's dh has its own digits
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,d,V", [(60, 40, 700), (128, 64, 5000), (200, 64, 700), (700, 128, 3001)])
def test_loss_gradient_of_light_tokens(T, d, V, t):
    h, w, y, _ = loss_case(T, d, V, t, seed=T + V)
    # f16 results hold 2^-24 and more: its weights stay above that
    kinds = [2.0 ** 9, 2.0 ** -1, 2.0 ** -9] if t == F16 else [1.0, 1e-4, 1e-9, 1e-15]
    dl = torch.tensor(kinds, device="cuda")[torch.arange(T, device="cuda") % len(kinds)]
    dl = dl * (0.5 + torch.rand(T, device="cuda", generator=gen(1)))
    dlse = dl * torch.randn(T, device="cuda", generator=gen(2))
    loss, lse, dh, dw = run_loss(h, w, y, dl, dlse, check=True)
    for i in range(len(kinds)):
        at = torch.arange(i, T, len(kinds), device="cuda")
        ref = LossRef(h[at], w, y[at], dl[at], dlse[at])
        # part of the tokens stands for all of them: where more than 128 are
        # given, an entry of dz is rounded once to the type
        mag = dl[at].double() + dlse[at].double().abs()
        p = (h[at].double() @ w.double().T - ref.lse[:, None]).exp() * mag[:, None]
        p.scatter_add_(1, y[at].long()[:, None], dl[at].double()[:, None])
        extra = half_step(t) * (p @ w.double().abs()) if T > 128 and t != F32 else 0
        within(dh[at], ref.dh, ref.dh_tol + extra, f"dh of weight {kinds[i]}")
    ref = LossRef(h, w, y, dl, dlse)
    ref.check(loss, lse, dh, dw)


# padding with anything in it: an ignored token's h reaches nothing but its own lse
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), "largest"])
@pytest.mark.parametrize("T,d,V", [(3, 40, 200), (9, 513, 300), (16, 1024, 129), (30, 64, 500), (100, 72, 257), (300, 100, 700), (280, 33, 400)])
def test_loss_padding_may_hold_anything(T, d, V, fill, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + d)
    pad = torch.arange(T, device="cuda") % 3 == 1
    y[pad] = -100
    clean = h.clone()
    clean[pad] = 0
    h[pad] = torch.finfo(t).max if fill == "largest" else fill
    dl[pad] = float("nan")                                        # not read
    want, got = run_loss(clean, w, y, dl, check=True), run_loss(h, w, y, dl, check=True)
    keep = ~pad
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][keep], want[1][keep])
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    assert not got[2][pad].any()
    LossRef(clean, w, y, dl).check(got[0], torch.where(pad, want[1], got[1]), got[2], got[3])
    # the same of a target that is no id
    y[1] = V + 3
    want, got = run_loss(clean, w, y, dl), run_loss(h, w, y, dl)
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])


# ---- norm: the first and last widths of each layout --------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [512, 516, 1022, 2042, 2046, 2048, 2052, 2056, 4090, 4094, 4096, 4100, 4104, 8186, 8190, 8192,
                               8196, 8200, 16378, 16380, 16384])
def test_norm_at_the_borders_of_the_layouts(d, t):
    x, r, scale, bias, dy, dr = norm_case(5, d, t, seed=d)
    params = torch.empty(2, d + 4, device="cuda")
    params[0, 1:d + 1], params[1, 1:d + 1] = scale, bias
    for sc, bi in ((scale, bias), (params[0, 1:d + 1], params[1, 1:d + 1])):      # parameters beside a 16-byte boundary, too
        y, s = mb.layer_norm(x, sc, bi, residual=r)
        want, tol, *_ = norm_ref(s, scale, bias, 1e-6)
        within(y, want, tol + half_step(t) * want.abs() + tiny(t), "y")
        dx, dp = mb.layer_norm_backward(dy, s, sc, dresidual=dr, check=True)
        check_norm_backward(dx, dp, dy, s, scale, dr, 1e-6, t)


# ---- loss: sums cut into slices -----------------------------------------------------------
# few tiles and many tokens: dW's sum over tokens is cut (s_w 2 to 5), joined by vectors or entry by entry;
# (5003, 65, 501): rows that TMA cannot address, an odd number of entries
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,d,V", [(4096, 128, 1000), (5003, 65, 501), (3000, 72, 777), (2500, 200, 640)])
def test_loss_sliced_dweight(T, d, V, t):
    h, w, y, dl = loss_case(T, d, V, t, seed=T + d, gap=5)
    dlse = 0.1 * dl * torch.randn(T, device="cuda", generator=gen(3))
    got = run_loss(h, w, y, dl, dlse, check=True)
    LossRef(h, w, y, dl, dlse).check(*got)
    assert all(torch.equal(a, b) for a, b in zip(got, run_loss(h, w, y, dl, dlse)))


@pytest.mark.parametrize("T,d,V", [(3000, 64, 60000), (2600, 65, 56001), (4200, 520, 40001)])
def test_loss_several_vocabulary_pieces_f16(T, d, V):
    h, w, y, dl = loss_case(T, d, V, F16, seed=15, gap=9)
    dl = dl * 1000                                    # its results are above f16's subnormals
    loss, lse, dh, dw = run_loss(h, w, y, dl, check=True)
    again = run_loss(h, w, y, dl)
    assert all(torch.equal(a, b) for a, b in zip((loss, lse, dh, dw), again))
    ref = LossRef(h, w, y, dl)
    ref.check(loss, lse, dh, dw)


# ---- norm: rows whose mean is far larger than their spread --------------------------------
# The mean as first summed is off by at most m0 = 32 u mean|x|; the centred values (exact beside such a mean, else u of
# themselves) are summed again, which leaves 32 u (spread + m0) of it, and 64 u m0^2 of the variance.
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("value,spread", [(1e4, 0.0), (-773.3, 0.0), (1e4, 0.05), (3e5, 1.0), (0.3, 1e-6), (1e-3, 0.0)])
@pytest.mark.parametrize("d", [7, 33, 256, 300, 768, 1003, 1500, 2048, 2498, 5000, 8200, 12288, 16384])
def test_norm_of_nearly_constant_rows(d, value, spread, t):
    if t == F16:
        value = max(-6e4, min(6e4, value))
    g = gen(d)
    x = (value * (1 + torch.rand(37, 1, device="cuda", generator=g) * 0.1)
         + spread * torch.randn(37, d, device="cuda", generator=g)).to(t)
    _, _, scale, bias, dy, _ = norm_case(37, d, t, seed=d)
    v = x.double()
    mean, sd = v.mean(-1, keepdim=True), v.std(-1, unbiased=False, keepdim=True)
    rstd = (sd ** 2 + 1e-6).rsqrt()
    xhat = (v - mean) * rstd
    m0 = 32 * U * v.abs().mean(-1, keepdim=True)
    e_rstd = 32 * U + 64 * U * (m0 * rstd) ** 2                       # relative
    e = 32 * U * (sd + m0) * rstd + (8 * U + e_rstd) * xhat.abs()
    want = xhat * scale.double() + bias.double()
    within(mb.layer_norm(x, scale, bias), want, scale.double().abs() * e + (4 * U + half_step(t)) * (want.abs() + bias.double().abs())
           + tiny(t), "y")
    dx, dp = mb.layer_norm_backward(dy, x, scale)
    gy = dy.double() * scale.double()
    c1, c2, mg = gy.mean(-1, keepdim=True), (gy * xhat).mean(-1, keepdim=True), gy.abs().mean(-1, keepdim=True)
    want = rstd * (gy - c1 - xhat * c2)
    mag = rstd * (gy.abs() + mg + xhat.abs() * (gy * xhat).abs().mean(-1, keepdim=True))
    # c2 from the first centred values less off times sum gy: 32 u of both, and the means' error once more
    e2 = (gy.abs() * e).mean(-1, keepdim=True) + 64 * U * m0 * rstd * mg
    tol = (64 * U + e_rstd) * mag + rstd * (e * c2.abs() + xhat.abs() * e2)
    within(dx, want, tol + half_step(t) * want.abs() + tiny(t), "dx")
    within(dp["scale"], (dy.double() * xhat).sum(0), (dy.double().abs() * (e + 96 * U * xhat.abs())).sum(0) + 1e-30, "dscale")


# the forward and the gradient of 17 to 24 float32 tokens add their logits in different orders: p stays at most 1
@pytest.mark.parametrize("T", [16, 17, 20, 24, 25])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e11])
def test_loss_gradient_of_large_logits_is_bounded(T, size):
    for seed in range(12):
        h, w, y, dl = loss_case(T, 36 + 4 * seed, 500, F32, seed=seed + T)
        y[::2] = (h.double() @ w.double().T).argmax(1)[::2].int()
        a = (size / 3) ** 0.5
        h, w = h * a, w * a
        _, _, dh, dw = run_loss(h, w, y, dl, check=True)
        # |dz| <= dl and the sum of p is 1 but for roundings of large logits, which leave each p below 1
        assert torch.isfinite(dh).all() and torch.isfinite(dw).all()
        near = ((h.double() @ w.double().T) > (h.double() @ w.double().T).max(1, keepdim=True).values - size * 1e-5 - 50).sum(1)
        assert (dh.abs() <= (near + 2)[:, None] * dl[:, None] * w.abs().max()).all()


def test_model_head_on_a_stream_and_captured():
    from model_b200 import MemoryPoolLM, ModelConfig
    cfg = ModelConfig(vocab_size=300, max_len=32, d_model=64, n_layers=2, n_heads=2, ffn_mult=2, memory_layers=(1,),
                      n_sub_keys=16, pool_heads=2, d_key=32, d_value=64, top_k=4)
    m = MemoryPoolLM(cfg)
    prep = m.prepare(m.init(2))
    tok = torch.randint(0, 300, (3, 32), device="cuda", generator=gen(60))
    tgt = torch.randint(0, 300, (3, 32), device="cuda", generator=gen(61))
    tgt[:, -3:] = -100

    def flat(out):
        loss, g = out
        return [loss, g["hidden"], g["ln_final"]["scale"], g["ln_final"]["bias"], g["embed"]["embedding"]]
    want = flat(m.loss_and_head_grads(prep, tok, tgt, check=True))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = flat(m.loss_and_head_grads(prep, tok, tgt, stream=s, check=True))
    alone, _ = m.loss(prep, tok, tgt, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(alone, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = flat(m.loss_and_head_grads(prep, tok, tgt))
    for shift in (0, 1):
        tok.copy_((tok + shift) % 300)
        graph.replay()
        torch.cuda.synchronize()
        want = flat(m.loss_and_head_grads(prep, tok, tgt))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# two threads on streams of their own, one of them through the general way
def test_calls_from_two_threads():
    import threading
    h, w, y, dl = loss_case(200, 128, 3000, BF16, seed=70, gap=5)
    x, r, scale, bias, dy, dr = norm_case(300, 1003, F16, seed=71)
    u = torch.randn(3, 100, 200, device="cuda", generator=gen(72))

    def run(it):
        n, s = mb.layer_norm(x, scale, bias, residual=r)
        dx, dp = mb.layer_norm_backward(dy, s, scale, dresidual=dr)
        return [n, dx, dp["scale"], mb.orthogonalize(u), *run_loss(h, w, y.to(it), dl)]
    want = run(torch.int32)
    torch.cuda.synchronize()
    failed = []

    def work(it):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = run(it)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        failed.append(it)
        except Exception as e:                       # reported by the test, not lost in the thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(it,)) for it in (torch.int32, torch.int64)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
