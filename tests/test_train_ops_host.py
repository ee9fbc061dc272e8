"""Argument checks of the training operators (layer norm, vocabulary cross
entropy, orthogonalised update): every refusal happens on the host, before
anything touches a GPU."""

import ctypes as C

import pytest
import torch

import model_b200 as mb
from model_b200 import _lib as L

FAKE = 1 << 20   # an aligned address that no call gets to read


def test_struct_sizes_match_header_layout():
    assert C.sizeof(L.MemlayerNormConfig) == 8 + 3 * 4 + 4          # padded to 8
    assert C.sizeof(L.MemlayerNormArgs) == 8 * 8
    assert C.sizeof(L.MemlayerNormGrads) == 10 * 8
    assert C.sizeof(L.MemlayerLossConfig) == 8 + 4 * 4
    assert C.sizeof(L.MemlayerLossArgs) == 7 * 8
    assert C.sizeof(L.MemlayerLossGrads) == 5 * 8
    assert C.sizeof(L.MemlayerOrthConfig) == 8 + 8 * 4


# ---- layer norm -------------------------------------------------------------------
def norm_cfg(**kw):
    base = dict(rows=64, d_model=256, dtype=L.F32, epsilon=1e-6)
    base.update(kw)
    return L.MemlayerNormConfig(**base)


def norm_args(**kw):
    base = dict(x=FAKE, x_stride=256, scale=FAKE, bias=FAKE, y=FAKE)
    base.update(kw)
    return L.MemlayerNormArgs(**base)


def norm_grads(**kw):
    base = dict(dy=FAKE, dy_stride=256, x=FAKE, x_stride=256, scale=FAKE, dx=FAKE, dscale=FAKE, dbias=FAKE)
    base.update(kw)
    return L.MemlayerNormGrads(**base)


BAD_NORM = [(dict(rows=-1), L.ERR_BAD_SHAPE), (dict(d_model=0), L.ERR_BAD_SHAPE), (dict(epsilon=0.0), L.ERR_BAD_SHAPE),
            (dict(epsilon=-1e-6), L.ERR_BAD_SHAPE), (dict(epsilon=float("nan")), L.ERR_BAD_SHAPE),
            (dict(epsilon=float("inf")), L.ERR_BAD_SHAPE), (dict(d_model=16385), L.ERR_UNSUPPORTED),
            (dict(dtype=3), L.ERR_UNSUPPORTED), (dict(dtype=-1), L.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("bad,status", BAD_NORM)
def test_norm_sizes_refused(bad, status):
    lib = L.lib()
    c, n = norm_cfg(**bad), C.c_size_t()
    assert lib.memlayer_layer_norm(C.byref(c), C.byref(norm_args()), None) == status
    assert lib.memlayer_layer_norm_backward_workspace_size(C.byref(c), C.byref(n)) == status
    assert lib.memlayer_layer_norm_backward(C.byref(c), C.byref(norm_grads()), FAKE, 1 << 30, None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), L.ERR_BAD_POINTER), (dict(scale=None), L.ERR_BAD_POINTER), (dict(bias=None), L.ERR_BAD_POINTER),
    (dict(y=None), L.ERR_BAD_POINTER), (dict(x=FAKE + 2), L.ERR_BAD_POINTER), (dict(y=FAKE + 1), L.ERR_BAD_POINTER),
    (dict(x_stride=255), L.ERR_BAD_SHAPE), (dict(x_stride=-256), L.ERR_BAD_SHAPE),
    (dict(residual=FAKE, residual_stride=0), L.ERR_BAD_SHAPE),
    (dict(residual=FAKE + 3, residual_stride=256), L.ERR_BAD_POINTER)])
def test_norm_arguments_refused(bad, status):
    assert L.lib().memlayer_layer_norm(C.byref(norm_cfg()), C.byref(norm_args(**bad)), None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(dy=None), L.ERR_BAD_POINTER), (dict(x=None), L.ERR_BAD_POINTER), (dict(scale=None), L.ERR_BAD_POINTER),
    (dict(dx=None), L.ERR_BAD_POINTER), (dict(dscale=None), L.ERR_BAD_POINTER), (dict(dbias=None), L.ERR_BAD_POINTER),
    (dict(dy_stride=8), L.ERR_BAD_SHAPE), (dict(dresidual=FAKE, dresidual_stride=1), L.ERR_BAD_SHAPE)])
def test_norm_backward_arguments_refused(bad, status):
    c = norm_cfg()
    assert L.lib().memlayer_layer_norm_backward(C.byref(c), C.byref(norm_grads(**bad)), FAKE, 1 << 30, None) == status


def test_norm_backward_workspace_refused():
    lib, c, n = L.lib(), norm_cfg(), C.c_size_t()
    assert lib.memlayer_layer_norm_backward_workspace_size(C.byref(c), C.byref(n)) == L.OK and n.value > 0
    g = norm_grads()
    for ws, size in ((None, n.value), (FAKE, n.value - 1), (FAKE + 16, n.value)):
        assert lib.memlayer_layer_norm_backward(C.byref(c), C.byref(g), ws, size, None) == L.ERR_WORKSPACE
    assert lib.memlayer_layer_norm(None, C.byref(norm_args()), None) == L.ERR_BAD_POINTER
    assert lib.memlayer_layer_norm(C.byref(c), None, None) == L.ERR_BAD_POINTER


# ---- cross entropy ------------------------------------------------------------------
def loss_cfg(**kw):
    base = dict(tokens=32, d_model=64, vocab_size=1000, dtype=L.BF16, ignore_index=-100)
    base.update(kw)
    return L.MemlayerLossConfig(**base)


def loss_args(**kw):
    base = dict(h=FAKE, h_stride=64, weight=FAKE, weight_stride=64, targets=FAKE, loss=FAKE, lse=FAKE)
    base.update(kw)
    return L.MemlayerLossArgs(**base)


def loss_grads(**kw):
    base = dict(lse=FAKE, dloss=FAKE, dh=FAKE, dweight=FAKE)
    base.update(kw)
    return L.MemlayerLossGrads(**base)


@pytest.mark.parametrize("bad,status", [
    (dict(tokens=-1), L.ERR_BAD_SHAPE), (dict(tokens=1 << 31), L.ERR_BAD_SHAPE), (dict(d_model=0), L.ERR_BAD_SHAPE),
    (dict(vocab_size=0), L.ERR_BAD_SHAPE), (dict(dtype=9), L.ERR_UNSUPPORTED), (dict(d_model=65537), L.ERR_UNSUPPORTED),
    # 2^23 x 2^23 tiles would not fit the kernels' tile counter
    (dict(tokens=(1 << 31) - 1, vocab_size=(1 << 31) - 1), L.ERR_UNSUPPORTED),
    (dict(tokens=(1 << 31) - 1, vocab_size=(1 << 31) - 256), L.ERR_UNSUPPORTED),
    # the last column tile would end past 2^31
    (dict(tokens=1, vocab_size=(1 << 31) - 255), L.ERR_UNSUPPORTED)])
def test_loss_sizes_refused(bad, status):
    lib, n = L.lib(), C.c_size_t()
    c = loss_cfg(**bad)
    for backward in (0, 1):
        assert lib.memlayer_cross_entropy_workspace_size(C.byref(c), backward, C.byref(n)) == status
    assert lib.memlayer_cross_entropy(C.byref(c), C.byref(loss_args()), FAKE, 1 << 40, None) == status
    assert lib.memlayer_cross_entropy_backward(C.byref(c), C.byref(loss_args()), C.byref(loss_grads()), FAKE, 1 << 40,
                                               None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(h=None), L.ERR_BAD_POINTER), (dict(weight=None), L.ERR_BAD_POINTER), (dict(targets=None), L.ERR_BAD_POINTER),
    (dict(loss=None), L.ERR_BAD_POINTER), (dict(lse=None), L.ERR_BAD_POINTER), (dict(h=FAKE + 1), L.ERR_BAD_POINTER),
    (dict(targets=FAKE + 2), L.ERR_BAD_POINTER), (dict(h_stride=63), L.ERR_BAD_SHAPE),
    (dict(weight_stride=0), L.ERR_BAD_SHAPE)])
def test_loss_arguments_refused(bad, status):
    c = loss_cfg()
    assert L.lib().memlayer_cross_entropy(C.byref(c), C.byref(loss_args(**bad)), FAKE, 1 << 40, None) == status


@pytest.mark.parametrize("bad", [dict(lse=None), dict(dloss=None), dict(dh=None), dict(dweight=None),
                                 dict(dh=FAKE + 1), dict(dlse=FAKE + 2), dict(dweight=FAKE + 1)])
def test_loss_backward_arguments_refused(bad):
    c = loss_cfg()
    assert L.lib().memlayer_cross_entropy_backward(C.byref(c), C.byref(loss_args()), C.byref(loss_grads(**bad)), FAKE,
                                                   1 << 40, None) == L.ERR_BAD_POINTER


def test_loss_workspace_refused():
    lib, c, n = L.lib(), loss_cfg(), C.c_size_t()
    for backward in (0, 1):
        assert lib.memlayer_cross_entropy_workspace_size(C.byref(c), backward, C.byref(n)) == L.OK
        for ws, size in ((None, n.value), (FAKE, n.value - 1), (FAKE + 128, n.value)):
            st = (lib.memlayer_cross_entropy_backward(C.byref(c), C.byref(loss_args()), C.byref(loss_grads()), ws,
                                                      size, None) if backward else
                  lib.memlayer_cross_entropy(C.byref(c), C.byref(loss_args()), ws, size, None))
            assert st == L.ERR_WORKSPACE
    code = C.c_int32()
    assert lib.memlayer_train_status(None, C.byref(code), None) == L.ERR_BAD_POINTER


def test_loss_workspace_does_not_hold_the_logits():
    # the backward's piece of the vocabulary is bounded: twice the vocabulary
    # does not double it
    n = C.c_size_t()
    sizes = []
    for V in (1 << 17, 1 << 18):
        c = loss_cfg(tokens=8192, d_model=64, vocab_size=V)
        L.check(L.lib().memlayer_cross_entropy_workspace_size(C.byref(c), 1, C.byref(n)), "size")
        sizes.append(n.value - 2 * V * 64)               # without the 16-bit form of the weight
    assert sizes[1] <= sizes[0] * 1.05 and sizes[1] < 8192 * (1 << 18) * 2 // 4


# ---- orthogonalised update ------------------------------------------------------------
def orth_cfg(**kw):
    base = dict(batch=2, rows=64, cols=48, dtype=L.F32, steps=5, a=3.4445, b=-4.7750, c=2.0315, epsilon=1e-7)
    base.update(kw)
    return L.MemlayerOrthConfig(**base)


@pytest.mark.parametrize("bad,status", [
    (dict(batch=-1), L.ERR_BAD_SHAPE), (dict(rows=0), L.ERR_BAD_SHAPE), (dict(cols=0), L.ERR_BAD_SHAPE),
    (dict(steps=0), L.ERR_BAD_SHAPE), (dict(epsilon=-1.0), L.ERR_BAD_SHAPE),
    (dict(epsilon=float("nan")), L.ERR_BAD_SHAPE), (dict(rows=32769), L.ERR_UNSUPPORTED),
    (dict(cols=32769), L.ERR_UNSUPPORTED), (dict(steps=65), L.ERR_UNSUPPORTED), (dict(dtype=4), L.ERR_UNSUPPORTED),
    # singular values grow without bound / are not numbers
    (dict(a=5.0, b=1.0, c=0.0), L.ERR_UNSUPPORTED), (dict(a=float("nan")), L.ERR_UNSUPPORTED),
    (dict(a=0.0, b=-40.0, c=40.0), L.ERR_UNSUPPORTED)])
def test_orth_sizes_and_coefficients_refused(bad, status):
    lib, n = L.lib(), C.c_size_t()
    c = orth_cfg(**bad)
    assert lib.memlayer_orthogonalize_workspace_size(C.byref(c), C.byref(n)) == status
    assert lib.memlayer_orthogonalize(C.byref(c), FAKE, FAKE, FAKE, 1 << 40, None) == status


@pytest.mark.parametrize("coef", [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)])
def test_orth_usual_coefficients_accepted(coef):
    n = C.c_size_t()
    c = orth_cfg(a=coef[0], b=coef[1], c=coef[2], steps=10)
    assert L.lib().memlayer_orthogonalize_workspace_size(C.byref(c), C.byref(n)) == L.OK


def test_orth_arguments_refused():
    lib, c, n = L.lib(), orth_cfg(), C.c_size_t()
    assert lib.memlayer_orthogonalize_workspace_size(C.byref(c), C.byref(n)) == L.OK
    for u, o in ((None, FAKE), (FAKE, None), (FAKE + 2, FAKE), (FAKE, FAKE + 2)):
        assert lib.memlayer_orthogonalize(C.byref(c), u, o, FAKE, n.value, None) == L.ERR_BAD_POINTER
    for ws, size in ((None, n.value), (FAKE, n.value - 1), (FAKE + 64, n.value)):
        assert lib.memlayer_orthogonalize(C.byref(c), FAKE, FAKE, ws, size, None) == L.ERR_WORKSPACE


# ---- the Python entry points ------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, s = torch.zeros(4, 8), torch.zeros(8)
    t = torch.zeros(4, dtype=torch.int32)
    w = torch.zeros(16, 8)
    for call in (lambda: mb.layer_norm(x, s, s), lambda: mb.layer_norm_backward(x, x, s),
                 lambda: mb.linear_cross_entropy(x, w, t),
                 lambda: mb.linear_cross_entropy_backward(x, w, t, torch.zeros(4), torch.zeros(4)),
                 lambda: mb.orthogonalize(w)):
        with pytest.raises(TypeError):
            call()


def test_model_hidden_arguments_refused():
    pool = L.MemlayerConfig(tokens=0, heads=1, n_sub_keys=1, d_key=2, d_value=4, top_k=1, d_model=64)
    c = L.MemlayerModelConfig(vocab_size=16, max_len=8, d_model=64, n_layers=0, n_heads=2, ffn_mult=1, pool=pool)
    p = L.MemlayerModelParams(embedding=FAKE, pos_embed=FAKE, ln_final_scale=FAKE, ln_final_bias=FAKE)
    f = L.lib().memlayer_model_hidden
    assert f(C.byref(c), C.byref(p), FAKE, 2, 9, FAKE, FAKE, 1 << 30, None) == L.ERR_BAD_SHAPE       # seq > max_len
    assert f(C.byref(c), C.byref(p), None, 2, 8, FAKE, FAKE, 1 << 30, None) == L.ERR_BAD_POINTER
    assert f(C.byref(c), C.byref(p), FAKE, 2, 8, None, FAKE, 1 << 30, None) == L.ERR_BAD_POINTER
    assert f(C.byref(c), C.byref(p), FAKE, 2, 8, FAKE, None, 0, None) == L.ERR_WORKSPACE


def test_extension_declines_what_it_does_not_take():
    import torch
    from model_b200 import train_ops
    fast = train_ops._fast
    assert fast is not None, "csrc/fast_calls.cpp is not built"
    x, v = torch.zeros(2, 4), torch.zeros(4)
    calls = [(fast.layer_norm, (x, v, v, None, 1e-6)), (fast.layer_norm_backward, (x, x, v, None, 1e-6)),
             (fast.linear_cross_entropy, (x, x, torch.zeros(2, dtype=torch.int32), -100)),
             (fast.linear_cross_entropy_backward, (x, x, torch.zeros(2, dtype=torch.int32), v, v, None, -100)),
             (fast.orthogonalize, (x, 5, 3.4445, -4.775, 2.0315, 1e-7))]
    for f, args in calls:                    # tensors without a GPU, other things, too few and too many of them
        assert f(*args) is None and f(*args[:-1]) is None and f(*args, 1) is None and f() is None
        assert f(*([None] * len(args))) is None and f(*(["x"] * len(args))) is None and f(*([3] * len(args))) is None
    for call in (lambda: train_ops.layer_norm(x, v, v), lambda: train_ops.layer_norm_backward(x, x, v),
                 lambda: train_ops.linear_cross_entropy(x, x, v), lambda: train_ops.orthogonalize(x),
                 lambda: train_ops.linear_cross_entropy_backward(x, x, v, v, v)):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()


# ---- targets of every integer type --------------------------------------------------------
@pytest.mark.parametrize("t", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64])
def test_targets_of_any_integer_type_keep_their_ids(t):
    from model_b200 import train_ops
    h, w = torch.zeros(2, 3, 4), torch.zeros(100, 4)
    y = torch.tensor([[0, 1, 99], [7, 100, 127]]).to(t)
    assert train_ops._loss_args(h, w, y, -100)[-1].tolist() == [[0, 1, 99], [7, 100, 127]]
    if t.is_signed:
        y[0, 0] = -100
        assert train_ops._loss_args(h, w, y, -100)[-1].tolist() == [[-100, 1, 99], [7, 100, 127]]


def test_targets_beyond_32_bits_are_neither_ids_nor_ignored():
    from model_b200 import train_ops
    h, w = torch.zeros(4, 4), torch.zeros(100, 4)
    y = torch.tensor([3 + 2 ** 32, -1 - 2 ** 32, 2 ** 31, 5])
    for ignore in (-100, -1, -2, 3):
        t = train_ops._loss_args(h, w, y, ignore)[-1]
        assert t.dtype == torch.int32 and t[3] == 5 and not ((t[:3] >= 0) | (t[:3] == ignore)).any()
    t = train_ops._loss_args(h, w, torch.tensor([2 ** 32 - 100, 1, 2, 3], dtype=torch.uint32), -100)[-1]
    assert t.tolist() == [-1, 1, 2, 3]


@pytest.mark.parametrize("t", [torch.bool, torch.float32, torch.complex64, torch.uint64])
def test_targets_of_other_types_refused(t):
    from model_b200 import train_ops
    with pytest.raises(ValueError, match="targets must be integers"):
        train_ops._loss_args(torch.zeros(4, 4), torch.zeros(100, 4), torch.zeros(4, dtype=t), -100)


@pytest.mark.parametrize("check", [False, True])
def test_head_gradients_pass_check_to_every_call(monkeypatch, check):
    from model_b200 import model as M
    seen = {}

    def record(name, result):
        def call(*args, check=None, **kw):
            seen[name] = check
            return result
        return call
    x, v = torch.zeros(2, 3, 4), torch.zeros(2, 3)
    monkeypatch.setattr(M.PreparedModel, "hidden", record("hidden", x))
    monkeypatch.setattr(M, "layer_norm", lambda *a, **k: x)                # has no status to check
    monkeypatch.setattr(M, "linear_cross_entropy", record("loss", (v, v)))
    monkeypatch.setattr(M, "linear_cross_entropy_backward", record("loss gradient", (x, x)))
    monkeypatch.setattr(M, "layer_norm_backward", record("norm gradient", (x, {})))
    prep = object.__new__(M.PreparedModel)
    prep.device, prep.embedding, prep.ln_final = torch.device("cpu"), x, {"scale": v, "bias": v}
    tokens = torch.zeros(2, 3, dtype=torch.int32)
    prep.loss_and_head_grads(tokens, tokens, check=check)
    assert seen == {k: check for k in ("hidden", "loss", "loss gradient", "norm gradient")}
    seen.clear()
    prep.loss(tokens, tokens, check=check)
    assert seen == {"hidden": check, "loss": check}


# ---- the range of the update's iteration ---------------------------------------------------
def leaves_range(a, b, c, steps):
    """Whether some singular value in [0, 1] leaves the documented range (by a grid finer than any that the library needs)."""
    import numpy as np
    x = np.linspace(0, 1, 400001)
    for _ in range(steps):
        p = x * x
        r = b + c * p
        q = a + r * p
        if max(p.max() / 7.5, abs(r).max() / 12, abs(q).max() / 12) > 1:
            return True
        x = abs(x * q)
    return x.max() > 3


def orth_accepts(a, b, c, steps):
    n, cfg = C.c_size_t(), orth_cfg(a=a, b=b, c=c, steps=steps)
    return L.lib().memlayer_orthogonalize_workspace_size(C.byref(cfg), C.byref(n)) == L.OK


@pytest.mark.parametrize("a,b,c,steps", [(-1.3941725320194571, 3.485549324717482, -1.0893582225835132, 11),
                                         (0.9655603461302071, -8.625747304512245, 7.939453129480508, 3)])
def test_orth_iterations_that_few_singular_values_leave_refused(a, b, c, steps):
    # most values stay below 1.5, those of a narrow band grow to 1e290 (first case) or past 3
    assert leaves_range(a, b, c, steps) and not orth_accepts(a, b, c, steps)


def test_orth_iterations_inside_their_range_accepted():
    import numpy as np
    rng = np.random.default_rng(5)
    taken = 0
    for _ in range(300):
        a, b, c = (float(np.float32(v)) for v in (rng.uniform(-5, 5), rng.uniform(-10, 10), rng.uniform(-6, 6)))
        steps = int(rng.integers(1, 6))
        ok = orth_accepts(a, b, c, steps)
        taken += ok
        if ok:
            assert not leaves_range(a, b, c, steps), (a, b, c, steps)
    assert taken > 30
    for coef in ((3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)):
        for steps in (1, 5, 64):
            assert orth_accepts(*coef, steps) == (not leaves_range(*coef, steps))


# ---- the extension module's build -----------------------------------------------------------
@pytest.fixture
def elsewhere(monkeypatch, tmp_path):
    from model_b200 import build as B
    monkeypatch.setattr(B, "FAST", str(tmp_path / "_fast.so"))
    monkeypatch.setattr(B, "FAST_STAMP", str(tmp_path / "stamp"))
    runs = []

    def compiler(fails):
        def run(cmd, **kw):
            runs.append(cmd)
            if fails == "missing":
                raise FileNotFoundError(cmd[0])
            if not fails:
                (tmp_path / "_fast.so").write_text("built")
            return type("R", (), {"returncode": int(bool(fails)), "stdout": "", "stderr": "no such header"})()
        monkeypatch.setattr(B.subprocess, "run", run)
    return B, compiler, runs


@pytest.mark.parametrize("fails", [True, "missing"])
def test_extension_that_does_not_compile_is_a_warning(elsewhere, capsys, fails):
    B, compiler, runs = elsewhere
    with open(B.FAST, "w") as f:                     # one of another torch
        f.write("old")
    compiler(fails)
    assert B.build_fast() is False and "go over ctypes" in capsys.readouterr().err
    import os
    assert not os.path.exists(B.FAST) and not os.path.exists(B.FAST_STAMP)


def test_extension_is_built_again_for_another_torch(elsewhere, monkeypatch):
    B, compiler, runs = elsewhere
    compiler(False)
    assert B.build_fast() and B.build_fast() and len(runs) == 1
    monkeypatch.setattr(torch, "__version__", "0.0+other")
    assert B.build_fast() and B.build_fast() and len(runs) == 2


def test_extension_of_another_torch_is_not_used(monkeypatch):
    from model_b200 import train_ops
    fast = train_ops._fast
    assert fast is not None and fast.torch_version == torch.__version__ and train_ops._usable(fast) is fast
    assert train_ops._usable(None) is None
    monkeypatch.setattr(torch, "__version__", "0.0+other")
    assert train_ops._usable(fast) is None
