"""What is measured of the training operators: layer norm with its gradient, the softmax cross entropy over
the vocabulary fused with the output projection and its gradient, and the orthogonalised update of the Dense
kernels.  ``run`` computes them either from elementary torch operations in 32 bits (``own`` false) or through
the package's entry points (``own`` true)."""

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6                                  # flax's LayerNorm epsilon
IGNORE = -100                               # targets that carry no loss
STEPS, COEF, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed():
    return [
        # one new token per sequence of a small batch: the norm between two decode-sized Dense layers
        {"name": "norm_decode_8x256_f32", "op": "norm", "rows": 8, "d": 256, "type": "f32", "train": False},
        # the norm of a training step: batch 32 x 256 tokens, the model's width, in the parameters' type
        {"name": "norm_train_8192x256_f32", "op": "norm", "rows": 8192, "d": 256, "type": "f32", "train": True},
        # a wider model in half precision, forward and backward
        {"name": "norm_train_16384x2048_bf16", "op": "norm", "rows": 16384, "d": 2048, "type": "bf16", "train": True},
        # a ragged batch and a width that is no power of two
        {"name": "norm_train_5003x1000_f16", "op": "norm", "rows": 5003, "d": 1000, "type": "f16", "train": True},
        # scoring a handful of candidate tokens over the 16,384-entry vocabulary
        {"name": "loss_16x256_v16384_f32", "op": "loss", "tokens": 16, "d": 256, "vocab": 16384, "type": "f32",
         "train": False},
        # held-out loss of one batch of the whole model (8192 tokens, vocabulary 16,384)
        {"name": "loss_8192x256_v16384_f32", "op": "loss", "tokens": 8192, "d": 256, "vocab": 16384, "type": "f32",
         "train": False},
        # a training step of the same model
        {"name": "loss_train_8192x256_v16384_f32", "op": "loss", "tokens": 8192, "d": 256, "vocab": 16384,
         "type": "f32", "train": True},
        # ragged: padded rows, an odd vocabulary, half precision
        {"name": "loss_train_1999x512_v30011_f16", "op": "loss", "tokens": 1999, "d": 512, "vocab": 30011,
         "type": "f16", "train": True},
        # a wide model with a large vocabulary
        {"name": "loss_train_8192x1024_v32768_bf16", "op": "loss", "tokens": 8192, "d": 1024, "vocab": 32768,
         "type": "bf16", "train": True},
        # the attention kernels of the four layers of the model in one call
        {"name": "orth_4x256x256_f32", "op": "orth", "batch": 4, "m": 256, "n": 256, "type": "f32"},
        # tall feed-forward kernels of a wider model, momentum kept in half precision
        {"name": "orth_2x2048x512_bf16", "op": "orth", "batch": 2, "m": 2048, "n": 512, "type": "bf16"},
        # a large square projection
        {"name": "orth_1x4096x4096_f32", "op": "orth", "batch": 1, "m": 4096, "n": 4096, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "loss", "orth"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        d = _log(rng, 32, 4096)
        if rng.random() < 0.6:
            d = max(32, d // 8 * 8)
        rows = min(_log(rng, 1, 32768), max(1, (1 << 25) // d))
        return {"op": op, "rows": rows, "d": d, "type": kind, "train": rng.random() < 0.7}
    if op == "loss":
        d = _log(rng, 64, 1024)
        if rng.random() < 0.75:
            d = max(64, d // 8 * 8)
        tokens, vocab = _log(rng, 1, 8192), _log(rng, 500, 65536)
        if kind == "f32":                    # three products for one: no more work than the largest listed case
            tokens = min(tokens, max(1, (1 << 36) // (vocab * d)))
        tokens = min(tokens, max(1, (1 << 37) // (vocab * d)))
        return {"op": op, "tokens": tokens, "d": d, "vocab": vocab, "type": kind, "train": rng.random() < 0.6}
    m, n = _log(rng, 32, 3000), _log(rng, 32, 3000)
    batch = min(_log(rng, 1, 12), max(1, (1 << 33) // (min(m, n) ** 2 * max(m, n))))
    return {"op": op, "batch": batch, "m": m, "n": n, "type": kind}


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["type"]]
    s = dict(case)
    if case["op"] == "norm":
        M, d = case["rows"], case["d"]
        s["x"] = (_randn(g, M, d) * (0.5 + 2.0 * torch.rand(M, 1, device="cuda", generator=g)) + 0.3).to(dt)
        s["r"] = (_randn(g, M, d) * 0.5).to(dt)
        s["scale"], s["bias"] = 1.0 + 0.2 * _randn(g, d), 0.1 * _randn(g, d)
        if case["train"]:
            s["dy"], s["dres"] = _randn(g, M, d).to(dt), _randn(g, M, d).to(dt)
    elif case["op"] == "loss":
        T, d, V = case["tokens"], case["d"], case["vocab"]
        s["h"] = _randn(g, T, d).to(dt)                               # the output of the last layer norm
        w = _randn(g, V, d) * (2.0 / d ** 0.5)
        s["targets"] = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
        s["w"] = w.to(dt)
        # a trained model puts weight on its targets: move the states towards theirs
        s["h"] = (s["h"].float() + w[s["targets"].long()] * (0.5 * torch.rand(T, 1, device="cuda", generator=g))).to(dt)
        if T > 4:                                                     # padding carries no loss
            s["targets"] = s["targets"].masked_fill(torch.rand(T, device="cuda", generator=g) < 0.1, IGNORE)
        if case["train"]:                                             # mean over the batch, weighted tokens
            s["dloss"] = (0.5 + torch.rand(T, device="cuda", generator=g)) / T
    else:
        B, m, n = case["batch"], case["m"], case["n"]
        k = max(1, min(m, n) // 8)                                    # gradients: a strong low-rank part and noise
        u = _randn(g, B, m, k) @ _randn(g, B, k, n) / k ** 0.5 + _randn(g, B, m, n)
        s["u"] = (u * 1e-3).to(dt)
    return s


def _norm(s):
    dt = DTYPES[s["type"]]
    x = (s["x"].float() + s["r"].float()).to(dt)                      # the residual stream as it is stored
    v = x.float()
    c = v - v.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    xhat = c * rstd
    y = (xhat * s["scale"] + s["bias"]).to(dt)
    if not s["train"]:
        return {"y": y, "x": x}
    dy = s["dy"].float()
    gy = dy * s["scale"]
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - xhat * (gy * xhat).mean(-1, keepdim=True)) + s["dres"].float()
    return {"y": y, "x": x, "dx": dx.to(dt), "dscale": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _loss(s):
    dt = DTYPES[s["type"]]
    h, w = s["h"].float(), s["w"].float()
    z = h @ w.T
    top = z.max(-1, keepdim=True).values
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(-1))
    keep = s["targets"] != IGNORE
    at = s["targets"].long().clamp(min=0)[:, None]
    loss = torch.where(keep, lse - z.gather(1, at)[:, 0], 0.0)
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    g = torch.where(keep, s["dloss"], 0.0)[:, None]
    dz = torch.exp(z - lse[:, None]) * g
    dz.scatter_add_(1, at, -g)
    return {"loss": loss, "lse": lse, "dh": (dz @ w).to(dt), "dw": (dz.T @ h).to(dt)}


def _orth(s):
    a, b, c = COEF
    u = s["u"].float()
    x = u / (torch.sqrt((u * u).sum((-2, -1), keepdim=True)) + NS_EPS)
    tall = s["m"] > s["n"]
    x = x.transpose(-2, -1) if tall else x
    for _ in range(STEPS):
        p = x @ x.transpose(-2, -1)
        x = a * x + (b * p + c * (p @ p)) @ x
    return {"x": (x.transpose(-2, -1) if tall else x).contiguous().to(s["u"].dtype)}


def _own_norm(s):
    import model_b200 as mb
    y, x = mb.layer_norm(s["x"], s["scale"], s["bias"], residual=s["r"], eps=EPS)
    if not s["train"]:
        return {"y": y, "x": x}
    dx, dp = mb.layer_norm_backward(s["dy"], x, s["scale"], dresidual=s["dres"], eps=EPS)
    return {"y": y, "x": x, "dx": dx, "dscale": dp["scale"], "dbias": dp["bias"]}


def _own_loss(s):
    import model_b200 as mb
    loss, lse = mb.linear_cross_entropy(s["h"], s["w"], s["targets"], ignore_index=IGNORE)
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    dh, dw = mb.linear_cross_entropy_backward(s["h"], s["w"], s["targets"], lse, s["dloss"], ignore_index=IGNORE)
    return {"loss": loss, "lse": lse, "dh": dh, "dw": dw}


def _own_orth(s):
    import model_b200 as mb
    return {"x": mb.orthogonalize(s["u"], steps=STEPS, coefficients=COEF, eps=NS_EPS)}


def run(state):
    if own:
        return {"norm": _own_norm, "loss": _own_loss, "orth": _own_orth}[state["op"]](state)
    return {"norm": _norm, "loss": _loss, "orth": _orth}[state["op"]](state)


def work(case):
    e = DTYPES[case["type"]].itemsize
    if case["op"] == "norm":
        n = case["rows"] * case["d"]
        # in: x, r (and dy, dres); out: y, x (and dx); parameters and their gradients
        return {"bytes": n * e * (7 if case["train"] else 4) + case["d"] * 4 * (4 if case["train"] else 2),
                "flops": n * (23 if case["train"] else 9)}
    if case["op"] == "loss":
        T, d, V = case["tokens"], case["d"], case["vocab"]
        both = T * d + V * d
        # the logits once, and the two products of the gradient; three 11-bit products make one of 22 bits,
        # which is how a float32 product runs: the flops counted are the operator's own
        return {"bytes": both * e * (2 if case["train"] else 1) + T * (16 if case["train"] else 12),
                "flops": 2.0 * T * V * d * (3 if case["train"] else 1) + 4.0 * T * V}
    B, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # per step: the symmetric m x m products need half of their entries
    return {"bytes": 2 * B * m * n * e, "flops": B * STEPS * (1.0 * m * m * n + 1.0 * m * m * m + 2.0 * m * m * n)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        dt = DTYPES[case["type"]]
        x = (s["x"].double() + s["r"].double()).to(dt)
        v = x.double()
        mean, var = v.mean(-1, keepdim=True), v.var(-1, unbiased=False, keepdim=True)
        xhat = (v - mean) / torch.sqrt(var + EPS)
        out = {"y": torch.addcmul(s["bias"].double(), xhat, s["scale"].double()), "x": x.double()}
        if case["train"]:
            dy = s["dy"].double()
            gh = dy * s["scale"].double()
            proj = gh - gh.mean(-1, keepdim=True) - xhat * torch.einsum("md,md->m", gh, xhat)[:, None] / case["d"]
            out["dx"] = proj / torch.sqrt(var + EPS) + s["dres"].double()
            out["dscale"], out["dbias"] = torch.einsum("md,md->d", dy, xhat), dy.sum(0)
        return out
    if case["op"] == "loss":
        h, w, t = s["h"].double(), s["w"].double(), s["targets"].long()
        loss, lse, dh, dw = [], [], [], torch.zeros_like(w)
        for i in range(0, case["tokens"], 2048):                      # tokens in pieces, float64 logits
            hi, ti = h[i:i + 2048], t[i:i + 2048]
            z = torch.mm(hi, w.t())
            l = torch.logsumexp(z, 1)
            on = (ti != IGNORE).double()
            loss.append(on * (l - torch.einsum("td,td->t", hi, w[ti.clamp(min=0)])))
            lse.append(l)
            if case["train"]:
                g = on * s["dloss"][i:i + 2048].double()
                p = torch.softmax(z, 1)
                p[torch.arange(len(ti), device=p.device), ti.clamp(min=0)] -= 1.0
                p.mul_(g[:, None])
                dh.append(torch.mm(p, w))
                dw += torch.mm(p.t(), hi)
        out = {"loss": torch.cat(loss), "lse": torch.cat(lse)}
        return dict(out, dh=torch.cat(dh), dw=dw) if case["train"] else out
    a, b, c = COEF
    x = s["u"].double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NS_EPS)
    left = case["m"] <= case["n"]
    for _ in range(STEPS):
        if left:                                                      # (a I + b P + c P^2) X, P = X X^T
            p = torch.bmm(x, x.mT)
            x = a * x + torch.bmm(b * p, x) + torch.bmm(c * p, torch.bmm(p, x))
        else:
            p = torch.bmm(x.mT, x)
            x = a * x + torch.bmm(x, b * p) + torch.bmm(torch.bmm(x, p), c * p)
    return {"x": x}
