"""Measured cases of the layer normalisation and the vocabulary loss.

Two operators that every block and every loss of the TTT-E2E model go through,
each with its first and its second gradient (the meta step differentiates the
inner step's gradient):

* layer norm: ``layer_norm(x, weight, bias, eps)`` over rows of ``x``;
* the linear cross entropy: ``linear_cross_entropy(hidden, weight, targets,
  mask, reduction=...)``, the token loss of ``hidden @ weight.T`` without the
  logits in memory.

With ``own`` false, ``run`` computes them in elementary torch operations in 32
bits and rounds once at the end; with ``own`` true it calls the framework.
"""

import math
import random

import torch

own = False

EPS = 1e-5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases
def _ln(name, mode, rows, dim, dtype, param_dtype=None, pad=0):
    """pad: x is a slice of rows that are `pad` elements longer."""
    return {"name": name, "op": "ln", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype,
            "param_dtype": param_dtype or dtype, "pad": pad}


def _lce(name, mode, rows, dim, vocab, dtype, masked, reduction="mean"):
    """masked: a quarter of the positions is masked out of the loss."""
    return {"name": name, "op": "lce", "mode": mode, "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype,
            "masked": masked, "reduction": reduction}


def listed():
    return [
        # one token of a stream through a block's norm: pure latency
        _ln("ln_fwd_one_token", "fwd", 1, 512, "bf16"),
        # a block's norm over the meta step's sequence (8192 tokens, width 768), forward only (streaming inference)
        _ln("ln_fwd_8192x768", "fwd", 8192, 768, "bf16"),
        # an odd width and row count, 32-bit activations, rows cut out of a wider buffer
        _ln("ln_train_odd_fp32", "train", 4099, 1001, "fp32", pad=23),
        # a wide model's training batch; 32-bit norm weights beside 16-bit activations
        _ln("ln_train_16384x4096", "train", 16384, 4096, "bf16", param_dtype="fp32"),
        # the meta step's norm: forward, gradient, and the gradient of the gradient
        _ln("ln_gradgrad_8192x768", "gradgrad", 8192, 768, "bf16"),
        # scoring one token of a stream against the whole vocabulary
        _lce("lce_score_one_token", "fwd", 1, 768, 32000, "bf16", False, "none"),
        # per-token perplexity of a long document, odd vocabulary
        _lce("lce_eval_16384_odd_vocab", "fwd", 16384, 1024, 50001, "fp16", False, "none"),
        # an inner step on one chunk of the streaming demo's model (width 512, vocabulary 4096), loss scaling in fp16
        _lce("lce_train_demo_chunk", "train", 512, 512, 4096, "fp16", True),
        # test-time adaptation of the meta step's model: 8192 tokens, width 768, vocabulary 32000, a quarter masked
        _lce("lce_train_8192x768x32000", "train", 8192, 768, 32000, "bf16", True),
        # a wide model with a large vocabulary
        _lce("lce_train_4096x4096x128000", "train", 4096, 4096, 128000, "bf16", False),
        # the meta step's loss on a short ragged chunk: loss, gradient, and the gradient of the gradient
        _lce("lce_gradgrad_ragged", "gradgrad", 1000, 512, 4096, "bf16", True),
        # the same over the whole sequence
        _lce("lce_gradgrad_8192x768x32000", "gradgrad", 8192, 768, 32000, "bf16", False),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LCE_COST = {"fwd": 1, "train": 3, "gradgrad": 9}  # in units of one product of the logits' size
MAX_LCE = 3 * 4096 * 4096 * 128000 // 2
MAX_LN = 16384 * 4096


def draw(rng):
    mode = rng.choice(["fwd", "train", "gradgrad"])
    if rng.random() < 0.4:
        rows, dim = _loguniform(rng, 1, 65536), _loguniform(rng, 64, 8192)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        weight = {"fwd": 0.4, "train": 1.0, "gradgrad": 2.0}[mode]
        rows = max(1, min(rows, int(MAX_LN / weight) // dim))
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        return {"op": "ln", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype,
                "param_dtype": rng.choice([dtype, "fp32"]), "pad": rng.choice([0, 0, 0, 8, 13])}
    rows, dim, vocab = _loguniform(rng, 1, 16384), _loguniform(rng, 64, 4096), _loguniform(rng, 256, 131072)
    if rng.random() < 0.7:
        dim = max(64, dim // 64 * 64)
    rows = max(1, min(rows, MAX_LCE // (LCE_COST[mode] * dim * vocab)))
    return {"op": "lce", "mode": mode, "rows": rows, "dim": dim, "vocab": vocab, "dtype": rng.choice(["fp16", "bf16"]),
            "masked": rng.random() < 0.5, "reduction": rng.choice(["mean", "mean", "sum", "none"])}


def _kept(case):
    """Positions that enter the loss."""
    n = case["rows"]
    return max(1, n - n // 4) if case["masked"] else n


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    n, d = case["rows"], case["dim"]
    need = case["mode"] != "fwd"
    st = {"case": case}
    if case["op"] == "ln":
        pt = DTYPES[case["param_dtype"]]
        # a residual stream: unit noise, an offset per row, a few large channels
        wide = torch.randn(n, d + case["pad"], device="cuda", generator=g)
        wide += 0.5 * torch.randn(n, 1, device="cuda", generator=g)
        wide[:, :: max(1, d // 5)] *= 8.0
        st["x"] = wide.to(dt)[:, case["pad"] // 2: case["pad"] // 2 + d].detach().requires_grad_(need)
        st["w"] = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(pt).requires_grad_(need)
        st["b"] = randn(d, scale=0.2, dtype=pt).requires_grad_(need)
        if need:
            st["dy"] = randn(n, d).requires_grad_(case["mode"] == "gradgrad")
        if case["mode"] == "gradgrad":
            st["ux"], st["uw"], st["ub"] = randn(n, d), randn(d, dtype=pt), randn(d, dtype=pt)
        return st
    v = case["vocab"]
    # normalised hidden states; head weights that give logits a spread of 2.5
    st["h"] = randn(n, d).requires_grad_(need)
    st["w"] = randn(v, d, scale=2.5 / math.sqrt(d)).requires_grad_(need)
    st["targets"] = torch.randint(0, v, (n,), device="cuda", generator=g)
    if case["masked"]:
        mask = torch.zeros(n, device="cuda")
        mask[torch.randperm(n, device="cuda", generator=g)[: _kept(case)]] = 1.0
        st["mask"] = mask
    else:
        st["mask"] = None
    if need:
        # 16-bit floats of 5 exponent bits train with a scaled loss; per-token losses get per-token weights
        scale = 1024.0 if case["dtype"] == "fp16" else 1.0
        if case["reduction"] == "mean":
            st["dloss"] = torch.full((), scale, device="cuda")
        elif case["reduction"] == "sum":
            st["dloss"] = torch.full((), scale / n, device="cuda")
        else:
            st["dloss"] = (0.5 + torch.rand(n, device="cuda", generator=g)) * (scale / n)
    if case["mode"] == "gradgrad":
        st["uh"], st["uw"] = randn(n, d), randn(v, d, scale=1.0 / math.sqrt(d))
    return st


# ---------------------------------------------------------------- the framework's operators
def _run_own(st):
    from testtimeideas_b200 import layer_norm, linear_cross_entropy

    case = st["case"]
    grad = torch.autograd.grad
    second = case["mode"] == "gradgrad"
    if case["op"] == "ln":
        y = layer_norm(st["x"], st["w"], st["b"], EPS)
        if case["mode"] == "fwd":
            return {"y": y}
        dx, dw, db = grad(y, (st["x"], st["w"], st["b"]), st["dy"], create_graph=second)
        out = {"y": y.detach(), "dx": dx.detach(), "dw": dw.detach(), "db": db.detach()}
        if second:
            out["gx"], out["gw"], out["gdy"] = grad((dx, dw, db), (st["x"], st["w"], st["dy"]),
                                                    (st["ux"], st["uw"], st["ub"]))
        return out
    loss = linear_cross_entropy(st["h"], st["w"], st["targets"], st["mask"], reduction=case["reduction"])
    if case["mode"] == "fwd":
        return {"loss": loss}
    dh, dw = grad(loss, (st["h"], st["w"]), st["dloss"], create_graph=second)
    out = {"loss": loss.detach(), "dh": dh.detach(), "dw": dw.detach()}
    if second:
        out["gh"], out["gw"] = grad((dh, dw), (st["h"], st["w"]), (st["uh"], st["uw"]))
    return out


# ---------------------------------------------------------------- the plain form
def _plain_ln(st):
    case = st["case"]
    xd, pd = DTYPES[case["dtype"]], DTYPES[case["param_dtype"]]
    x, w, b = st["x"].detach().float(), st["w"].detach().float(), st["b"].detach().float()
    mu = x.mean(1, keepdim=True)
    xc = x - mu
    r = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * r
    out = {"y": (xh * w + b).to(xd)}
    if case["mode"] == "fwd":
        return out

    def project(u):
        return u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True)

    dy = st["dy"].detach().float()
    gy = dy * w
    out["dx"] = (r * project(gy)).to(xd)
    out["dw"] = (dy * xh).sum(0).to(pd)
    out["db"] = dy.sum(0).to(pd)
    if case["mode"] == "train":
        return out
    ux, uw, ub = st["ux"].float(), st["uw"].float(), st["ub"].float()
    pu = project(ux)
    a, c = (gy * xh).mean(1, keepdim=True), (ux * xh).mean(1, keepdim=True)
    s = (gy * pu).mean(1, keepdim=True)
    out["gx"] = (r * project(dy * uw - r * (c * gy + a * ux)) - r * r * s * xh).to(xd)
    out["gw"] = (dy * (r * pu)).sum(0).to(pd)
    out["gdy"] = (w * (r * pu) + xh * uw + ub).to(xd)
    return out


def _plain_lce(st):
    case = st["case"]
    dt = DTYPES[case["dtype"]]
    h, w, t, mask = st["h"].detach().float(), st["w"].detach().float(), st["targets"], st["mask"]
    n = h.shape[0]
    rows = torch.arange(n, device=h.device)
    z = h @ w.t()
    zt = z[rows, t]
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    del z
    total = p.sum(1, keepdim=True)
    ce = (top + torch.log(total))[:, 0] - zt
    weight = torch.ones(n, device=h.device) if mask is None else mask
    if case["reduction"] == "mean":
        weight = weight / weight.sum().clamp_min(1.0)
    loss = ce * weight
    if case["reduction"] != "none":
        loss = loss.sum()
    out = {"loss": loss}
    if case["mode"] == "fwd":
        return out
    p /= total
    coef = (st["dloss"] * weight)[:, None]
    gz = p * coef
    gz[rows, t] -= coef[:, 0]
    out["dh"], out["dw"] = (gz @ w).to(dt), (gz.t() @ h).to(dt)
    if case["mode"] == "train":
        return out
    uh, uw = st["uh"].float(), st["uw"].float()
    a = uh @ w.t() + h @ uw.t()
    rho = (p * a).sum(1, keepdim=True)
    dz = coef * p * (a - rho)
    out["gh"] = (dz @ w + gz @ uw).to(dt)
    out["gw"] = (dz.t() @ h + gz.t() @ uh).to(dt)
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_ln(state) if state["case"]["op"] == "ln" else _plain_lce(state)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    need = case["mode"] != "fwd"
    second = case["mode"] == "gradgrad"

    def leaf(name):
        return st[name].detach().double().requires_grad_(need)

    with torch.enable_grad():
        if case["op"] == "ln":
            x, w, b = leaf("x"), leaf("w"), leaf("b")
            var, mu = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            y = (x - mu) / torch.sqrt(var + EPS) * w + b
            if not need:
                return {"y": y}
            dy = leaf("dy")
            dx, dw, db = torch.autograd.grad(y, (x, w, b), dy, create_graph=second)
            out = {"y": y.detach(), "dx": dx.detach(), "dw": dw.detach(), "db": db.detach()}
            if second:
                up = [st[k].double() for k in ("ux", "uw", "ub")]
                out["gx"], out["gw"], out["gdy"] = torch.autograd.grad((dx, dw, db), (x, w, dy), up)
            return out
        h, w, t = leaf("h"), leaf("w"), st["targets"]
        z = torch.matmul(h, w.t())
        ce = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
        if st["mask"] is not None:
            ce = torch.where(st["mask"] != 0, ce * st["mask"].double(), torch.zeros_like(ce))
        if case["reduction"] == "mean":
            count = float(len(t)) if st["mask"] is None else max(1.0, float(st["mask"].double().sum()))
            loss = ce.sum() / count
        else:
            loss = ce.sum() if case["reduction"] == "sum" else ce
        if not need:
            return {"loss": loss}
        dh, dw = torch.autograd.grad(loss, (h, w), st["dloss"].double(), create_graph=second)
        out = {"loss": loss.detach(), "dh": dh.detach(), "dw": dw.detach()}
        if second:
            out["gh"], out["gw"] = torch.autograd.grad((dh, dw), (h, w), (st["uh"].double(), st["uw"].double()))
        return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, d, s = case["rows"], case["dim"], SIZE[case["dtype"]]
    if case["op"] == "ln":
        ps = SIZE[case["param_dtype"]]
        tensors, params, flops = {"fwd": (2, 2, 8), "train": (4, 4, 20), "gradgrad": (7, 7, 60)}[case["mode"]]
        return {"bytes": n * d * s * tensors + d * ps * params, "flops": n * d * flops}
    kept, v = _kept(case), case["vocab"]
    tensors, products = {"fwd": (1, 1), "train": (2, 3), "gradgrad": (4, 9)}[case["mode"]]
    # the masked rows are never read; their gradients are written
    rows = {"fwd": kept, "train": kept + n, "gradgrad": 2 * kept + 2 * n}[case["mode"]]
    index = n * 8 + (n * 4 if case["masked"] else 0) + (n * 4 if case["reduction"] == "none" else 4)
    return {"bytes": rows * d * s + v * d * s * tensors + index, "flops": 2 * kept * v * d * products}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c.get("name", "drawn"), c, work(c))
