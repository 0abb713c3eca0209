"""The norm and loss operators as PyTorch operators: torch.library's checks of the
raw ones, torch.compile through the public functions, CUDA graph capture, and
tensors of more than 2^31 elements."""

import pytest
import torch

import testtimeideas_b200 as tb
from testtimeideas_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    _lib.load_torch_ops()
    yield
    _lib.check_device_errors()


def _inputs(n=300, d=128, v=500, dtype=torch.bfloat16, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return {"h": r(n, d).to(dtype), "w": r(v, d).to(dtype), "lw": 1 + 0.1 * r(d), "lb": r(d),
            "t": torch.randint(0, v, (n,), generator=g, device="cuda"),
            "m": (torch.rand(n, generator=g, device="cuda") < 0.6).float()}


def test_opcheck():
    x = _inputs()
    ops = torch.ops.ttt
    check = torch.library.opcheck
    check(ops.layer_norm.default, (x["h"], x["lw"], x["lb"], 1e-5, True))
    check(ops.layer_norm.default, (x["h"], None, None, 1e-5, False))
    _, stats = ops.layer_norm(x["h"], x["lw"], x["lb"], 1e-5, True)
    dy = torch.randn_like(x["h"])
    check(ops.layer_norm_bwd.default, (dy, x["h"], x["lw"], stats, True, True, True, torch.float32))
    check(ops.layer_norm_bwd.default, (dy, x["h"], x["lw"], stats, False, True, False, torch.float32))
    check(ops.layer_norm_bwd2.default, (dy, x["h"], x["lw"], stats, dy, x["lb"], None))
    # state is bytes whose padding is never written, so only its shape and type can be compared
    for reduction in (0, 1):
        for need in (False, True):
            args = (x["h"], x["w"], x["t"], x["m"], reduction, -100, need)
            check(ops.linear_ce.default, args, test_utils=("test_schema", "test_faketensor"))
        loss, state = ops.linear_ce(*args)
        dl = torch.ones_like(loss)
        check(ops.linear_ce_bwd.default, (dl, x["h"], x["w"], state, reduction, True, True))
        check(ops.linear_ce_bwd.default, (dl, x["h"], x["w"], state, reduction, False, True))
        check(ops.linear_ce_bwd2.default, (dl, x["h"], x["w"], state, reduction, x["h"], x["w"], True, True, True))


def _loss(h, w, lw, lb, t, m):
    return tb.linear_cross_entropy(tb.layer_norm(h, lw, lb), w, t, m)


def _leaves(x):
    return [x[k].clone().requires_grad_(True) for k in ("h", "w", "lw", "lb")]


def test_compiled_matches_eager():
    x = _inputs(seed=2)
    f = torch.compile(_loss, fullgraph=True)
    with torch.no_grad():
        args = [x[k] for k in ("h", "w", "lw", "lb")]
        assert torch.equal(f(*args, x["t"], x["m"]), _loss(*args, x["t"], x["m"]))
    res = []
    for fn in (f, _loss):
        p = _leaves(x)
        res.append(torch.autograd.grad(fn(*p, x["t"], x["m"]), p))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("second", [False, True])
def test_captured_in_a_cuda_graph(second):
    """Forward, gradient and second gradient record into a graph; a replay on new inputs gives what
    the eager call gives (no result and no size is baked in, the number of kept rows included)."""
    x, y = _inputs(seed=3), _inputs(seed=4)
    p = _leaves(x)
    t, m = x["t"].clone(), x["m"].clone()

    def step():
        loss = _loss(*p, t, m)
        g = torch.autograd.grad(loss, p, create_graph=second)
        if second:
            g = g + torch.autograd.grad([gi.float().square().sum() for gi in g], p)
        return [loss.detach()] + [gi.detach() for gi in g]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    y["m"] = (torch.arange(300, device="cuda") % 7 == 0).float()  # far fewer rows
    with torch.no_grad():
        for leaf, k in zip(p, ("h", "w", "lw", "lb")):
            leaf.copy_(y[k])
        t.copy_(y["t"])
        m.copy_(y["m"])
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in out]
    ref = step()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_score_of_a_token_in_a_cuda_graph():
    x = _inputs(n=1, d=256, v=3000, seed=5)
    with torch.no_grad():
        ref = tb.linear_cross_entropy(x["h"], x["w"], x["t"], reduction="none")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tb.linear_cross_entropy(x["h"], x["w"], x["t"], reduction="none")
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_layer_norm_past_32_bit_offsets():
    """2^31 + elements: the last rows equal those of a small call on them."""
    n, d = 131075, 16384
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    x.normal_(generator=g)
    w, b = torch.randn(d, device="cuda", generator=g), torch.randn(d, device="cuda", generator=g)
    dy = x.detach()  # the upstream gradient may share x's storage
    x.requires_grad_(True)
    y = tb.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    tail = x.detach()[-64:].clone().requires_grad_(True)
    yt = tb.layer_norm(tail, w, b)
    dt, = torch.autograd.grad(yt, tail, tail.detach())
    assert torch.equal(y[-64:], yt) and torch.equal(dx[-64:], dt)


def test_vocabulary_past_32_bit_offsets():
    """A weight of 2^31 + elements: loss, hidden gradient and the last rows of the weight gradient
    against float64 over the whole vocabulary (in pieces)."""
    n, d, v = 4, 4096, 530000
    g = torch.Generator(device="cuda").manual_seed(7)
    h = torch.randn(n, d, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_(std=2.5 / d**0.5, generator=g)
    t = torch.tensor([0, v - 1, v - 2, 12345], device="cuda")
    hd = h.double()
    z = torch.cat([hd @ c.double().t() for c in w.split(65536)], 1)
    lse = torch.logsumexp(z, 1)
    ref = (lse - z.gather(1, t[:, None])[:, 0])
    p = torch.exp(z - lse[:, None])
    p[torch.arange(n), t] -= 1
    ref_dh = sum(p[:, i:i + 65536] @ w[i:i + 65536].double() for i in range(0, v, 65536))
    ref_dw = p[:, -300:].t() @ hd
    with torch.no_grad():
        score = tb.linear_cross_entropy(h, w, t, reduction="none")
    hh, ww = h.requires_grad_(True), w.requires_grad_(True)
    loss = tb.linear_cross_entropy(hh, ww, t, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (hh, ww))
    # fp32 sums of 4096 products of |z| < 16 (and their truncation in the tensor cores)
    assert float((score.double() - ref).abs().max()) <= 2e-4
    assert abs(float(loss.detach().double() - ref.sum())) <= 4 * 2e-4
    tol = 4 * 2.0**-9  # as in test_gpu_linear_ce.py
    assert float((dh.double() - ref_dh).abs().max() / ref_dh.abs().max()) <= tol
    assert float((dw[-300:].double() - ref_dw).abs().max() / ref_dw.abs().max()) <= tol


def test_gradients_refuse_what_is_not_the_forwards():
    """The bytes and statistics that a gradient reads: not those of a forward without them, of another
    size, type or device, or strided."""
    x, ops = _inputs(n=5, d=64, v=90), torch.ops.ttt
    for n in (5, 2):  # the second takes the path of a few rows
        h, t = x["h"][:n], x["t"][:n]
        loss, none = ops.linear_ce(h, x["w"], t, None, 1, -100, False)
        _, state = ops.linear_ce(h, x["w"], t, None, 1, -100, True)
        assert none.numel() == 0 and none.dtype == state.dtype
        one = torch.ones_like(loss)
        for bad in (none, state[:-256], state.cpu(), state.float(), state.repeat_interleave(2)[::2]):
            with pytest.raises(RuntimeError, match="state must be"):
                ops.linear_ce_bwd(one, h, x["w"], bad, 1, True, True)
            with pytest.raises(RuntimeError, match="state must be"):
                ops.linear_ce_bwd2(one, h, x["w"], bad, 1, h, x["w"], True, True, True)
    _, stats = ops.layer_norm(x["h"], None, None, 1e-5, True)
    _, none = ops.layer_norm(x["h"], None, None, 1e-5, False)
    for bad in (none, stats[:, :4], stats.cpu(), stats.double(), stats.repeat_interleave(2, 1)[:, ::2]):
        with pytest.raises(RuntimeError, match="stats must be"):
            ops.layer_norm_bwd(x["h"], x["h"], None, bad, True, False, False, torch.bfloat16)
        with pytest.raises(RuntimeError, match="stats must be"):
            ops.layer_norm_bwd2(x["h"], x["h"], None, bad, x["h"], None, None)


def test_gradients_do_not_copy_hidden():
    """The gradients read the rows that the forward gathered; a transposed hidden costs them no copy."""
    x, ops = _inputs(n=4096, d=512, v=600, seed=8), torch.ops.ttt
    loss, state = ops.linear_ce(x["h"], x["w"], x["t"], None, 1, -100, True)
    one = torch.ones_like(loss)
    peaks, outs = [], []
    for h in (x["h"], x["h"].t().contiguous().t()):
        for call in (lambda: ops.linear_ce_bwd(one, h, x["w"], state, 1, True, True),
                     lambda: ops.linear_ce_bwd2(one, h, x["w"], state, 1, x["h"], x["w"], True, True, True)):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            outs.append(call())
            torch.cuda.synchronize()
            peaks.append(torch.cuda.max_memory_allocated() - before)
    assert peaks[:2] == peaks[2:]
    assert all(torch.equal(a, b) for i in (0, 1) for a, b in zip(outs[i], outs[i + 2]))


def test_gradients_refuse_a_state_of_other_rows():
    x, ops = _inputs(n=6, d=64, v=90), torch.ops.ttt
    loss, state = ops.linear_ce(x["h"][:5], x["w"], x["t"][:5], None, 1, -100, True)
    for n in (4, 6):
        h = x["h"][:n]
        with pytest.raises(RuntimeError, match="state must be"):
            ops.linear_ce_bwd(torch.ones_like(loss), h, x["w"], state, 1, True, True)
        with pytest.raises(RuntimeError, match="state must be"):
            ops.linear_ce_bwd2(torch.ones_like(loss), h, x["w"], state, 1, h, x["w"], True, True, True)
