"""Layer norm kernels (forward, gradient, gradient of the gradient) against the
definition in float64, at widths around every boundary of the row layouts, for
each type, with strided, broadcast, misaligned and empty inputs, rows with large
offsets, and rows that hold infinities or NaN.

Tolerances (normalized by the largest reference magnitude): an output is fp32
arithmetic rounded once, so half a unit in the last place of its type (2^-11
fp16, 2^-9 bf16), doubled for the fp32 part; fp32 outputs sum up to 16384 terms
with errors that add up like a random walk: 128 * 2^-24 ~ 8e-6, doubled."""

import pytest
import torch

import testtimeideas_b200 as tb
from testtimeideas_b200 import _lib

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 2.0**-10, torch.bfloat16: 2.0**-8, torch.float32: 1.6e-5}
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _library():
    _lib.load_library()
    yield
    _lib.check_device_errors()


def _inputs(n, d, dtype, p_dtype, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": (r(n, d) + offset).to(dtype), "w": (1 + 0.3 * r(d)).to(p_dtype), "b": r(d).to(p_dtype),
            "dy": r(n, d).to(dtype), "ux": r(n, d).to(dtype), "uw": r(d).to(p_dtype), "ub": r(d).to(p_dtype)}


def _definition(x, w, b):
    var, mu = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mu) / torch.sqrt(var + EPS)
    return y * (1 if w is None else w) + (0 if b is None else b)


def _all(fn, x, w, b, dy, ux, uw, ub):
    """y, first and second gradients of fn at the given (leaf) tensors."""
    x, w, b, dy = (None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, dy))
    ps = [t for t in (x, w, b) if t is not None]
    y = fn(x, w, b)
    g1 = torch.autograd.grad(y, ps, dy, create_graph=True)
    ups = [u for t, u in ((x, ux), (w, uw), (b, ub)) if t is not None]
    g2 = torch.autograd.grad(g1, [t for t in (x, w, dy) if t is not None], ups, allow_unused=True)
    names = ["y"] + ["d" + n for n, t in (("x", x), ("w", w), ("b", b)) if t is not None]
    names += ["g" + n for n, t in (("x", x), ("w", w), ("dy", dy)) if t is not None]
    return dict(zip(names, (t.detach() for t in (y, *g1, *g2))))


def _compare(got, ref, tol=None):
    assert set(got) == set(ref)
    for name, x in got.items():
        r = ref[name]
        assert x.shape == r.shape, name
        if r.numel() == 0:
            continue
        bound = tol or TOL[x.dtype]
        err = (x.double().cpu() - r).abs().max() / r.abs().max().clamp_min(1e-30)
        assert err <= bound, f"{name}: {err:.3e} > {bound:.1e}"


def _check(inp, **over):
    inp = {**inp, **over}
    got = _all(lambda x, w, b: tb.layer_norm(x, w, b, EPS), **{k: None if v is None else v.cuda() for k, v in inp.items()})
    ref = _all(_definition, **{k: None if v is None else v.double().cpu() for k, v in inp.items()})
    _compare(got, ref)
    for k in ("y", "dx", "gx"):
        assert got[k].dtype == inp["x"].dtype
    return got


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]
DIMS = (1, 7, 8, 64, 255, 256, 257, 512, 513, 768, 1000, 1024, 1025, 2048, 2049, 4096, 4100, 8192, 8200, 16384)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("d", DIMS)
def test_widths(d, types):
    # d = 1 has zero variance everywhere: y = b exactly and every x gradient is 0
    inp = _inputs(37, d, *types, seed=d)
    if d == 1:
        got = tb.layer_norm(inp["x"].cuda(), inp["w"].cuda(), inp["b"].cuda(), EPS)
        assert torch.equal(got.cpu(), inp["b"].expand(37, 1).to(got.dtype))
        return
    _check(inp)


@pytest.mark.parametrize("n", (1, 2, 8, 9, 2401, 5000))
@pytest.mark.parametrize("d", (96, 768, 1500))
def test_row_counts(n, d):
    _check(_inputs(n, d, torch.bfloat16, torch.float32, seed=n + d))


def test_no_rows():
    x = torch.empty(3, 0, 768, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(768, device="cuda", requires_grad=True)
    y = tb.layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("d", (4096, 5001, 8200, 9001, 9002, 16384))
def test_several_wide_rows_a_block(d, dtype):
    # more rows than blocks that fit on the SMs: the column sums run over a block's rows
    _check(_inputs(640, d, dtype, dtype, seed=d))


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_optional_parameters(weight, bias):
    inp = _inputs(40, 300, torch.float16, torch.float16, seed=3)
    over = {}
    if not weight:
        over.update(w=None, uw=None)
    if not bias:
        over.update(b=None, ub=None)
    _check(inp, **over)


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("d", (96, 301, 2050))
def test_fp32_bias_alone(dtype, d):
    """A bias in fp32 beside 16-bit x and no weight: the gradients take its upstream gradient as it is. ub
    nearly cancels the rest of gdy here (one row), so that rounding it first would show: what is left
    is 1e-2 of it, and carries a few fp32 roundings of terms near 4 (2e-6) and its own."""
    inp = {**_inputs(1, d, dtype, torch.float32, seed=d), "w": None, "uw": None}
    _check(inp)
    with_zero = {k: None if v is None else v.double() for k, v in inp.items()}
    with_zero["ub"] = torch.zeros_like(with_zero["ub"])
    rest = _all(_definition, **with_zero)["gdy"][0]
    small = 1e-2 * torch.randn(d, generator=torch.Generator().manual_seed(d), dtype=torch.float64)
    got = _check(inp, ub=(small - rest).float())
    assert float(got["gdy"].abs().max()) < 0.1


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_layouts(dtype):
    """Row slices, misaligned starts, a broadcast row, transposed storage, broadcast upstream gradients."""
    inp = _inputs(64, 520, dtype, dtype, seed=9)
    wide = torch.randn(64, 533, dtype=torch.float32).to(dtype).cuda()
    d = 520
    for x in (wide[:, :d], wide[:, 3:3 + d], wide[:, 8:8 + d], wide[:1, :d].expand(64, d),
              torch.randn(d, 64).to(dtype).cuda().t(), wide[::2, :d].repeat(2, 1)[::1]):
        ref = _all(_definition, x.double().cpu(), *(inp[k].double() for k in ("w", "b", "dy", "ux", "uw", "ub")))
        xs = x.detach().requires_grad_(True)
        w, b, dy = (inp[k].cuda().requires_grad_(True) for k in ("w", "b", "dy"))
        y = tb.layer_norm(xs, w, b, EPS)
        g1 = torch.autograd.grad(y, (xs, w, b), dy, create_graph=True)
        g2 = torch.autograd.grad(g1, (xs, w, dy), [inp[k].cuda() for k in ("ux", "uw", "ub")])
        _compare(dict(zip(("y", "dx", "dw", "db", "gx", "gw", "gdy"), (t.detach() for t in (y, *g1, *g2)))), ref)
    # y.sum(): the upstream gradient is a broadcast scalar
    x = inp["x"].cuda().requires_grad_(True)
    w = inp["w"].cuda().requires_grad_(True)
    dx, dw = torch.autograd.grad(tb.layer_norm(x, w, None, EPS).sum(), (x, w))
    xr, wr = inp["x"].double().requires_grad_(True), inp["w"].double().requires_grad_(True)
    rx, rw = torch.autograd.grad(_definition(xr, wr, None).sum(), (xr, wr))
    _compare({"dx": dx, "dw": dw}, {"dx": rx, "dw": rw})


@pytest.mark.parametrize("d", (64, 258, 301, 520, 768, 2050, 9002))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_parameters_inside_a_flat_buffer(dtype, d):
    """16-bit weight, bias and their upstream gradients as slices at odd and even offsets: aligned
    rows beside parameters on 2-byte, 4-byte and 8-byte boundaries, alone and together."""
    inp = _inputs(70, d, dtype, dtype, seed=d)
    names = ("w", "b", "uw", "ub")

    def at(v, off):
        flat = torch.zeros(d + 16, dtype=dtype, device="cuda")
        flat[off:off + d] = v.cuda()
        return flat[off:off + d]

    for off in (1, 2, 4, 7):
        for moved in (names, ("w",), ("b",), ("uw",), ("ub",)):
            _check(inp, **{k: at(inp[k], off) for k in moved})


def test_batched_shape():
    inp = _inputs(24, 128, torch.bfloat16, torch.bfloat16, seed=1)
    x = inp["x"].cuda()
    y = tb.layer_norm(x.view(2, 3, 4, 128), inp["w"].cuda(), inp["b"].cuda())
    assert torch.equal(y.view(24, 128), tb.layer_norm(x, inp["w"].cuda(), inp["b"].cuda()))


def test_large_offsets():
    """Rows at 1000 +- 1 in fp32: the variance is a sum of squared differences, not a difference of
    sums. Inputs carry 2^-14 of absolute error relative to their spread, so the definition is taken
    at the rounded inputs; fp32 differences from a mean near 1000 are exact to 2^-14."""
    inp = _inputs(50, 1000, torch.float32, torch.float32, seed=4, offset=1000.0)
    got = _all(lambda x, w, b: tb.layer_norm(x, w, b, EPS), **{k: v.cuda() for k, v in inp.items()})
    ref = _all(_definition, **{k: v.double() for k, v in inp.items()})
    _compare(got, ref, tol=4 * 2.0**-14)


def test_nonfinite_rows_stay_in_their_rows():
    inp = _inputs(16, 300, torch.float32, torch.float32, seed=5)
    bad = inp["x"].clone()
    bad[3, 7], bad[5, 0], bad[9] = float("nan"), float("inf"), float("-inf")
    x, w, dy = bad.cuda().requires_grad_(True), inp["w"].cuda(), inp["dy"].cuda()
    y = tb.layer_norm(x, w, None, EPS)
    dx, = torch.autograd.grad(y, x, dy)
    rows = torch.ones(16, dtype=torch.bool)
    rows[[3, 5, 9]] = False
    assert y[~rows].isnan().any(1).all() and dx[~rows].isnan().any(1).all()
    xr = inp["x"].double().requires_grad_(True)
    yr = _definition(xr, inp["w"].double(), None)
    dr, = torch.autograd.grad(yr, xr, inp["dy"].double())
    _compare({"y": y.detach()[rows], "dx": dx[rows]}, {"y": yr.detach()[rows], "dx": dr[rows]})


def test_gradients_against_differences():
    """<gradient, direction> against central differences of the definition in float64."""
    inp = _inputs(12, 96, torch.float32, torch.float32, seed=6)
    x, w, b, dy = (inp[k].cuda().requires_grad_(True) for k in ("x", "w", "b", "dy"))
    up = [inp[k].cuda() for k in ("ux", "uw", "ub")]
    y = tb.layer_norm(x, w, b, EPS)
    g1 = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    g2 = torch.autograd.grad(g1, (x, w, dy), up)
    d64 = {k: v.double() for k, v in inp.items()}
    gen = torch.Generator().manual_seed(7)
    dirs = {k: torch.randn(d64[k].shape, generator=gen, dtype=torch.float64) for k in ("x", "w", "dy")}

    def first(x, w, dy):  # <y, dy>
        return (_definition(x, w, d64["b"]) * dy).sum()

    def second(x, w, dy):  # <dx, ux> + <dw, uw> + <db, ub>
        x, w, b = (t.detach().requires_grad_(True) for t in (x, w, d64["b"]))
        gs = torch.autograd.grad(_definition(x, w, b), (x, w, b), dy)
        return sum((g * d64[u]).sum() for g, u in zip(gs, ("ux", "uw", "ub")))

    h = 1e-5
    for f, grads in ((first, {"x": g1[0], "w": g1[1]}), (second, {"x": g2[0], "w": g2[1], "dy": g2[2]})):
        for k, grad in grads.items():
            at = {n: d64[n] for n in ("x", "w", "dy")}
            plus, minus = dict(at), dict(at)
            plus[k], minus[k] = at[k] + h * dirs[k], at[k] - h * dirs[k]
            num = (f(**plus) - f(**minus)) / (2 * h)
            ana = (grad.detach().double().cpu() * dirs[k]).sum()
            # differences: h^2 truncation and 1e-16 / h rounding ~ 1e-9; the kernel: fp32 sums over 1152 terms
            assert abs(num - ana) <= 1e-4 * max(1.0, abs(num)), (k, float(num), float(ana))


def test_runs_agree_and_streams():
    """Bitwise equal results from run to run and from a side stream."""
    inp = {k: v.cuda() for k, v in _inputs(3000, 768, torch.bfloat16, torch.float32, seed=8).items()}
    one = _all(lambda x, w, b: tb.layer_norm(x, w, b, EPS), **inp)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = _all(lambda x, w, b: tb.layer_norm(x, w, b, EPS), **inp)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(one[k], two[k]) for k in one)


def test_third_derivative_raises():
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(tb.layer_norm(x).square().sum(), x, create_graph=True)
    gx, = torch.autograd.grad(dx.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


def test_module_matches_torch_parameters():
    m = tb.LayerNorm(128).cuda().to(torch.bfloat16)
    m.load_state_dict(torch.nn.LayerNorm(128).state_dict())
    x = torch.randn(5, 128, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        y = m(x)
    ref = _definition(x.double().cpu(), None, None)
    _compare({"y": y}, {"y": ref})


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        tb.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="must be \\[64\\]"):
        tb.layer_norm(x, w[:32])
    with pytest.raises(RuntimeError, match="x's dtype or fp32"):
        tb.layer_norm(x, w.half())
    with pytest.raises(RuntimeError, match="share one dtype"):
        tb.layer_norm(x.half(), w.half(), w)
    with pytest.raises(RuntimeError, match="device"):
        tb.layer_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="at most"):
        tb.layer_norm(torch.randn(1, 16385, device="cuda"))
    with pytest.raises(RuntimeError, match="last dimension"):
        tb.layer_norm(torch.empty(3, 0, device="cuda"))
