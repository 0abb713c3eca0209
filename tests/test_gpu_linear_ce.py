"""Linear cross entropy kernels (loss, gradient, gradient of the gradient) against
the definition in float64: sizes around the tile sides, odd widths and
vocabularies, each reduction and mask kind, rows left out by mask or ignored
target (with NaN in them), strided and broadcast inputs, more than one piece of
the vocabulary, small probabilities in fp16, empty problems and refusals.

Tolerances, normalized by the largest reference magnitude. u is half a unit in
the last place of the type (2^-11 fp16, 2^-9 bf16). The stored derivative G is
rounded once (u per term) and its absolute row sum is at most twice its target
entry, so dh and dw carry at most 2u from it, u from their own rounding and a
little from fp32: 4u. The second gradient sums two such products with
independent terms: 8u. Losses are fp32: |z| < 16 with sums of at most 600
products, 600 * 2^-24 of 16 in the worst case and its root on average: 2e-5."""

import pytest
import torch

import testtimeideas_b200 as tb
from testtimeideas_b200 import _lib

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-9}
LOSS_TOL = 2e-5


@pytest.fixture(scope="module", autouse=True)
def _library():
    _lib.load_library()
    yield
    _lib.check_device_errors()


def _inputs(n, d, v, dtype, seed, spread=2.5, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"h": r(n, d).to(dtype).cuda(), "w": (r(v, d) * spread / d**0.5).to(dtype).cuda(),
            "t": torch.randint(0, v, (n,), generator=g).cuda(), "uh": (r(n, d) * scale).to(dtype).cuda(),
            "uw": (r(v, d) * scale / d**0.5).to(dtype).cuda()}


def _mask(n, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind is None:
        return None
    if kind == "bool":
        return (torch.rand(n, generator=g) < 0.7).cuda()
    if kind == "weights":
        m = torch.rand(n, generator=g) * 2
        m[torch.rand(n, generator=g) < 0.3] = 0.0
        return m.cuda()
    return torch.zeros(n).cuda() if kind == "none" else torch.ones(n).cuda()


def _definition(h, w, t, m, reduction, ignore=-100):
    """float64, rows left out removed before anything is computed."""
    weight = torch.ones(t.shape, dtype=torch.float64, device=h.device) if m is None else m.double()
    keep = (weight != 0) & (t != ignore)
    hk, tk = h[keep], t[keep]
    z = hk @ w.t()
    ce = (torch.logsumexp(z, 1) - z.gather(1, tk[:, None])[:, 0]) * weight[keep]
    if reduction == "none":
        return torch.zeros(t.shape, dtype=torch.float64, device=h.device).masked_scatter(keep, ce)
    if reduction == "sum":
        return ce.sum()
    return ce.sum() / (max(t.numel(), 1) if m is None else weight.sum().clamp_min(1.0))


def _all(fn, h, w, dloss, uh, uw):
    """loss, first gradients, second gradients (with the one by dloss) of fn(h, w)."""
    h, w, dloss = (x.detach().requires_grad_(True) for x in (h, w, dloss))
    loss = fn(h, w)
    dh, dw = torch.autograd.grad(loss, (h, w), dloss, create_graph=True)
    ups = [(g, u) for g, u in ((dh, uh), (dw, uw)) if u is not None]
    gh, gw, gd = torch.autograd.grad([g for g, _ in ups], (h, w, dloss), [u for _, u in ups])
    names = ("loss", "dh", "dw", "gh", "gw", "gd")
    return dict(zip(names, (x.detach() for x in (loss, dh, dw, gh, gw, gd))))


def _norm(x, r, floor=1e-30):
    return float((x.double() - r).abs().max() / r.abs().max().clamp_min(floor))


def _compare(got, ref, dtype, row_scale=None):
    u = U[dtype]
    assert abs(got["loss"].double() - ref["loss"]).max() <= LOSS_TOL * max(1.0, float(ref["loss"].abs().max()))
    for name, tol in (("dh", 4 * u), ("dw", 4 * u), ("gh", 8 * u), ("gw", 8 * u)):
        assert got[name].dtype == dtype and got[name].shape == ref[name].shape
        assert torch.equal(got[name].isnan(), ref[name].isnan()), name
        if ref[name].numel():
            err = _norm(got[name], ref[name])
            assert err <= tol, f"{name}: {err:.3e} > {tol:.1e}"
    # each row's rho - A_t is an fp32 sum of terms up to row_scale; a scalar adds n of them
    if row_scale is not None:
        assert float((got["gd"].double() - ref["gd"]).abs().max()) <= 1e-5 * row_scale


def _check(inp, m=None, reduction="mean", ignore=-100, uh=True, uw=True, up=1.0):
    h, w, t = inp["h"], inp["w"], inp["t"]
    dtype = h.dtype
    dloss = torch.full((), up, device="cuda")
    if reduction == "none":
        dloss = up * torch.linspace(0.5, 1.5, t.numel(), device="cuda").view(t.shape)
    uh, uw = inp["uh"] if uh else None, inp["uw"] if uw else None
    got = _all(lambda h, w: tb.linear_cross_entropy(h, w, t, m, reduction=reduction, ignore_index=ignore), h, w, dloss,
               uh, uw)
    ref = _all(lambda h, w: _definition(h, w, t, m, reduction, ignore), h.double(), w.double(), dloss.double(),
               None if uh is None else uh.double(), None if uw is None else uw.double())
    a = 0.0
    if uh is not None:
        a = a + uh.double() @ w.double().t()
    if uw is not None:
        a = a + h.double() @ uw.double().t()
    a = a[torch.isfinite(a).all(1)]
    scale = float(a.abs().max()) if a.numel() else 1.0
    if reduction == "sum":
        scale *= t.numel()
    _compare(got, ref, dtype, row_scale=2 * scale * (2.0 if m is not None else 1.0))
    return got


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("n,d,v", [
    (1, 64, 256), (1, 8, 1), (2, 1, 3), (3, 13, 7), (5, 100, 101), (17, 72, 127), (64, 128, 128), (127, 64, 129),
    (128, 63, 255), (129, 65, 256), (130, 512, 257), (200, 256, 513), (256, 264, 1000), (300, 520, 2049),
    (1, 512, 5000), (511, 96, 4096), (1000, 333, 777)])
def test_sizes(n, d, v, dtype):
    _check(_inputs(n, d, v, dtype, seed=n + d + v), up=64.0)


@pytest.mark.parametrize("mask", (None, "bool", "weights", "none", "ones"))
@pytest.mark.parametrize("reduction", ("mean", "sum", "none"))
def test_masks_and_reductions(mask, reduction):
    n = 333
    inp = _inputs(n, 96, 700, torch.bfloat16, seed=11)
    inp["t"][::7] = -100
    inp["t"][5::11] = 4
    got = _check(inp, _mask(n, mask, seed=12), reduction)
    if mask == "none":
        assert float(got["loss"].abs().max()) == 0.0
        for k in ("dh", "dw", "gh", "gw", "gd"):
            assert not got[k].any(), k
    # another ignored value, inside the vocabulary
    _check(inp | {"t": inp["t"].clamp_min(0)}, _mask(n, mask, seed=13), reduction, ignore=4)


@pytest.mark.parametrize("uh,uw", [(True, False), (False, True)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_one_upstream_only(uh, uw, dtype):
    _check(_inputs(150, 200, 600, dtype, seed=3), _mask(150, "bool", 4), uh=uh, uw=uw, up=128.0)


def test_rows_left_out_are_not_read():
    """NaN and infinities in rows without weight or with an ignored target change no bit."""
    n = 260
    inp = _inputs(n, 136, 500, torch.bfloat16, seed=21)
    m = _mask(n, "weights", seed=22)
    inp["t"][3::17] = -100
    out = (m == 0) | (inp["t"] == -100)
    assert 0 < int(out.sum()) < n
    clean = _check(inp, m)
    dirty = dict(inp)
    for k in ("h", "uh"):
        dirty[k] = inp[k].clone()
        dirty[k][out] = float("nan")
        dirty[k][out.nonzero()[0]] = float("inf")
    # a target that is out of range does not matter either where the mask is 0
    dirty["t"] = torch.where(m == 0, torch.full_like(inp["t"], 10**9), inp["t"])
    dl = torch.ones((), device="cuda")
    got = _all(lambda h, w: tb.linear_cross_entropy(h, w, dirty["t"], m), dirty["h"], dirty["w"], dl, dirty["uh"],
               dirty["uw"])
    for k in ("loss", "dh", "dw", "gh", "gw"):
        assert torch.equal(got[k], _all(lambda h, w: tb.linear_cross_entropy(h, w, inp["t"], m), inp["h"], inp["w"],
                                        dl, inp["uh"], inp["uw"])[k]), k
    assert not got["dh"][out].any() and not got["gh"][out].any()
    _lib.check_device_errors()
    assert clean


def test_nonfinite_row_that_takes_part():
    """A NaN row makes its loss and the weight gradient NaN, and no other row's hidden gradient."""
    inp = _inputs(140, 64, 300, torch.bfloat16, seed=23)
    h = inp["h"].clone()
    h[131] = float("nan")
    h = h.requires_grad_(True)
    loss = tb.linear_cross_entropy(h, inp["w"], inp["t"], reduction="none")
    dh, = torch.autograd.grad(loss, h, torch.ones_like(loss))
    ref = tb.linear_cross_entropy(inp["h"], inp["w"], inp["t"], reduction="none")
    assert loss[131].isnan() and dh[131].isnan().all()
    rows = torch.arange(140, device="cuda") != 131
    assert torch.equal(loss[rows], ref[rows]) and not dh[rows].isnan().any()


def test_layouts():
    """[b, t, d] hidden states, row slices, a broadcast row, weights with padded, misaligned and transposed rows."""
    inp = _inputs(96, 128, 400, torch.float16, seed=31)
    base = _check(inp, up=32.0)
    fn = lambda h, w, t=inp["t"]: tb.linear_cross_entropy(h, w, t)  # noqa: E731
    dl = torch.full((), 32.0, device="cuda")

    def same(h, w, uh=inp["uh"], uw=inp["uw"]):
        got = _all(fn, h, w, dl, uh, uw)
        for k in base:
            assert torch.equal(got[k], base[k]), k

    h, w = inp["h"], inp["w"]
    wide = torch.zeros(96, 150, dtype=h.dtype, device="cuda")
    for off in (0, 3, 8):
        wide[:, off:off + 128] = h
        same(wide[:, off:off + 128], w)
        wbuf = torch.zeros(400, 150, dtype=w.dtype, device="cuda")
        wbuf[:, off:off + 128] = w
        same(h, wbuf[:, off:off + 128], uw=wbuf.clone()[:, off:off + 128] * 0 + inp["uw"])
    same(h.t().contiguous().t(), w.t().contiguous().t(), uh=inp["uh"].t().contiguous().t())
    got = _all(lambda h, w: tb.linear_cross_entropy(h, w, inp["t"].view(4, 24)), h.view(4, 24, 128), w, dl,
               inp["uh"].view(4, 24, 128), inp["uw"])
    assert all(torch.equal(got[k].reshape(base[k].shape), base[k]) for k in base)
    # a broadcast hidden state: autograd sums the rows' gradients
    one = h[:1].clone().requires_grad_(True)
    g1, = torch.autograd.grad(tb.linear_cross_entropy(one.expand(96, 128), w, inp["t"]), one)
    d1 = h[:1].double().requires_grad_(True)
    r1, = torch.autograd.grad(_definition(d1.expand(96, 128), w.double(), inp["t"], None, "mean"), d1)
    assert _norm(g1, r1) <= 8 * U[torch.float16]
    # 32-bit targets
    assert torch.equal(tb.linear_cross_entropy(h, w, inp["t"].int()), base["loss"])


def test_more_than_one_piece():
    """512 MB of stored derivatives hold 3824 columns of 70016 rows: the 4096 columns take two pieces
    (the second gradient, with two arrays, also), and dh is summed over them."""
    inp = _inputs(70000, 24, 4096, torch.bfloat16, seed=41)
    _check(inp, _mask(70000, "bool", 42), "sum", up=1.0)


@pytest.mark.parametrize("n,d,v", [(32768, 64, 253953), (16384, 24, 253953), (16384, 512, 262208)])
def test_last_piece_shorter_than_its_shares(n, d, v):
    """The hidden gradient is cut into shares of a piece's columns, two (or three) here, and the last
    piece is a single column (or 64): shares without columns leave the sums alone. First gradient for
    the first size, second for the others. Few rows are kept, which the plan does not look at."""
    inp = _inputs(n, d, v, torch.bfloat16, seed=v + d)
    m = torch.zeros(n, device="cuda")
    m[:: n // 130] = 1.0
    dl = torch.full((), 64.0, device="cuda")
    got = _all(lambda h, w: tb.linear_cross_entropy(h, w, inp["t"], m), inp["h"], inp["w"], dl, inp["uh"], inp["uw"])
    ref = _all(lambda h, w: _definition(h, w, inp["t"], m, "mean"), inp["h"].double(), inp["w"].double(), dl.double(),
               inp["uh"].double(), inp["uw"].double())
    _compare(got, ref, torch.bfloat16)
    _lib.check_device_errors()


def test_few_rows_split_the_vocabulary():
    """One token tile, a long vocabulary: the dh product is shared between CTAs."""
    _check(_inputs(3, 160, 40000, torch.bfloat16, seed=43), up=4.0)


def test_small_probabilities_in_fp16():
    """Probabilities near 1e-9: G stays normal in fp16 because of its power-of-two scale, so the dw of a
    vocabulary entry that is no row's target is still right to fp16 (times an upstream scale that
    keeps dw itself normal)."""
    n, d, v = 64, 64, 512
    inp = _inputs(n, d, v, torch.float16, seed=44, spread=0.0)
    h = inp["h"].abs() + 0.5
    w = torch.zeros(v, d, dtype=torch.float16, device="cuda")
    w[0] = 20.0 / d**0.5 / 0.8  # logit of entry 0: about 20 above the others
    inp = dict(inp, h=h, w=w, t=torch.zeros(n, dtype=torch.long, device="cuda"))
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(tb.linear_cross_entropy(hh, ww, inp["t"], reduction="sum"), ww,
                              torch.full((), 2.0**20, device="cuda"))
    wd = w.double().requires_grad_(True)
    rw, = torch.autograd.grad(_definition(h.double(), wd, inp["t"], None, "sum"), wd,
                              torch.full((), 2.0**20, device="cuda", dtype=torch.float64))
    p = torch.softmax(h.double() @ w.double().t(), 1)[:, 1:].max()
    assert float(p) < 1e-6
    assert _norm(dw[1:], rw[1:]) <= 4 * U[torch.float16]


@pytest.mark.parametrize("n,d,v", [(1, 8, 1), (1, 768, 32000), (2, 512, 63), (3, 8192, 65), (4, 1000, 4097),
                                   (4, 100, 300), (5, 256, 1000), (1, 8200, 500)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_scores_without_gradients(n, d, v, dtype):
    """Few rows without gradients (their own kernel up to four) agree with the definition and with
    the path that keeps state, for each reduction, with a row left out and NaN in it."""
    inp = _inputs(n, d, v, dtype, seed=n + d + v)
    h = inp["h"].clone()
    for mask in (None, "bool", "weights", "none"):
        m = _mask(n, mask, seed=n)
        if m is not None and mask != "none":
            m[0] = 1
            if n > 2:
                m[1] = 0
                h[1] = float("nan")
        for reduction in ("none", "mean", "sum"):
            loss = tb.linear_cross_entropy(h, inp["w"], inp["t"], m, reduction=reduction)
            ref = _definition(inp["h"].double(), inp["w"].double(), inp["t"], m, reduction)
            assert loss.shape == ref.shape
            # up to 8192 products of |z| < 16 in fp32: 2^-24 sqrt(8192) 16 on average, as in LOSS_TOL
            assert float((loss.double() - ref).abs().max()) <= 5 * LOSS_TOL * max(1.0, float(ref.abs().max()))
            kept = tb.linear_cross_entropy(h.clone().requires_grad_(True), inp["w"], inp["t"], m, reduction=reduction)
            assert float((loss - kept.detach()).abs().max()) <= 5 * LOSS_TOL * max(1.0, float(ref.abs().max()))
        h = inp["h"].clone()
    t = inp["t"].clone()
    t[n - 1] = v
    tb.linear_cross_entropy(inp["h"], inp["w"], t)
    with pytest.raises(_lib.KernelError, match="target outside"):
        _lib.check_device_errors()


def test_large_logits():
    """Logits of several hundred: the running maximum keeps the exponentials finite; u per unit of logit
    error does not enter, as z is exact products summed in fp32 (256 * 2^-24 * 400 < 0.01 absolute)."""
    inp = _inputs(100, 256, 900, torch.bfloat16, seed=45, spread=100.0)
    loss = tb.linear_cross_entropy(inp["h"], inp["w"], inp["t"], reduction="none")
    ref = _definition(inp["h"].double(), inp["w"].double(), inp["t"], None, "none")
    assert float((loss.double() - ref).abs().max()) <= 0.01


def test_gradients_against_differences():
    inp = _inputs(20, 40, 60, torch.float16, seed=51)
    m = _mask(20, "weights", 52)
    up = torch.full((), 256.0, device="cuda")
    got = _all(lambda h, w: tb.linear_cross_entropy(h, w, inp["t"], m), inp["h"], inp["w"], up, inp["uh"], inp["uw"])
    h, w, uh, uw = (inp[k].double() for k in ("h", "w", "uh", "uw"))
    gen = torch.Generator(device="cuda").manual_seed(53)
    dirs = {k: torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64) for k, x in (("h", h), ("w", w))}

    def first(h, w):
        return 256.0 * _definition(h, w, inp["t"], m, "mean")

    def second(h, w):
        h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        gh, gw = torch.autograd.grad(first(h, w), (h, w))
        return (gh * uh).sum() + (gw * uw).sum()

    eps = 1e-5
    for f, names in ((first, ("dh", "dw")), (second, ("gh", "gw"))):
        for k, name in zip(("h", "w"), names):
            plus, minus = {"h": h, "w": w}, {"h": h, "w": w}
            plus[k], minus[k] = plus[k] + eps * dirs[k], minus[k] - eps * dirs[k]
            num = float((f(**plus) - f(**minus)) / (2 * eps))
            terms = got[name].double() * dirs[k]
            # every entry of the gradient is within 8u of the largest; the errors add up like a random walk
            bound = 8 * U[torch.float16] * float(got[name].abs().max()) * float(dirs[k].norm())
            assert abs(num - float(terms.sum())) <= bound, name


def test_gradient_by_the_upstream_is_the_loss_direction():
    """d<dh, uh>/d dloss_i = <d l_i / dh_i, uh_i>, so with uh = dh of dloss = 1 it is |dh_i|^2."""
    inp = _inputs(40, 64, 100, torch.bfloat16, seed=54)
    got = _check(inp, None, "none", uw=False)
    assert got["gd"].shape == (40,)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("n,d,v", [(40, 64, 100), (300, 136, 1500)])
def test_gradient_by_the_upstream_along_the_gradient(n, d, v, dtype):
    """With uh = dh of dloss = 1 the gradient by dloss_i is |dh_i|^2. dh is within 4u of its largest entry of
    what the second gradient forms in fp32, and that is within 1e-5 of the terms' scale (twice the largest A)."""
    inp = _inputs(n, d, v, dtype, seed=n)
    h, dloss = inp["h"].requires_grad_(True), torch.ones(n, device="cuda", requires_grad=True)
    loss = tb.linear_cross_entropy(h, inp["w"], inp["t"], reduction="none")
    dh, = torch.autograd.grad(loss, h, dloss, create_graph=True)
    uh = dh.detach()
    gd, = torch.autograd.grad(dh, dloss, uh)
    x = uh.double()
    scale = 2 * float((x @ inp["w"].double().t()).abs().max())
    bound = 4 * U[dtype] * float(x.abs().max()) * x.abs().sum(1) + 1e-5 * scale
    assert bool(((gd.double() - x.square().sum(1)).abs() <= bound).all())
    assert float(bound.max()) < 0.2 * float(x.square().sum(1).median())


def test_only_one_gradient_wanted():
    inp = _inputs(70, 64, 300, torch.bfloat16, seed=55)
    h, w = inp["h"].clone().requires_grad_(True), inp["w"].clone().requires_grad_(True)
    both = torch.autograd.grad(tb.linear_cross_entropy(h, w, inp["t"]), (h, w))
    dh, = torch.autograd.grad(tb.linear_cross_entropy(h, inp["w"], inp["t"]), h)
    dw, = torch.autograd.grad(tb.linear_cross_entropy(inp["h"], w, inp["t"]), w)
    assert torch.equal(dh, both[0]) and torch.equal(dw, both[1])


def test_no_rows():
    w = torch.randn(50, 32, device="cuda", dtype=torch.float16, requires_grad=True)
    h = torch.empty(2, 0, 32, device="cuda", dtype=torch.float16, requires_grad=True)
    t = torch.empty(2, 0, dtype=torch.long, device="cuda")
    for reduction in ("mean", "sum"):
        loss = tb.linear_cross_entropy(h, w, t, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, (h, w), create_graph=True)
        assert float(loss) == 0.0 and dh.shape == h.shape and not dw.any()
        gw, = torch.autograd.grad(dw, w, torch.ones_like(dw))
        assert not gw.any()
    assert tb.linear_cross_entropy(h, w, t, reduction="none").shape == (2, 0)


def test_runs_agree_and_streams():
    inp = _inputs(1500, 256, 5000, torch.bfloat16, seed=61)
    m = _mask(1500, "weights", 62)
    dl = torch.ones((), device="cuda")
    run = lambda: _all(lambda h, w: tb.linear_cross_entropy(h, w, inp["t"], m), inp["h"], inp["w"], dl,  # noqa: E731
                       inp["uh"], inp["uw"])
    one = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(one[k], two[k]) for k in one)


def test_third_derivative_raises():
    inp = _inputs(20, 32, 40, torch.bfloat16, seed=63)
    h, w = inp["h"].requires_grad_(True), inp["w"].requires_grad_(True)
    dh, = torch.autograd.grad(tb.linear_cross_entropy(h, w, inp["t"]), h, create_graph=True)
    gh, = torch.autograd.grad(dh.float().square().sum(), h, create_graph=True)
    with pytest.raises(RuntimeError, match="third derivative"):
        torch.autograd.grad(gh.float().sum(), h)


def test_target_outside_the_vocabulary_raises_at_the_next_call():
    inp = _inputs(20, 32, 40, torch.bfloat16, seed=64)
    for bad in (40, -1, 10**12):
        t = inp["t"].clone()
        t[13] = bad
        tb.linear_cross_entropy(inp["h"], inp["w"], t)
        torch.cuda.synchronize()
        with pytest.raises(_lib.KernelError, match="target outside the vocabulary.*row 13"):
            tb.linear_cross_entropy(inp["h"], inp["w"], inp["t"])
        tb.linear_cross_entropy(inp["h"], inp["w"], t)
        with pytest.raises(_lib.KernelError, match="target outside the vocabulary"):
            _lib.check_device_errors()
    _check(inp)


def test_refusals():
    inp = _inputs(8, 32, 40, torch.bfloat16, seed=65)
    h, w, t = inp["h"], inp["w"], inp["t"]
    with pytest.raises(ValueError, match="reduction"):
        tb.linear_cross_entropy(h, w, t, reduction="avg")
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        tb.linear_cross_entropy(h.float(), w.float(), t)
    with pytest.raises(RuntimeError, match="share one dtype"):
        tb.linear_cross_entropy(h, w.half(), t)
    with pytest.raises(RuntimeError, match="expected hidden"):
        tb.linear_cross_entropy(h, w[:, :16], t)
    with pytest.raises(RuntimeError, match="leading shape"):
        tb.linear_cross_entropy(h, w, t[:4])
    with pytest.raises(RuntimeError, match="integers"):
        tb.linear_cross_entropy(h, w, t.float())
    with pytest.raises(RuntimeError, match="mask must have"):
        tb.linear_cross_entropy(h, w, t, torch.ones(4, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA tensors|device"):
        tb.linear_cross_entropy(h, w.cpu(), t)


@pytest.mark.parametrize("dtype", (torch.uint8, torch.int8, torch.bool, torch.float8_e4m3fn, torch.float64, torch.int64))
def test_weights_of_other_types_are_refused_with_gradients(dtype):
    """Before the copy into aligned rows, which an odd width asks for and which moves 16-bit elements."""
    inp = _inputs(8, 33, 40, torch.bfloat16, seed=66)
    h = inp["h"].requires_grad_(True)
    w = torch.ones(40, 33, device="cuda").to(dtype)
    with pytest.raises(RuntimeError, match="share one dtype"):
        tb.linear_cross_entropy(h, w, inp["t"])
    with pytest.raises(RuntimeError, match="expected hidden"):
        tb.linear_cross_entropy(h, torch.ones(40, 31, device="cuda", dtype=torch.bfloat16), inp["t"])


@pytest.mark.parametrize("n,d,v", [(2, 2**32, 3), (2, 2**32 + 8, 3), (2, 65537, 3), (2**24 + 1, 1, 3), (2, 1, 2**24 + 1)])
@pytest.mark.parametrize("grad", (False, True))
def test_sizes_past_the_limits_are_refused(n, d, v, grad):
    """Broadcast tensors: no memory behind the sizes, 2^32 columns among them."""
    h = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda").expand(n, d).requires_grad_(grad)
    w = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda").expand(v, d)
    t = torch.zeros(1, dtype=torch.long, device="cuda").expand(n)
    with pytest.raises(RuntimeError, match="at most 2\\^24 rows"):
        tb.linear_cross_entropy(h, w, t)


@pytest.mark.parametrize("grad", (False, True))
@pytest.mark.parametrize("n,v", [(1, 700), (4, 700), (4, 5000), (64, 250), (300, 2000)])
def test_nearly_certain_tokens(n, v, grad):
    """Logits near 520 that are exact in fp32, with one entry 16 or 24 above the others: the losses of tokens
    that have it as their target are 1e-4 to 1e-8, far below an ulp of the logits, and never negative.

    With the maximum taken out first, what is left are the errors of l, the sum of exponentials (2^-22
    each and for each of two rescalings, their sum at most as much again), and of its logarithm: below
    2^-19 in all, of 1 or of the loss."""
    g = torch.Generator().manual_seed(n + v)
    for gap in (0.25, 0.375):
        h = torch.randint(1, 3, (n, 32), generator=g).float()
        w = torch.randint(-2, 3, (v, 32), generator=g).float() / 8
        h[:, -1], w[:, -1], w[5, -1] = 64.0, 8.0, 8.0 + gap
        h, w = (x.to(torch.bfloat16).cuda() for x in (h, w))
        t = torch.randint(0, v, (n,), generator=g)
        t[::2] = 5
        t = t.cuda()
        ref = _definition(h.double(), w.double(), t, None, "none")
        assert 0.0 < float(ref[0]) < 1e-2
        loss = tb.linear_cross_entropy(h.requires_grad_(grad), w, t, reduction="none").detach()
        assert float(loss.min()) >= 0.0
        assert float(((loss.double() - ref).abs() / ref.clamp_min(1.0)).max()) <= 2.0**-19


@pytest.mark.parametrize("up", (float("inf"), float("nan")))
@pytest.mark.parametrize("reduction", ("mean", "sum", "none"))
def test_rows_left_out_stay_zero_when_the_upstream_is_not_finite(reduction, up):
    """An overflowed loss scale: the rows that take part lose their gradients, those left out keep exact
    zeros; with none that takes part the weight gradients are zeros too."""
    n = 150
    inp = _inputs(n, 72, 300, torch.float16, seed=67)
    m = _mask(n, "weights", 68)
    inp["t"][1::9] = -100
    out = (m == 0) | (inp["t"] == -100)
    fn = lambda m: lambda h, w: tb.linear_cross_entropy(h, w, inp["t"], m, reduction=reduction)  # noqa: E731
    dl = torch.full((n,) if reduction == "none" else (), up, device="cuda")
    got = _all(fn(m), inp["h"], inp["w"], dl, inp["uh"], inp["uw"])
    for k in ("dh", "gh"):
        assert not got[k][out].any(), k
        assert not got[k][~out].isfinite().all(), k
    none = _all(fn(torch.zeros(n, device="cuda")), inp["h"], inp["w"], dl, inp["uh"], inp["uw"])
    for k in ("dh", "gh", "dw", "gw", "gd"):
        assert not none[k].any(), k


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("n,v", [(1, 700), (5, 3000), (300, 2000)])
def test_gradients_of_nearly_certain_tokens(n, v, dtype):
    """The logits of the test above, every target the likely entry: G there is p - 1, 1e-2 to 1e-4, and column 0
    of the hidden gradient is that entry alone (w is 0 in it except for a 1 in the target's row). It is rounded
    twice (2u); p is within 2^-19 as l is there."""
    g = torch.Generator().manual_seed(n + v)
    h = torch.randint(1, 3, (n, 32), generator=g).float()
    w = torch.randint(-2, 3, (v, 32), generator=g).float() / 8
    h[:, -1], w[:, -1], w[5, -1] = 64.0, 8.0, 8.25
    h[:, 0], w[:, 0], w[5, 0] = 0.0, 0.0, 1.0
    h, w = (x.to(dtype).cuda().requires_grad_(True) for x in (h, w))
    t = torch.full((n,), 5, device="cuda")
    p = torch.softmax(h.detach().double() @ w.detach().double().t(), 1)[:, 5]
    assert 1e-5 < float((1 - p).min()) and float((1 - p).max()) < 0.05
    up = 1024.0
    dh, = torch.autograd.grad(tb.linear_cross_entropy(h, w, t, reduction="sum"), h, torch.full((), up, device="cuda"))
    err = (dh[:, 0].double() - up * (p - 1)).abs()
    assert bool((err <= up * (2 * U[dtype] * (1 - p) + 2.0**-19)).all())
    # one entry of the vocabulary: p is 1, and what 2^-19 of it leaves is all there is
    dh, = torch.autograd.grad(tb.linear_cross_entropy(h, w[:1], t * 0, reduction="sum"), h)
    assert float(dh.abs().max()) <= 2.0**-19 * float(w[:1].detach().abs().max())
