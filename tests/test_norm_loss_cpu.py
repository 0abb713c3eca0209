"""The norm and loss operators on CPU (the PyTorch formulation of the same values),
the model with kernel_norm_loss against the one without (float64, one meta step,
test-time adaptation, scores), the C ABI's declarations, its refusals before any
launch, and its buffer sizes."""

import ctypes
import re
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import testtimeideas_b200 as tb
from testtimeideas_b200 import _lib, ttt_model

HEADER = Path(__file__).resolve().parents[1] / "include" / "ttt_ops.h"


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from testtimeideas_b200 import build
        build.build()
    return _lib.load_library()


# ---------------------------------------------------------------- values on CPU
def test_linear_cross_entropy_is_the_models_loss():
    g = torch.Generator().manual_seed(1)
    h = torch.randn(3, 7, 16, generator=g, dtype=torch.float64)
    w = torch.randn(29, 16, generator=g, dtype=torch.float64)
    t = torch.randint(0, 29, (3, 7), generator=g)
    t[0, 3] = -100
    m = (torch.rand(3, 7, generator=g) < 0.6).double() * 1.5
    for mask in (None, m):
        ref = ttt_model.compute_loss(h @ w.t(), t, mask)
        # the mask of compute_loss passes through float32, its sum with it
        assert abs(float(tb.linear_cross_entropy(h, w, t, mask) - ref)) < 1e-6
    ce = F.cross_entropy((h @ w.t()).flatten(0, 1), t.flatten(), reduction="none").view(3, 7)
    assert torch.allclose(tb.linear_cross_entropy(h, w, t, m, reduction="none"), ce * m)
    assert torch.allclose(tb.linear_cross_entropy(h, w, t, reduction="sum"), ce.sum())
    assert float(tb.linear_cross_entropy(h, w, t, torch.zeros(3, 7))) == 0.0
    assert float(tb.linear_cross_entropy(h[:0], w, t[:0])) == 0.0


def test_linear_cross_entropy_left_out_rows_and_second_gradients():
    g = torch.Generator().manual_seed(2)
    h = torch.randn(6, 5, generator=g, dtype=torch.float64)
    w = torch.randn(11, 5, generator=g, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([1, 2, -100, 4, 10, 99])
    m = torch.tensor([1.0, 0.0, 1.0, 0.5, 2.0, 0.0])
    dirty = h.clone()
    dirty[[1, 2, 5]] = float("nan")
    dirty.requires_grad_(True)
    h.requires_grad_(True)
    a = torch.autograd.grad(tb.linear_cross_entropy(h, w, t, m), (h, w))
    b = torch.autograd.grad(tb.linear_cross_entropy(dirty, w, t, m), (dirty, w))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[0][[1, 2, 5]].any()
    assert torch.autograd.gradgradcheck(lambda h, w: tb.linear_cross_entropy(h, w, t, m), (h, w))
    with pytest.raises(ValueError, match="outside the vocabulary"):
        tb.linear_cross_entropy(h, w, t)
    with pytest.raises(ValueError, match="reduction"):
        tb.linear_cross_entropy(h, w, t, m, reduction="max")


def test_linear_cross_entropy_sums_16_bit_losses_in_32():
    """Equal logits: every loss is log(8) rounded to bf16, and so is their mean under any mask. 70000
    positions: neither the sum of their losses nor their count is a number of fp16."""
    w, t = torch.zeros(8, 4, dtype=torch.bfloat16), torch.zeros(1300, dtype=torch.long)
    h = torch.ones(1300, 4, dtype=torch.bfloat16)
    one = tb.linear_cross_entropy(h[:1], w, t[:1])
    assert one.dtype == torch.bfloat16 and abs(float(one) - 2.0794) < 0.005
    for kept in (1001, 1005, 1011, 1300):
        for weight in (1.0, 1 / 3):
            m = torch.zeros(1300)
            m[:kept] = weight
            assert torch.equal(tb.linear_cross_entropy(h, w, t, m), one)
    n = 70000
    h, w, t = torch.ones(n, 2).half(), torch.zeros(8, 2).half().requires_grad_(True), torch.zeros(n, dtype=torch.long)
    for m in (None, torch.ones(n)):
        loss = tb.linear_cross_entropy(h, w, t, m)
        assert loss.dtype == torch.float16 and abs(float(loss.detach()) - 2.0794) < 0.005
        dw, = torch.autograd.grad(loss, w)
        assert (dw[0].float() + 0.875).abs().max() < 0.01 and (dw[1:].float() - 0.125).abs().max() < 0.01


def test_layer_norm_module_keeps_the_state_dict():
    ref, m = torch.nn.LayerNorm(24).double(), tb.LayerNorm(24).double()
    with torch.no_grad():
        ref.weight.normal_()
        ref.bias.normal_()
    m.load_state_dict(ref.state_dict())
    x = torch.randn(4, 24, dtype=torch.float64)
    assert torch.equal(m(x), ref(x))
    with pytest.raises(ValueError, match="one dimension"):
        tb.LayerNorm((2, 3))(torch.zeros(2, 3))


# ---------------------------------------------------------------- the model
def _pair(**over):
    kw = dict(vocab_size=48, max_seq_len=32, d_model=32, n_heads=2, n_layers=2, d_ff=64, **over)
    torch.manual_seed(3)
    plain = ttt_model.TTTModel(ttt_model.ModelConfig(**kw)).double()
    fused = ttt_model.TTTModel(ttt_model.ModelConfig(kernel_norm_loss=True, **kw)).double()
    fused.load_state_dict(plain.state_dict())
    return plain, fused


@pytest.mark.parametrize("over,chunk,pfilter", [(dict(window_size=None), None, None),
                                                (dict(window_size=8, suffix_layers=1), 8, "mlp_fast")])
def test_model_with_kernel_norm_loss_is_the_same_model(over, chunk, pfilter):
    plain, fused = _pair(**over)
    g = torch.Generator().manual_seed(4)
    ids, tgt = (torch.randint(0, 48, (2, 16), generator=g) for _ in range(2))
    inner = (torch.rand(2, 16, generator=g) < 0.5).float()
    outer = 1.0 - inner
    res = []
    for m in (plain, fused):
        li, lo = ttt_model.meta_step(m, ids, tgt, inner, outer, inner_lr=0.1, inner_steps=1, param_filter=pfilter,
                                     chunk_size=chunk)
        lo.backward()
        # a second step needs every updated parameter in the suffix (the embeddings are not)
        steps = 1 if pfilter is None else 2
        adapted = ttt_model.ttt_apply(m, ids, tgt, inner, inner_lr=0.1, inner_steps=steps, param_filter=pfilter,
                                      chunk_size=chunk)
        scores = ttt_model.token_losses(m, adapted, ids, tgt, outer, chunk_size=chunk)
        res.append((li.detach(), lo.detach(), {n: p.grad for n, p in m.named_parameters() if p.grad is not None},
                    {n: p.detach() for n, p in adapted.items()}, scores))
    a, b = res
    assert abs(a[0] - b[0]) < 1e-6 and abs(a[1] - b[1]) < 1e-6  # float32 masks in compute_loss
    assert set(a[2]) == set(b[2])
    for i in (2, 3):
        for n in a[i]:
            assert torch.allclose(a[i][n], b[i][n], rtol=1e-5, atol=1e-8), n
    assert torch.allclose(a[4], b[4], rtol=1e-5, atol=1e-8) and a[4].shape == tgt.shape
    assert not b[4][outer == 0].any()


# ---------------------------------------------------------------- the C ABI
class NormProblem(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("dim", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("p_dtype", ctypes.c_int32), ("eps", ctypes.c_float)]


class NormFwd(ctypes.Structure):
    _fields_ = [("pb", NormProblem), ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("w", ctypes.c_void_p),
                ("b", ctypes.c_void_p), ("y", ctypes.c_void_p), ("mean", ctypes.c_void_p), ("rstd", ctypes.c_void_p)]


class LceProblem(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64), ("vocab", ctypes.c_int64), ("dim", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("reduction", ctypes.c_int32), ("mask_kind", ctypes.c_int32), ("ignore_index", ctypes.c_int64)]


class LceFwd(ctypes.Structure):
    _fields_ = [("pb", LceProblem), ("h", ctypes.c_void_p), ("h_stride", ctypes.c_int64), ("w", ctypes.c_void_p),
                ("w_stride", ctypes.c_int64), ("targets", ctypes.c_void_p), ("mask", ctypes.c_void_p),
                ("loss", ctypes.c_void_p), ("state", ctypes.c_void_p), ("need_state", ctypes.c_int32),
                ("err", ctypes.c_void_p), ("work", ctypes.c_void_p), ("work_bytes", ctypes.c_int64)]


def test_header_and_library_agree(lib):
    names = sorted(set(re.findall(r"^\s*(?:int64_t|int)\s+(ttt_\w+)\s*\(", HEADER.read_text(), flags=re.M)))
    assert names == sorted(_lib.EXPORTED_OPS)
    for n in names:
        assert hasattr(lib, n), n


@pytest.mark.parametrize("field,value,status", [("dtype", 9, 2), ("p_dtype", 1, 2), ("rows", -1, 4), ("dim", 0, 4),
                                                ("dim", 16385, 4), ("rows", 2**31, 4)])
def test_norm_refusals(lib, field, value, status):
    pb = NormProblem(4, 64, 0, 0, 1e-5)
    dummy = 4096  # never dereferenced: refused before a launch
    a = NormFwd(pb, dummy, 64, None, None, dummy, None, None)
    setattr(a.pb, field, value)
    assert lib.ttt_norm_fwd(ctypes.byref(a), None) == status
    assert lib.ttt_norm_fwd(None, None) == 1
    a = NormFwd(pb, None, 64, None, None, dummy, None, None)
    assert lib.ttt_norm_fwd(ctypes.byref(a), None) == 1
    a = NormFwd(pb, dummy, 64, None, None, dummy, dummy, None)
    assert lib.ttt_norm_fwd(ctypes.byref(a), None) == 1
    a = NormFwd(pb, dummy, -64, None, None, dummy, None, None)
    assert lib.ttt_norm_fwd(ctypes.byref(a), None) == 5


def _lce(**over):
    dummy = 4096
    a = LceFwd(LceProblem(4, 100, 64, 1, 1, 0, -100), dummy, 64, dummy, 64, dummy, None, dummy, dummy, 1, None, dummy,
               1 << 40)
    for k, v in over.items():
        setattr(a.pb if k in ("n", "vocab", "dim", "dtype", "reduction", "mask_kind") else a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(dtype=2), 2), (dict(n=-1), 4), (dict(vocab=0), 4), (dict(vocab=2**24 + 1), 4), (dict(dim=0), 4),
    (dict(dim=65537), 4), (dict(reduction=3), 10), (dict(mask_kind=3), 10), (dict(w=None), 1), (dict(w=4096 + 2), 6),
    (dict(w_stride=63), 5), (dict(w_stride=68), 5), (dict(loss=None), 1), (dict(state=None), 1), (dict(targets=None), 1),
    (dict(mask_kind=1), 1), (dict(mask=4096), 1), (dict(work=None), 11), (dict(work_bytes=64), 11),
    (dict(work=4096 + 16), 6), (dict(need_state=2), 10)])
def test_loss_refusals(lib, over, status):
    a = _lce(**over)
    assert lib.ttt_lce_fwd(ctypes.byref(a), None) == status
    assert lib.ttt_lce_fwd(None, None) == 1


def test_buffer_sizes(lib):
    lib.ttt_lce_state_bytes.restype = lib.ttt_lce_work_bytes.restype = ctypes.c_int64
    for n in (0, 1, 255, 256, 257, 8192):
        for d in (1, 8, 100, 768):
            pb = LceProblem(n, 32000, d, 1, 1, 0, -100)
            assert lib.ttt_lce_state_bytes(ctypes.byref(pb)) == _lib._lce_state_bytes(n, d)
    # the stored derivatives of a piece stay within 512 MB as the vocabulary and the rows grow
    for n, v in ((8192, 32000), (16384, 131072), (65536, 4096)):
        pb = LceProblem(n, v, 64, 1, 1, 0, -100)
        for p, extra in ((1, n * 64 * 4 * 74), (2, n * 64 * 4 * 74 + v // 64 * n * 8)):
            assert lib.ttt_lce_work_bytes(ctypes.byref(pb), p) <= (513 << 20) + extra + 256 * n
    assert lib.ttt_lce_work_bytes(ctypes.byref(LceProblem(1, 0, 64, 1, 1, 0, 0)), 1) == 0
    assert lib.ttt_lce_state_bytes(None) == 0


# ---------------------------------------------------------------- forward mode
@pytest.fixture()
def stand_ins(lib):
    """The raw operators on CPU tensors, so that what surrounds them can be run here."""
    _lib.load_torch_ops()
    with torch.library._scoped_library("ttt", "IMPL") as impl:
        impl.impl("layer_norm", lambda x, w, b, eps, need: (
            F.layer_norm(x, x.shape[-1:], w, b, eps), x.new_zeros(2, x.numel() // x.shape[-1] if need else 0)), "CPU")
        impl.impl("layer_norm_bwd", lambda dy, x, w, stats, need_dx, need_dw, need_db, p_type: (
            dy.clone(), x.new_zeros(x.shape[-1]), x.new_zeros(x.shape[-1])), "CPU")
        impl.impl("linear_ce", lambda h, w, t, m, reduction, ignore, need: (
            F.cross_entropy(h @ w.t(), t), h.new_zeros(0, dtype=torch.uint8)), "CPU")
        impl.impl("linear_ce_bwd", lambda dloss, h, w, state, reduction, need_dh, need_dw: (
            dloss * h, dloss * w), "CPU")
        yield torch.ops.ttt


def test_forward_mode_is_refused(stand_ins):
    """Neither operator has a forward-mode derivative: a tensor with a tangent raises, whichever input it is,
    and so does a tangent on the upstream gradient. Without one (or with the mode off) nothing changes."""
    import torch.autograd.forward_ad as fwd

    x, w, b = torch.randn(5, 8), torch.randn(8), torch.randn(8)
    head, t, m = torch.randn(9, 8), torch.randint(0, 9, (5,)), torch.ones(5)
    norm = lambda x, w, b: stand_ins.layer_norm_ad(x, w, b, 1e-5)  # noqa: E731
    loss = lambda h, w, m: stand_ins.linear_ce_ad(h, w, t, m, 1, -100)  # noqa: E731
    for fn, args in ((norm, (x, w, b)), (loss, (x, head, m))):
        plain = fn(*args)
        for i in range(3):
            tangents = [torch.zeros_like(a) for a in args]
            tangents[i] = torch.ones_like(args[i])

            def one(a, i=i):
                return fn(*args[:i], a, *args[i + 1:])

            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.func.jvp(one, (args[i],), (tangents[i],))
            with fwd.dual_level():
                dual = fwd.make_dual(args[i], tangents[i])
                with pytest.raises(RuntimeError, match="forward-mode"):
                    one(dual)
                with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                    one(dual)
                with fwd._set_fwd_grad_enabled(False):
                    assert torch.equal(one(dual), plain)
        # reverse mode is as before, and a tangent of the upstream gradient is refused
        leaf = args[0].clone().requires_grad_(True)
        y = fn(leaf, *args[1:])
        torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
        with fwd.dual_level():
            up = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
            for create in (False, True):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad(y, leaf, up, retain_graph=True, create_graph=create)


def test_a_mask_that_wants_a_gradient_is_refused(stand_ins):
    """The kernels form no gradient by the mask's weights; none was returned without a word."""
    h, w, t = torch.randn(5, 8), torch.randn(9, 8), torch.randint(0, 9, (5,))
    mask = torch.rand(5).requires_grad_(True)
    for hidden in (h, h.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="gradient by the mask"):
            stand_ins.linear_ce_ad(hidden, w, t, mask, 1, -100)
        with pytest.raises(RuntimeError, match="gradient by the mask"):
            stand_ins.linear_ce_ad(hidden, w, t, mask * 2, 0, -100)
        stand_ins.linear_ce_ad(hidden, w, t, mask.detach(), 1, -100)
        with torch.no_grad():
            stand_ins.linear_ce_ad(hidden, w, t, mask, 1, -100)


def test_state_sizes_tell_row_counts_apart(lib):
    """The gradients know a state by its size, and index with the rows it lists."""
    lib.ttt_lce_state_bytes.restype = ctypes.c_int64
    for d in (8, 72, 768):
        sizes = [lib.ttt_lce_state_bytes(ctypes.byref(LceProblem(n, 100, d, 1, 1, 0, -100))) for n in range(600)]
        assert len(set(sizes)) == 600 and sizes == [_lib._lce_state_bytes(n, d) for n in range(600)]
