"""The TTT-E2E model with kernel_norm_loss on CUDA (attention, norms and token loss
on the kernels, bf16) against the plain model in float64 on CPU: meta step with its
meta-gradient, test-time adaptation, and the scores of the adapted model. The
tolerances are those of the plain bf16 model's test (tests/test_gpu_ttt_model.py):
they are set by bf16 weights and activations, which both share."""

import pytest
import torch

from testtimeideas_b200 import _lib, ttt_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,suffix,chunk,pfilter", [(None, -1, None, None), (96, 1, 128, "mlp_fast"),
                                                         (None, 1, None, "suffix_blocks,ln_f,head")])
def test_meta_step_and_scores_match_the_plain_model(window, suffix, chunk, pfilter):
    kw = dict(vocab_size=256, max_seq_len=512, d_model=128, n_heads=2, n_layers=2, d_ff=256, window_size=window,
              suffix_layers=suffix)
    torch.manual_seed(3)
    cpu = ttt_model.TTTModel(ttt_model.ModelConfig(**kw)).double()
    gpu = ttt_model.TTTModel(ttt_model.ModelConfig(kernel_norm_loss=True, **kw)).to("cuda", torch.bfloat16)
    gpu.load_state_dict({n: p.to(torch.bfloat16) for n, p in cpu.state_dict().items()})
    t = 256
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 256, (1, t), generator=g)
    tgt = torch.randint(0, 256, (1, t), generator=g)
    inner_mask = torch.zeros(1, t)
    inner_mask[:, : 3 * t // 4] = 1.0
    outer_mask = 1.0 - inner_mask

    def run(model, dev):
        a = [x.to(dev) for x in (ids, tgt, inner_mask, outer_mask)]
        inner, outer = ttt_model.meta_step(model, *a, inner_lr=0.05, inner_steps=1, param_filter=pfilter,
                                           chunk_size=chunk)
        outer.backward()
        params = ttt_model.ttt_apply(model, *a[:3], inner_lr=0.05, inner_steps=1, param_filter=pfilter,
                                     chunk_size=chunk)
        scores = ttt_model.token_losses(model, params, a[0], a[1], a[3], chunk_size=chunk)
        return inner.item(), outer.item(), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}, scores

    ri, ro, rg, rs = run(cpu, "cpu")
    _lib.profile_collect()
    _lib.profile_enable(True)
    gi, go, gg, gs = run(gpu, "cuda")
    torch.cuda.synchronize()
    _lib.profile_enable(False)
    prof = _lib.profile_collect()
    _lib.check_device_errors()
    assert prof["norm"][0] > 0 and prof["loss"][0] > 0 and prof["loss"][1] > 0.0
    assert abs(gi - ri) < 2e-2 * abs(ri) and abs(go - ro) < 2e-2 * abs(ro)
    assert set(gg) == set(rg)
    num = sum(float((gg[n].double().cpu() - rg[n]).pow(2).sum()) for n in rg)
    den = sum(float(rg[n].pow(2).sum()) for n in rg)
    assert (num / den) ** 0.5 < 5e-2
    assert float((gs.double().cpu() - rs).norm() / rs.norm()) < 3e-2
    assert not gs.cpu()[outer_mask == 0].any()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_fp32_weights_under_autocast(dtype):
    """fp32 parameters, 16-bit products: losses and meta-gradient of the model with kernel_norm_loss against
    float64. Tolerances as above (bf16); fp16 rounds finer."""
    kw = dict(vocab_size=256, max_seq_len=512, d_model=128, n_heads=2, n_layers=2, d_ff=256)
    torch.manual_seed(5)
    cpu = ttt_model.TTTModel(ttt_model.ModelConfig(**kw)).double()
    gpu = ttt_model.TTTModel(ttt_model.ModelConfig(kernel_norm_loss=True, **kw)).cuda()
    gpu.load_state_dict({n: p.float() for n, p in cpu.state_dict().items()})
    g = torch.Generator().manual_seed(6)
    ids, tgt = (torch.randint(0, 256, (1, 256), generator=g) for _ in range(2))
    inner = (torch.arange(256) < 192).float()[None]
    ref = ttt_model.meta_step(cpu, ids, tgt, inner, 1 - inner, inner_lr=0.05, inner_steps=1)
    ref[1].backward()
    with torch.autocast("cuda", dtype=dtype):
        a = [x.cuda() for x in (ids, tgt, inner, 1 - inner)]
        got = ttt_model.meta_step(gpu, *a, inner_lr=0.05, inner_steps=1)
        scores = ttt_model.token_losses(gpu, dict(gpu.named_parameters()), *a[:2])
    (got[1] * 64).backward()
    _lib.check_device_errors()
    for x, r in zip(got, ref):
        assert abs(x.item() - r.item()) < 2e-2 * abs(r.item())
    assert scores.shape == tgt.shape and abs(float(scores.mean()) - float(ref[0])) < 0.5 * float(ref[0])
    num = den = 0.0
    cpu_grads = dict(cpu.named_parameters())
    for n, p in gpu.named_parameters():
        if cpu_grads[n].grad is None:
            continue
        assert p.grad.dtype == torch.float32
        num += float((p.grad.double().cpu() / 64 - cpu_grads[n].grad).pow(2).sum())
        den += float(cpu_grads[n].grad.pow(2).sum())
    assert (num / den) ** 0.5 < 5e-2


def test_norm_under_autocast_is_as_torchs():
    """Autocast runs nn.LayerNorm in fp32 whatever the types of x and the parameters."""
    from testtimeideas_b200 import LayerNorm

    for x_dtype, p_dtype in ((torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                             (torch.float32, torch.bfloat16), (torch.float32, torch.float32)):
        ref, own = torch.nn.LayerNorm(96).to("cuda", p_dtype), LayerNorm(96).to("cuda", p_dtype)
        x = torch.randn(7, 96, device="cuda").to(x_dtype)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            a, b = ref(x), own(x)
        assert a.dtype == b.dtype == torch.float32
        assert float((a - b).abs().max()) <= 1.6e-5 * float(a.abs().max())  # fp32, as in test_gpu_layer_norm.py
