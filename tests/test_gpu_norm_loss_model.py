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
