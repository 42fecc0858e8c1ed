"""The engine's log-probs and gradients without stored logits (Qwen25VL.store_logits = False) on the tiny configuration, against the fp32 oracle.
Untied head: the bounds that the stored-logits path is held to (HF's own bf16 evaluation of this very model and batch,
tests/golden/bf16_yardstick.json).  Tied head: that yardstick was measured on another model, so the criterion is the side-by-side one, no more than
1.5 times the error of the other bf16 evaluation at hand, the stored-logits path on the same inputs."""
import json
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import tiny  # noqa: E402
from oracle import qwen25vl as Q  # noqa: E402
from oracle import rl_math as M  # noqa: E402


def build(tied):
    from spatialthinker_amd import model as mdl
    conf = dict(tiny.TINY, tie_word_embeddings=tied)
    cfg = mdl.VLConfig(**conf)
    params = tiny.make_params()
    if tied:
        params.pop("lm_head.weight", None)
    store = mdl.ParamStore(cfg, trainable=True)
    store.load_hf_state_dict({k: torch.from_numpy(v) for k, v in params.items()})
    return conf, params, store, mdl.Qwen25VL(cfg, store)


def run(eng, store, b, loss, **kw):
    store.grad.zero_()
    lp, metrics = eng.forward_backward(b, loss, 1.0, clip_low=0.2, clip_high=0.3, clip_dual=3.0, kl_kind="low_var_kl", kl_coef=1e-2, grad_accum=1.0, **kw)
    return lp.clone(), metrics.clone(), {k: v.float().cpu() for k, v in store.export_hf(store.g).items()}


@pytest.mark.parametrize("tied", [False, True])
def test_engine_without_stored_logits(tied, golden_dir):
    conf, params, store, eng = build(tied)
    z = np.load(os.path.join(golden_dir, "model_tiny.npz"))
    batch = tiny.make_batch()
    R = batch["R"]
    b = eng.stage(batch["input_ids"], batch["attention_mask"], z["position_ids"], R, batch["pixel_values"], batch["image_grid_thw"])
    assert eng.store_logits                                        # the default keeps them
    stored = eng.log_probs(b, 1.0).cpu().numpy()
    eng.store_logits = False
    got = eng.log_probs(b, 1.0).cpu().numpy()
    m = batch["attention_mask"][:, -R:].astype(bool)
    yard = json.load(open(os.path.join(golden_dir, "bf16_yardstick.json")))
    if not tied:
        want = z["logp"]
        assert np.abs(got[m] - want[m]).max() <= yard["logp"]["hf_bf16"]["max"]
    # the stored path rounds every logit to bf16: half a step of the largest logit in the label's logit and in the lse, 2 ub max|z|
    assert np.abs(got[m] - stored[m]).max() <= 2 * 2.0 ** -8 * 16.0
    assert (got[~m] == 0).all()

    rs = np.random.RandomState(0)
    old = (got + 0.2 * rs.standard_normal(got.shape)).astype(np.float32)
    adv = rs.standard_normal((m.shape[0], 1)).astype(np.float32).repeat(R, 1) * m
    dv = lambda a, dt=torch.float32: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dt)
    loss = dict(old_log_probs=dv(old), ref_log_probs=dv(old), advantages=dv(adv), response_mask=dv(m, torch.int64))
    lp0, met0, g0 = run(eng, store, b, dict(loss))
    lp1, met1, g1 = run(eng, store, b, dict(loss))
    assert torch.equal(lp0, lp1) and torch.equal(met0, met1)
    head = "model.language_model.embed_tokens.weight" if tied else "lm_head.weight"
    if not tied:
        assert torch.equal(g0[head], g1[head])                    # (a tied head also takes the embedding's gradient)
    # gradients against the oracle's autograd, in the bounds that the stored path is held to
    p32 = {k: torch.from_numpy(v).clone().requires_grad_(k.endswith(("q_proj.weight", "down_proj.weight", "lm_head.weight", "embed_tokens.weight"))) for k, v in params.items()}
    lp_o = Q.response_log_probs(p32, Q.VLConfig(**conf), torch.from_numpy(batch["input_ids"]), torch.from_numpy(batch["attention_mask"]),
                                torch.from_numpy(z["position_ids"]), R, 1.0, torch.from_numpy(batch["pixel_values"]), batch["image_grid_thw"])
    _, gl = M.actor_micro_batch_loss(lp_o.detach().numpy(), old, old, adv, m.astype(batch["attention_mask"].dtype), kl_kind="low_var_kl", kl_coef=1e-2, grad_accum=1)
    lp_o.backward(torch.from_numpy(gl))
    eng.store_logits = True
    _, _, gs = run(eng, store, b, dict(loss))
    names = [k for k, t in p32.items() if t.grad is not None and k.endswith(("q_proj.weight", "down_proj.weight"))]
    rel = lambda g, k: float((g[k] - p32[k].grad).norm() / p32[k].grad.norm())
    worst, worst_stored = max(rel(g1, k) for k in names), max(rel(gs, k) for k in names)
    print(f"tied={tied}: worst relative gradient error {worst:.4f}, with stored logits {worst_stored:.4f}; head {rel(g1, head):.4f} / {rel(gs, head):.4f}")
    assert worst <= (1.5 * worst_stored if tied else yard["grad_hf_bf16_rel_l2"]["worst_lm_q_and_down_proj"])
    assert rel(g1, head) <= 1.5 * rel(gs, head)


def test_worker_key_and_environment(monkeypatch):
    from spatialthinker_amd import model as mdl
    from verl.trainer.config import ActorConfig
    assert ActorConfig().store_logits is True
    cfg = mdl.VLConfig(**tiny.TINY)
    store = mdl.ParamStore(cfg, trainable=False)
    monkeypatch.setenv("ST_STORE_LOGITS", "0")
    assert mdl.Qwen25VL(cfg, store).store_logits is False
    monkeypatch.delenv("ST_STORE_LOGITS")
    assert mdl.Qwen25VL(cfg, store).store_logits is True
