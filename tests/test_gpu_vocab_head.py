"""Vocabulary-head operators (linear_log_probs, linear_topk_kl, top_log_probs) on the GPU against their definitions in 64 bits.

Tolerances are derived, not measured.  u32 = 2^-24, ub = 2^-8: the largest relative error of one rounding to fp32 / bf16.
  z    fp32 accumulation of H exact products in blocks of 32: |dz| <= ez = (H/32 + 32) u32 max_v sum_i |h_i w_vi| / temperature
  lse  the largest |dz| + a few fp32 roundings of values up to |z|: el = ez + 8 u32 max|z| + 2^-20 (2^-20: exp2 / log2 of about 1 ulp, sums of
       positive terms in a tree of depth < 16)
  d    = c q + target: |dd| <= ub |d| + |g| q (ez + el + 2^-20) / temperature
  dh   = d w: sum_v |dd| |w| + (V/32 + 96) u32 sum |d||w| + ub |dh|;   dw likewise over rows, + ub (bf16) or u32 (fp32), and ub |d| |h| more: a row's
       scale may stand in its bf16 hidden state."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U32, UB = 2.0 ** -24, 2.0 ** -8
F64, BF16 = torch.float64, torch.bfloat16


def make(T, H, V, seed, scale=1.0, pitch_h=0, pitch_w=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.empty(T, H + pitch_h, device="cuda", dtype=BF16).normal_(generator=g)[:, :H]
    w = torch.empty(V, H + pitch_w, device="cuda", dtype=BF16).normal_(0.0, 1.5 * scale / math.sqrt(H), generator=g)[:, :H]
    lab = torch.randint(0, V, (T,), device="cuda", generator=g)
    gr = torch.randn(T, device="cuda", generator=g)
    return g, h, w, lab, gr


def errors64(h, w, temperature):
    """(z, ez, el) in 64 bits, per row."""
    hd, wd = h.to(F64), w.to(F64)
    z = hd @ wd.t() / temperature
    mag = (hd.abs() @ wd.abs().t()).amax(1) / temperature
    ez = (h.shape[1] / 32 + 32) * U32 * mag
    el = ez + 8 * U32 * z.abs().amax(1) + 2.0 ** -20
    return z, ez, el


def check_grads(h, w, d, derr, dh, dw, dw_unit, dw_before=None):
    hd, wd = h.to(F64), w.to(F64)
    T, V = d.shape
    if dh is not None:
        want = d @ wd
        tol = derr @ wd.abs() + (V / 32 + 96) * U32 * (d.abs() @ wd.abs()) + UB * want.abs() + 1e-30
        assert dh.dtype == BF16
        over = ((dh.to(F64) - want).abs() / tol).max().item()
        assert over <= 1.0, f"dhidden: {over:.3f} of its tolerance"
    if dw is not None:
        want = d.t() @ hd
        tol = derr.t() @ hd.abs() + (UB * (1 + UB) + (T / 32 + 96) * U32) * (d.t().abs() @ hd.abs()) + 1e-30
        if dw_before is not None:
            want = want + dw_before.to(F64)
        tol = tol + 2 * dw_unit * (want.abs() + (dw_before.to(F64).abs() if dw_before is not None else 0.0))
        over = ((dw.to(F64) - want).abs() / tol).max().item()
        assert over <= 1.0, f"dweight: {over:.3f} of its tolerance"


SHAPES = [(1, 64, 1, 1.0), (1, 64, 2, 1.0), (1, 128, 300, 0.5), (3, 64, 7, 1.0), (5, 128, 255, 2.0), (17, 2048, 1000, 1.0), (64, 256, 256, 1.0),
          (65, 192, 257, 0.7), (255, 64, 1000, 1.0), (256, 512, 4096, 1.0), (257, 320, 511, 1.3), (300, 576, 2049, 1.0), (33, 64, 50257, 1.0),
          (100, 256, 3001, 1.0), (128, 512, 1111, 0.8), (129, 3584, 3001, 1.0), (700, 256, 9999, 1.0)]


@pytest.mark.parametrize("T,H,V,temperature", SHAPES)
def test_linear_log_probs_forward_and_gradients(T, H, V, temperature):
    from verl.utils import torch_functional as VF
    print(f"case T={T} H={H} V={V} temperature={temperature}", flush=True)
    g, h, w, lab, gr = make(T, H, V, T * 7 + V)
    lab[torch.rand(T, device="cuda", generator=g) < 0.1] = -100
    if T > 4:
        lab[1], lab[2] = V, 2 ** 40                                # outside the vocabulary: not scored
        gr[3] = 0.0
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    lp = VF.linear_log_probs(hh, ww, lab, temperature)
    z, ez, el = errors64(h, w, temperature)
    live = (lab >= 0) & (lab < V)
    lse = torch.logsumexp(z, 1)
    want = torch.where(live, z.gather(1, lab.clamp(0, V - 1)[:, None])[:, 0] - lse, 0.0)
    assert lp.dtype == torch.float32 and lp.shape == (T,)
    assert (lp[~live] == 0).all()
    assert ((lp.to(F64) - want).abs() <= ez + el + U32 * want.abs()).all(), ((lp.to(F64) - want).abs() / (ez + el)).max()
    dh, dw = torch.autograd.grad(lp, (hh, ww), gr)
    gt = torch.where(live, gr.to(F64), 0.0)[:, None] / temperature
    q = (z - lse[:, None]).exp()
    d = -gt * q
    d[live] = d[live].scatter_add(1, lab[live][:, None], gt[live])
    derr = UB * d.abs() + gt.abs() * q * (ez + el + 2.0 ** -20)[:, None]
    check_grads(h, w, d, derr, dh, dw, UB)
    assert (dh[~live] == 0).all()


@pytest.mark.parametrize("T", [1, 40, 100, 150, 200, 300])
def test_log_probs_of_nearly_certain_tokens_keep_their_digits(T):
    """logp = -log(1 + y), y = sum exp(z_v - z_label) down to 1e-12: each term's relative error is that of its exponent, at most 2 ez + 2^-20 (exp2, log1p
    and the sums of positive terms included), and so is logp's, however small it is."""
    from verl.utils import torch_functional as VF
    H, V = 64, 1003
    g, h, w, lab, gr = make(T, H, V, 31 + T)
    scale = torch.linspace(4.0, 18.0, T, device="cuda") if T > 1 else torch.tensor([9.0], device="cuda")
    h = (scale[:, None] * w[lab].float()).to(BF16)
    z, ez, _ = errors64(h, w, 1.0)
    rest = (z - z.gather(1, lab[:, None])).scatter(1, lab[:, None], -math.inf).exp().sum(1)
    want = -torch.log1p(rest)
    got = VF.linear_log_probs(h, w, lab)
    assert want.max() > -1e-4 and ((got.to(F64) - want).abs() <= want.abs() * (2 * ez + 2.0 ** -20)).all(), ((got.to(F64) - want).abs() / want.abs()).max()
    ids = lab.to(torch.int32)[:, None].contiguous()                # a teacher that is certain: kl = -logp
    kl = VF.linear_topk_kl(h, w, ids, torch.zeros(T, 1, device="cuda"))
    assert ((kl.to(F64) + want).abs() <= want.abs() * (2 * ez + 2.0 ** -20)).all()
    tied = w.clone()                                               # two equal maxima: log 2 each, and nothing lost
    other = (lab + 1) % V
    tied[other] = w[lab]
    z = h.to(F64) @ tied.to(F64).t()
    assert ((VF.linear_log_probs(h, tied, lab).to(F64) - (z.gather(1, lab[:, None])[:, 0] - torch.logsumexp(z, 1))).abs() <= 2 * ez + 2.0 ** -20).all()


def test_more_than_one_piece_of_the_vocabulary():
    """T = 2100 rows leave 127 488 columns per piece: V = 150 001 takes two, the second one ending inside a tile."""
    from verl.utils import torch_functional as VF
    T, H, V = 2100, 64, 150001
    g, h, w, lab, gr = make(T, H, V, 5)
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    lp = VF.linear_log_probs(hh, ww, lab)
    dh, dw = torch.autograd.grad(lp, (hh, ww), gr)
    z, ez, el = errors64(h, w, 1.0)
    lse = torch.logsumexp(z, 1)
    want = z.gather(1, lab[:, None])[:, 0] - lse
    assert ((lp.to(F64) - want).abs() <= ez + el + U32 * want.abs()).all()
    q = (z - lse[:, None]).exp_()
    del z
    gd = gr.to(F64)[:, None]
    derr = gd.abs() * q * (ez + el + 2.0 ** -20)[:, None]
    d = q.mul_(-gd).scatter_add_(1, lab[:, None], gd)
    derr += UB * d.abs()
    check_grads(h, w, d, derr, dh, dw, UB)


@pytest.mark.parametrize("T", [20, 100, 190, 250, 300])
@pytest.mark.parametrize("accumulate", [False, True])
def test_fp32_weight_gradient_and_single_gradients(T, accumulate):
    from spatialthinker_amd import ops
    H, V, temperature = 192, 1500, 1.0
    g, h, w, lab, gr = make(T, H, V, 11, pitch_h=8, pitch_w=16)
    assert h.stride(0) == H + 8 and w.stride(0) == H + 16
    logp, lse = ops.linear_logprob_fwd(h, w, lab, temperature)
    before = torch.randn(V, H, device="cuda", generator=g)
    pitched = torch.zeros(V, H + 4, device="cuda")
    pitched[:, :H] = before
    pitched[:, H:] = 7.0
    assert ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, temperature, want_dhidden=False, dweight_f32=pitched[:, :H], accumulate=accumulate) is None
    dh = ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, temperature)
    dwb = torch.empty(V, H, dtype=BF16, device="cuda")
    assert torch.equal(dh, ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, temperature, dweight=dwb))
    z, ez, el = errors64(h, w, temperature)
    q = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
    d = (-gr.to(F64)[:, None] * q).scatter_add(1, lab[:, None], gr.to(F64)[:, None])
    derr = UB * d.abs() + gr.to(F64).abs()[:, None] * q * (ez + el + 2.0 ** -20)[:, None]
    check_grads(h, w, d, derr, dh, pitched[:, :H], U32, before if accumulate else None)
    check_grads(h, w, d, derr, None, dwb, UB)
    assert (pitched[:, H:] == 7.0).all()                           # behind the rows: untouched


@pytest.mark.parametrize("T,H,V", [(150, 192, 50257), (250, 448, 50257), (190, 192, 100001), (256, 320, 100001), (140, 320, 140003), (200, 192, 140003)])
def test_column_ranges_of_the_weight_gradient(T, H, V):
    """Two, one and three column ranges (197, 391 and 547 row blocks on 256 compute units)."""
    test_weight_gradient_of_129_to_256_rows_over_a_large_vocabulary(T, H, V)


@pytest.mark.parametrize("T", [129, 160, 161, 192, 193, 256])
@pytest.mark.parametrize("H", [64, 192, 448])
def test_weight_gradient_of_129_to_256_rows_over_a_large_vocabulary(T, H, V=33001):
    """From 32 513 columns on (two row blocks of 256 per compute unit) these row counts have a weight-gradient kernel of their own: all of its row tiles and
    outputs, column ranges that are uneven or fewer than three, a vocabulary that ends inside a tile, logits kept and formed again, a pitched result."""
    from spatialthinker_amd import ops
    temperature = 0.8
    print(f"case T={T} H={H} V={V}", flush=True)
    g, h, w, lab, gr = make(T, H, V, T + H, pitch_h=8, pitch_w=24)
    dead = torch.rand(T, device="cuda", generator=g) < 0.1
    lab[dead] = -100
    h[dead] = float("nan")
    z, ez, el = errors64(h.masked_fill(dead[:, None], 0.0), w, temperature)
    kept = ops.head_logits_buffer(T, V, h.device)
    logp, lse = ops.linear_logprob_fwd(h, w, lab, temperature, logits=kept)
    gt = torch.where(dead, 0.0, gr.to(F64))[:, None] / temperature
    q = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
    d = (-gt * q).scatter_add(1, lab.clamp(min=0)[:, None], gt)
    derr = UB * d.abs() + gt.abs() * q * (ez + el + 2.0 ** -20)[:, None]
    hx = h.masked_fill(dead[:, None], 0.0)
    before = torch.randn(V, H, device="cuda", generator=g)
    for logits in (kept, None):
        for dtype, accumulate in ((BF16, False), (torch.float32, False), (torch.float32, True)):
            buf = torch.full((V + 1, H + 16), 7.0, dtype=dtype, device="cuda")
            out = buf[:V, :H]
            if accumulate:
                out.copy_(before)
            how = dict(dweight=out) if dtype == BF16 else dict(dweight_f32=out, accumulate=accumulate)
            dh = ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, temperature, logits=logits, **how)
            check_grads(hx, w, d, derr, dh, out, UB if dtype == BF16 else U32, before if accumulate else None)
            assert (buf[:, H:] == 7.0).all() and (buf[V] == 7.0).all()


@pytest.mark.parametrize("T", [3, 40, 70, 100, 150, 200, 300])
def test_rows_do_not_depend_on_their_neighbours_and_infinite_logits_give_nan(T):
    """Every third row is watched; the rows between are flat, then nearly certain, then overflow to a +inf logit.  The watched rows' outputs keep their bits,
    and a row with a +inf logit has NaN log-probs (what inf - inf gives in log_softmax) whatever stands beside it and however many rows there are."""
    from spatialthinker_amd import ops
    H, V, K = 64, 1003, 3
    g, h, w, lab, gr = make(T, H, V, 13 + T)
    h[:, 0] = 0
    w[:, 0] = 0
    w[5, 0] = 1e20                                                 # times 1e20: beyond fp32 in column 5 only
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g, dtype=torch.int32)
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    watched = torch.arange(T, device="cuda") % 3 == 1
    lab[0] = 5
    outs = []
    for kind in ("flat", "certain", "infinite"):
        x = h.clone()
        if kind == "flat":
            x[~watched] *= 0.01
        if kind == "certain":
            x[~watched] = (12.0 * w[(lab[~watched] + 7) % V].float()).masked_fill(torch.arange(H, device="cuda") == 0, 0.0).to(BF16)
        if kind == "infinite":
            x[~watched, 0] = 1e20
        logp, lse = ops.linear_logprob_fwd(x, w, lab)
        kl, lse2, logq = ops.linear_topk_kl_fwd(x, w, ids, a)
        outs.append([t[watched] for t in (logp, lse, kl, logq)])
        for t in (logp, lse, kl):
            assert (torch.isnan(t[~watched]).all() if kind == "infinite" else torch.isfinite(t).all()), kind
        assert all(torch.isfinite(t).all() for t in outs[-1])
        assert all(torch.equal(x0, x1) for x0, x1 in zip(outs[0], outs[-1])), kind
    x = h.clone()
    x[:, 0] = -1e20                                                # -inf in column 5: its probability is 0, nothing else changes
    logp, lse = ops.linear_logprob_fwd(x, w, lab)
    z = (h.to(F64) @ w.to(F64).t())
    z[:, 5] = -math.inf
    _, ez, el = errors64(h[:, 1:], w[:, 1:], 1.0)
    want = torch.log_softmax(z, 1).gather(1, lab[:, None])[:, 0]
    assert torch.equal(torch.isneginf(logp), torch.isneginf(want)) and torch.isneginf(logp[0])
    ok = torch.isfinite(want)
    assert ((logp.to(F64) - want).abs() <= ez + el + U32 * want.abs())[ok].all()


@pytest.mark.parametrize("op", ["labels", "topk"])
def test_rows_without_a_gradient_may_hold_anything(op):
    """Unscored rows with NaN / infinite hidden states: the other rows' results have the same bits as with zeros there."""
    from spatialthinker_amd import ops
    T, H, V, K = 70, 128, 777, 5
    g, h, w, lab, gr = make(T, H, V, 3)
    dead = torch.zeros(T, dtype=torch.bool, device="cuda")
    dead[[0, 13, 64, 69]] = True
    lab[dead] = -1
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g, dtype=torch.int32)
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1) - 0.1
    ids[dead] = -1
    a[dead] = float("nan")
    res = []
    for fill in (0.0, float("nan"), float("inf"), -float("inf")):
        x = h.clone()
        x[dead] = fill
        dw = torch.empty(V, H, dtype=BF16, device="cuda")
        if op == "labels":
            out, lse = ops.linear_logprob_fwd(x, w, lab)
            dh = ops.linear_logprob_bwd(x, w, lab, out, lse, gr, dweight=dw)
        else:
            out, lse, logq = ops.linear_topk_kl_fwd(x, w, ids, a)
            dh = ops.linear_topk_kl_bwd(x, w, ids, a, lse, logq, gr, dweight=dw)
        res.append((out, dh, dw))
        assert (out[dead] == 0).all() and (dh[dead] == 0).all() and torch.isfinite(dw).all()
        for x0, x1 in zip(res[0], res[-1]):
            assert torch.equal(x0, x1)


def kl64(z, ids, a, renorm):
    V = z.shape[1]
    have = (ids >= 0) & (ids < V)
    a = a.to(F64).masked_fill(~have, -math.inf)
    if renorm:
        a = a - torch.logsumexp(a, 1, keepdim=True).clamp(min=-1e300)
    p = a.exp()
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    at = logq.gather(1, ids.long().clamp(0, V - 1))
    kl = torch.where(p > 0, p * (a - at), 0.0).sum(1)
    return kl, p, logq, at


@pytest.mark.parametrize("T,H,V,K,temperature,renorm", [(1, 64, 5, 1, 1.0, False), (2, 64, 40, 3, 0.5, True), (37, 128, 333, 8, 2.0, True), (70, 192, 257, 64, 1.0, False),
                                                       (260, 64, 1999, 33, 1.0, True), (65, 2048, 1000, 100, 1.0, False), (9, 64, 600, 1024, 1.0, True), (128, 256, 700, 20, 1.0, True)])
def test_linear_topk_kl_forward_and_gradients(T, H, V, K, temperature, renorm):
    from verl.utils import torch_functional as VF
    print(f"case T={T} H={H} V={V} K={K} renorm={renorm}", flush=True)
    g, h, w, lab, gr = make(T, H, V, V + K)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)                  # ids repeat within rows
    a = torch.log_softmax(2.0 * torch.randn(T, K, device="cuda", generator=g), 1) - 0.3
    gone = torch.rand(T, K, device="cuda", generator=g) < 0.15
    ids[gone] = -1
    a[gone] = float("nan")
    if K >= 8:
        a[0, :2] = -math.inf                                       # a zero probability is present but weighs nothing
        ids[1, 0], a[1, 0] = V, 0.5                                # outside the vocabulary: absent
        ids[T // 2] = -1                                           # a row without entries
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    kl = VF.linear_topk_kl(hh, ww, ids, a, temperature, renorm)
    z, ez, el = errors64(h, w, temperature)
    want, p, logq, at = kl64(z, ids, a, renorm)
    P = p.sum(1)
    # log p: the given fp32 number (renorm: two roundings and a sum more), each p to about 4 ulp (+ |log p| ulp from exp's argument)
    rel_p = (8 + K / 64 + 2 * a.nan_to_num(0, 0, 0).abs().amax(1).to(F64)) * 2 * U32
    terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log().abs() + at.abs()), 0.0).sum(1)
    tol = P * (ez + el) + (rel_p + (K / 64 + 10) * U32) * (terms + P) + 1e-30
    assert kl.dtype == torch.float32 and ((kl.to(F64) - want).abs() <= tol).all(), ((kl.to(F64) - want).abs() / tol).max()
    dh, dw = torch.autograd.grad(kl, (hh, ww), gr)
    gt = gr.to(F64)[:, None] / temperature
    q = logq.exp()
    d = gt * q * P[:, None]
    dabs = d.abs()
    sparse = torch.zeros_like(d).scatter_add_(1, ids.clamp(0, V - 1), p)
    d = d - gt * sparse
    derr = UB * d.abs() + dabs * (ez + el + 2.0 ** -20 + rel_p)[:, None] + gt.abs() * sparse * (rel_p + 2.0 ** -20)[:, None]
    check_grads(h, w, d, derr, dh, dw, UB)
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("T", [5, 40, 100, 150, 200, 300])
@pytest.mark.parametrize("exponent", [20, 24, 27, 30, 34, 60])
def test_logits_whose_rounding_exceeds_one_stay_finite(T, exponent):
    """Logits of 2^exponent and more: their fp32 rounding is larger than any difference that counts, so log-probs are as good as that (ez + el), but the label
    that is its row's maximum still has between 1 / V and all of the probability, and nothing overflows, backward included."""
    from spatialthinker_amd import ops
    H, V = 64, 900
    print(f"case T={T} exponent={exponent}", flush=True)
    g, h, w, lab, gr = make(T, H, V, 3 * T + exponent)
    h = (h.float() * 2.0 ** exponent).to(BF16)
    z, ez, el = errors64(h, w, 1.0)
    lab[::2] = z.argmax(1)[::2]
    kept = ops.head_logits_buffer(T, V, h.device)
    logp, lse = ops.linear_logprob_fwd(h, w, lab, logits=kept)
    assert ((lse.to(F64) - torch.logsumexp(z, 1)).abs() <= el).all()
    want = torch.log_softmax(z, 1).gather(1, lab[:, None])[:, 0]
    assert ((logp.to(F64) - want).abs() <= ez + el + U32 * want.abs()).all()
    assert (logp <= 0).all() and (logp[::2] >= -math.log(V) - ez[::2]).all()
    if exponent >= 27:                                             # two logits of a row nearer than a rounding of them: none in these rows
        assert (logp[::2] == 0).all()
    grads = []
    for logits in (kept, None):
        dw = torch.empty(V, H, dtype=BF16, device="cuda")
        grads.append((ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw, logits=logits), dw))
    for x, y in zip(*grads):
        assert torch.isfinite(x).all() and torch.equal(x, y)


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T", [6, 200])
def test_a_teacher_of_nan_is_not_silent(T, renorm):
    """NaN log-probs of present entries, some or all of a row's: that row's KL and hidden gradient are NaN, the other rows' are what they are without it."""
    from spatialthinker_amd import ops
    H, V, K = 64, 300, 5
    g, h, w, lab, gr = make(T, H, V, 17)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g, dtype=torch.int32)
    ids[:, 4] = -1
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    a[:, 4] = float("nan")                                         # absent: not read as a number
    bad = a.clone()
    bad[1, 2] = float("nan")
    bad[4] = float("nan")
    res = []
    for x in (a, bad):
        kl, lse, logq = ops.linear_topk_kl_fwd(h, w, ids, x, 1.0, renorm)
        res.append((kl, ops.linear_topk_kl_bwd(h, w, ids, x, lse, logq, gr, 1.0, renorm)))
    rows = torch.zeros(T, dtype=torch.bool, device="cuda")
    rows[[1, 4]] = True
    for good, got in zip(*res):
        assert torch.isfinite(good).all() and torch.isnan(got[rows]).all() and torch.equal(got[~rows], good[~rows])


@pytest.mark.parametrize("T", [32, 33, 77, 96, 97, 128, 130, 160, 161])
@pytest.mark.parametrize("H", [64, 192, 2048])
def test_row_tiles_of_the_weight_stream(T, H):
    """The last and first row counts of each tile, with fewer, as many and more steps of 64 than copies in flight; H = 2048: rows at a pitch of 4 KiB."""
    test_linear_log_probs_forward_and_gradients(T, H, 701, 1.0)
    test_linear_topk_kl_forward_and_gradients(T, H, 519, 40, 1.0, True)


@pytest.mark.parametrize("T,V", [(1, 5), (31, 333), (33, 257), (64, 1000), (96, 701), (128, 640), (129, 701), (160, 4001), (161, 999), (256, 700), (257, 1111), (700, 3000)])
def test_kept_logits_give_the_same_bits(T, V):
    """Logits read back and logits formed again: outputs and gradients are equal, and only what has to be kept is allocated."""
    from verl.utils import torch_functional as VF
    H, K = 192, 7
    g, h, w, lab, gr = make(T, H, V, T + V)
    lab[torch.rand(T, device="cuda", generator=g) < 0.2] = -100
    h[lab < 0] = float("nan")
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)
    ids[lab < 0] = -1
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    for fn in (lambda x, y, keep: VF.linear_log_probs(x, y, lab, 0.7, keep_logits=keep), lambda x, y, keep: VF.linear_topk_kl(x, y, ids, a, 0.7, True, keep_logits=keep)):
        outs = []
        need = T * ((V + 63) // 64 * 64) * 4
        for keep in (0, need - 1, need, 8 << 30):
            hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            out = fn(hh, ww, keep)
            assert (out.grad_fn.saved_tensors[-1] is not None) == (keep >= need)
            outs.append((out.detach(),) + torch.autograd.grad(out, (hh, ww), gr))
            with pytest.raises(RuntimeError):                      # what was kept went with the backward
                out.grad_fn.saved_tensors
        live = lab >= 0
        for o in outs[1:]:
            assert torch.equal(o[0][live], outs[0][0][live]) and torch.equal(o[1], outs[0][1]) and torch.equal(o[2], outs[0][2])
        assert torch.isfinite(outs[0][1]).all() and torch.isfinite(outs[0][2]).all()
        with torch.no_grad():
            assert torch.equal(fn(h, w, 8 << 30)[live], outs[0][0][live])


@pytest.mark.parametrize("T,V", [(1, 5), (20, 70), (64, 129), (65, 70), (100, 300), (150, 70), (150, 257), (161, 70), (300, 70), (300, 577)])
def test_kept_logits_in_a_part_of_a_wider_buffer(T, V):
    """Kept logits as columns of a wider buffer, first and last columns of it: what lies in front of and behind the view is left alone, and the backward
    reads the view (bits as without kept logits)."""
    from spatialthinker_amd import ops
    print(f"case T={T} V={V}", flush=True)
    H, wide, cols = 64, 1024, (V + 63) // 64 * 64
    g, h, w, lab, gr = make(T, H, V, T + V)
    logp, lse = ops.linear_logprob_fwd(h, w, lab)
    dw = torch.empty(V, H, dtype=BF16, device="cuda")
    dh = ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw)
    for at in (0, 192, wide - cols):
        buf = torch.full((T + 1, wide), 7.0, device="cuda")
        view = buf[:T, at:at + cols]
        assert view.stride(0) == wide
        out = ops.linear_logprob_fwd(h, w, lab, logits=view)
        assert torch.equal(out[0], logp) and torch.equal(out[1], lse)
        assert (buf[:, :at] == 7.0).all() and (buf[:, at + cols:] == 7.0).all() and (buf[T] == 7.0).all()
        z, ez, _ = errors64(h, w, 1.0)
        assert ((view[:, :V].to(F64) - z).abs() <= ez[:, None]).all()
        dwz = torch.empty_like(dw)
        assert torch.equal(ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dwz, logits=view), dh) and torch.equal(dwz, dw)


def test_kept_logits_give_the_same_bits_over_pieces_of_a_pitched_weight():
    """130 rows leave 1 398 016 columns per piece; weight rows at a pitch of 4 KiB are summed from another K-step on per column block, which has to be the
    same one in a piece as in the whole vocabulary."""
    from spatialthinker_amd import ops
    T, H, V = 130, 192, 1400003
    g = torch.Generator(device="cuda").manual_seed(9)
    h = torch.empty(T, H, device="cuda", dtype=BF16).normal_(generator=g)
    w = torch.empty(V, 2048, device="cuda", dtype=BF16)[:, :H]
    w.copy_(torch.empty(V, H, device="cuda", dtype=BF16).normal_(0.0, 0.3, generator=g))
    lab = torch.randint(0, V, (T,), device="cuda", generator=g)
    lab[:40] = V - 1 - lab[:40] % 1000                             # targets in the second piece
    gr = torch.randn(T, device="cuda", generator=g)
    z = ops.head_logits_buffer(T, V, h.device)
    logp, lse = ops.linear_logprob_fwd(h, w, lab, logits=z)
    grads = []
    for kept in (z, None):
        dw = torch.empty(V, H, dtype=BF16, device="cuda")
        grads.append((ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw, logits=kept), dw))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


def test_kept_logits_of_several_pieces_and_in_a_captured_graph():
    from spatialthinker_amd import ops
    from verl.utils import torch_functional as VF
    T, H, V = 2100, 64, 150001
    g, h, w, lab, gr = make(T, H, V, 5)
    outs = []
    for keep in (0, 1 << 31):
        hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        lp = VF.linear_log_probs(hh, ww, lab, keep_logits=keep)
        outs.append((lp,) + torch.autograd.grad(lp, (hh, ww), gr))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    del outs
    T, V = 150, 3000
    g, h, w, lab, gr = make(T, H, V, 6)

    def step():
        z = ops.head_logits_buffer(T, V, h.device)
        logp, lse = ops.linear_logprob_fwd(h, w, lab, logits=z)
        dw = torch.empty_like(w)
        return logp, ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw, logits=z), dw
    step()
    torch.cuda.synchronize()
    gph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gph):
        out = step()
    for _ in range(3):
        h.copy_(torch.randn(T, H, device="cuda", generator=g).to(BF16))
        want = [t.clone() for t in step()]
        gph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("keep", [0, 8 << 30])
def test_millions_of_rows_over_a_small_vocabulary(keep):
    """More row blocks than a grid has in its second and third dimension."""
    from verl.utils import torch_functional as VF
    T, H, V = 65535 * 64 + 100, 64, 5
    g, h, w, lab, gr = make(T, H, V, 77)
    hh = h.clone().requires_grad_(True)
    lp = VF.linear_log_probs(hh, w, lab, keep_logits=keep)
    assert (lp.grad_fn.saved_tensors[-1] is not None) == (keep > 0)
    dh, = torch.autograd.grad(lp, hh, gr)
    rows = torch.tensor([0, 63, 64, 255, 256, T // 2, T - 101, T - 100, T - 65, T - 64, T - 1], device="cuda")
    z, ez, el = errors64(h[rows], w, 1.0)
    lse = torch.logsumexp(z, 1)
    want = z.gather(1, lab[rows][:, None])[:, 0] - lse
    assert ((lp[rows].to(F64) - want).abs() <= ez + el + U32 * want.abs()).all()
    gt, q = gr[rows].to(F64)[:, None], (z - lse[:, None]).exp()
    d = (-gt * q).scatter_add(1, lab[rows][:, None], gt)
    check_grads(h[rows], w, d, UB * d.abs() + gt.abs() * q * (ez + el + 2.0 ** -20)[:, None], dh[rows], None, UB)


def test_gradients_against_differences():
    """Central differences along random directions: <dh, h+ - h-> against the change of sum(g out), for steps that bf16 holds exactly.  The third-order
    rest of a difference of width e |h| (logits move by < 0.03) is below 1e-4 of the change's scale; 2 % covers it, the bf16 gradients (2^-8 per
    entry, two roundings) and the fp32 noise of the outputs, which is added on its own."""
    from verl.utils import torch_functional as VF
    T, H, V, K = 40, 256, 900, 12
    g, h, w, lab, gr = make(T, H, V, 21)
    teacher = (h.float() + torch.randn(T, H, device="cuda", generator=g)).to(BF16)
    ids, a, _ = VF.top_log_probs(teacher @ w.t(), K)
    for fn in (lambda x, y: VF.linear_log_probs(x, y, lab), lambda x, y: VF.linear_topk_kl(x, y, ids, a, renormalize=True)):
        hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        dh, dw = torch.autograd.grad(fn(hh, ww), (hh, ww), gr)
        for x, grad, which in ((h, dh, 0), (w, dw, 1)):
            step = 2.0 ** -6 * torch.sign(torch.randn(x.shape, device="cuda", generator=g)) * x.float().abs()
            plus, minus = (x.float() + step).to(BF16), (x.float() - step).to(BF16)
            diff = plus.to(F64) - minus.to(F64)
            args = ((plus, w), (minus, w)) if which == 0 else ((h, plus), (h, minus))
            change = ((fn(*args[0]).to(F64) - fn(*args[1]).to(F64)) * gr.to(F64)).sum().item()
            by_grad = (grad.to(F64) * diff).sum().item()
            scale = math.sqrt((grad.to(F64) * diff).square().sum().item())
            noise = gr.abs().sum().item() * 2 * 2e-5
            assert abs(change - by_grad) <= 0.02 * (abs(change) + scale) + noise, (which, change, by_grad, scale)


# ---------------------------------------------------------------- top_log_probs
def top64(z, k, temperature):
    order = torch.sort(z.to(F64), dim=1, descending=True, stable=True)
    zz = z.to(F64) / temperature
    lse = torch.logsumexp(zz, 1)
    ids = order.indices[:, :k]
    return ids.to(torch.int32), zz.gather(1, ids) - lse[:, None], lse


def check_top(z, k, temperature=1.0):
    from spatialthinker_amd import ops
    ids, logp, lse = ops.topk_logprob(z, k, temperature)
    wi, wl, we = top64(z, k, temperature)
    assert ids.dtype == torch.int32 and torch.equal(ids, wi)
    fin = torch.isfinite(we)
    tol = 8 * U32 * (z.to(F64).masked_fill(~torch.isfinite(z), 0).abs().amax(1) / temperature + we.masked_fill(~fin, 0).abs()) + 2.0 ** -20
    assert ((lse.to(F64) - we).abs()[fin] <= tol[fin]).all()
    ok = torch.isfinite(wl)
    assert torch.equal(torch.isneginf(logp.to(F64)[fin]), torch.isneginf(wl[fin]))
    assert ((logp.to(F64) - wl).abs() <= tol[:, None])[ok].all()


@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (1, 7, 7), (2, 9, 3), (3, 256, 256), (1, 4096, 20), (5, 4103, 1), (4, 16384, 128), (1, 152064, 64), (2, 151936, 256),
                                   (700, 1000, 33), (600, 5000, 200), (1030, 333, 8), (513, 40001, 64)])
def test_top_log_probs(T, V, k):
    print(f"case T={T} V={V} k={k}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + V + k)
    z = (3 * torch.randn(T, V, device="cuda", generator=g)).to(BF16)               # 16-bit values over 150 000 places: many ties
    check_top(z, k, 1.0)
    check_top(z, k, 0.6)


def test_top_log_probs_beyond_2_31_elements():
    V, k = 152064, 20
    T = 2 ** 31 // V + 40
    g = torch.Generator(device="cuda").manual_seed(8)
    z = torch.empty(T, V, device="cuda", dtype=BF16).normal_(generator=g)
    from spatialthinker_amd import ops
    ids, logp, lse = ops.topk_logprob(z, k)
    rows = torch.tensor([0, 1, T // 2, T - 41, T - 40, T - 39, T - 1], device="cuda")
    wi, wl, we = top64(z[rows], k, 1.0)
    assert torch.equal(ids[rows], wi)
    assert ((lse[rows].to(F64) - we).abs() <= 8 * U32 * (8 + we.abs()) + 2.0 ** -20).all()
    assert ((logp[rows].to(F64) - wl).abs() <= 8 * U32 * (8 + we.abs()[:, None]) + 2.0 ** -20).all()


@pytest.mark.parametrize("T", [1, 600])
def test_top_log_probs_adversarial_orders(T):
    """Rows that rise (every value passes the threshold), fall, are constant, hold -inf, -0 and few distinct values."""
    V, k = 50001, 100
    g = torch.Generator(device="cuda").manual_seed(1)
    ramp = torch.linspace(-20, 20, V, device="cuda")
    rows = [ramp, -ramp, torch.zeros(V, device="cuda"), torch.zeros(V, device="cuda"), ramp.round(), torch.full((V,), -math.inf, device="cuda"),
            torch.where(torch.rand(V, device="cuda", generator=g) < 0.5, 0.0, -0.0), torch.randint(0, 3, (V,), device="cuda", generator=g).float()]
    rows[3][::2] = -0.0
    rows[5][[3, 77, 4096, 50000]] = torch.tensor([1.0, -2.0, 0.0, -0.0], device="cuda")
    z = torch.stack(rows).to(BF16)
    for i in range(z.shape[0]):
        check_top(z[i:i + 1].expand(T, V).contiguous(), k if i != 5 else 256)


@pytest.mark.parametrize("T,V", [(1, 152064), (24, 152064), (600, 50001), (3, 300), (7, 400), (5, 1000)])
@pytest.mark.parametrize("k", [10, 16, 20, 32, 48, 64, 96, 128, 256])
def test_top_log_probs_with_a_kth_value_far_below_the_largest(T, V, k):
    """Rows whose k-th largest lies more than 1023 bf16 steps (8 octaves, or a change of sign) below the largest: a few large logits over a bulk that is
    negative, tiny, zero or -inf.  One slice and joined; as few candidates as one short row has, and as many as a vocabulary leaves."""
    print(f"case T={T} V={V} k={k}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + V + k)
    bulks = [lambda n: -6.0 + torch.randn(n, device="cuda", generator=g), lambda n: 0.03 * torch.rand(n, device="cuda", generator=g),
             lambda n: -12.0 * torch.rand(n, device="cuda", generator=g), lambda n: 1e-30 * torch.randn(n, device="cuda", generator=g),
             lambda n: torch.zeros(n, device="cuda"), lambda n: torch.full((n,), -1.0, device="cuda"), lambda n: torch.full((n,), -math.inf, device="cuda")]
    rows = []
    for t in range(max(T, 3 * len(bulks))):
        z = bulks[t % len(bulks)](V)
        p = (1, 5, k - 1)[t // len(bulks) % 3]
        z[torch.randperm(V, device="cuda", generator=g)[:p]] = 8.0 + 4.0 * torch.rand(p, device="cuda", generator=g)
        rows.append(z.to(BF16))
    z = torch.stack(rows)
    for i in range(0, z.shape[0], T):
        check_top(z[i:i + T], k)


@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 13, 13), (64, 300, 20), (600, 5003, 64), (2, 152064, 100)])
@pytest.mark.parametrize("exponent", [10, 24, 29, 31, 40, 100])
def test_top_log_probs_of_huge_logits(T, V, k, exponent):
    """Logits of 2^exponent: finite log-probs as good as their fp32 rounding, at every alignment; with a temperature that takes them beyond fp32, NaN."""
    from spatialthinker_amd import ops
    print(f"case T={T} V={V} k={k} exponent={exponent}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + V + exponent)
    buf = (torch.randn(T, V + 9, device="cuda", generator=g) * 2.0 ** exponent).to(BF16)
    for off in (0, 3, 8):
        z = buf[:, off:off + V]
        _, logp, lse = ops.topk_logprob(z, k)
        assert torch.isfinite(lse).all() and torch.isfinite(logp).all()
        check_top(z, k)
        check_top(-z.abs(), k)
        check_top(torch.where(z > 0, z, -1.0).to(BF16), k)         # huge and ordinary logits in a row
    check_top((buf[:, :V] * 2.0 ** -exponent).to(BF16), k, 2.0 ** -min(exponent, 60))              # ordinary logits, made huge by the temperature
    check_top((buf[:, :V] * 2.0 ** -exponent).to(BF16), k, 1.3 * 2.0 ** -min(exponent, 60))
    ids, logp, lse = ops.topk_logprob(buf[:, :V].abs() + 2.0 ** exponent, k, 2.0 ** -40 if exponent == 100 else 1.0)
    assert torch.isnan(logp).all() == (exponent == 100) and (ids >= 0).all() and (ids < V).all()


def test_top_log_probs_pitch_alignment_and_special_rows():
    from spatialthinker_amd import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    buf = torch.randn(9, 3011, device="cuda", generator=g).to(BF16)
    for off in range(0, 9):
        for n in (1, 5, 8, 15, 1500, 3002):
            check_top(buf[:, off:off + n], min(n, 5))
    z = buf[:4].clone()
    z[0, 100] = math.nan
    z[1] = -math.inf
    z[2, 5] = math.inf
    ids, logp, lse = ops.topk_logprob(z, 40)
    for r in range(3):
        assert torch.isnan(logp[r]).all()
        assert len(set(ids[r].tolist())) == 40 and 0 <= ids[r].min() and ids[r].max() < 3011
    check_top(z[3:], 40)
    e = ops.topk_logprob(z[:0], 3)
    assert e[0].shape == (0, 3) and e[2].shape == (0,)


# ---------------------------------------------------------------- together, streams, graphs
def test_teacher_to_student_run():
    """What a distillation step with a policy term does: teacher logits -> top_log_probs -> linear_topk_kl + linear_log_probs on one head, against the
    same in 64-bit autograd on the values the operators saw."""
    from verl.utils import torch_functional as VF
    B, L, H, V, K = 3, 21, 192, 3001, 16
    g, h, w, lab, gr = make(B * L, H, V, 31)
    teacher_h = (h.float() + 0.5 * torch.randn(B * L, H, device="cuda", generator=g)).to(BF16)
    ids, a, _ = VF.top_log_probs((teacher_h @ w.t()).view(B, L, V), K, temperature=1.5)
    assert ids.shape == (B, L, K)
    lab = lab.view(B, L)
    lab[0, :4] = -100
    hh, ww = h.view(B, L, H).clone().requires_grad_(True), w.clone().requires_grad_(True)
    kl = VF.linear_topk_kl(hh, ww, ids, a, temperature=1.5, renormalize=True)
    lp = VF.linear_log_probs(hh, ww, lab)
    loss = kl.mean() - 0.5 * (lp * (lab >= 0)).sum() / (lab >= 0).sum()
    loss.backward()
    hd, wd = h.to(F64).requires_grad_(True), w.to(F64).requires_grad_(True)
    kl_d = kl64(hd @ wd.t() / 1.5, ids.view(-1, K), a.view(-1, K), True)[0]
    live = lab.view(-1) >= 0
    lp_d = torch.log_softmax(hd @ wd.t(), 1).gather(1, lab.view(-1).clamp(min=0)[:, None])[:, 0]
    loss_d = kl_d.mean() - 0.5 * lp_d[live].sum() / live.sum()
    loss_d.backward()
    assert abs(loss.item() - loss_d.item()) < 1e-5 * (1 + abs(loss_d.item()))
    # two bf16 gradients (each within a rounding of d and one of the result, in norm below 2 ub) and the bf16 sum
    assert (hh.grad.view(-1, H).to(F64) - hd.grad).norm() <= 3 * UB * hd.grad.norm()
    assert (ww.grad.to(F64) - wd.grad).norm() <= 3 * UB * wd.grad.norm()


@pytest.mark.parametrize("op", ["labels", "topk"])
def test_outputs_may_be_changed_in_place(op):
    """Masking the result in place, one- and two-dimensional: the gradient of the masked result, as out of place."""
    from verl.utils import torch_functional as VF
    T, H, V, K = 66, 64, 500, 4
    g, h, w, lab, gr = make(T, H, V, 4)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    mask = torch.rand(T, device="cuda", generator=g) < 0.3
    for shape in ((T,), (6, T // 6)):
        grads = []
        for inplace in (False, True):
            hh, ww = h.view(*shape, H).clone().requires_grad_(True), w.clone().requires_grad_(True)
            if op == "labels":
                out = VF.linear_log_probs(hh, ww, lab.view(shape))
            else:
                out = VF.linear_topk_kl(hh, ww, ids.view(*shape, K), a.view(*shape, K))
            out = out.masked_fill_(mask.view(shape), 0.0).mul_(2.0) if inplace else out.masked_fill(mask.view(shape), 0.0) * 2.0
            grads.append(torch.autograd.grad(out, (hh, ww), gr.view(shape)))
        assert all(torch.equal(x, y) for x, y in zip(*grads))


def test_empty_batches_and_fp32_inputs():
    from verl.utils import torch_functional as VF
    w = torch.randn(300, 64, device="cuda", requires_grad=True)                    # fp32 leaf: cast inside, fp32 gradient back
    h = torch.randn(2, 0, 64, device="cuda", requires_grad=True)
    lp = VF.linear_log_probs(h, w, torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (2, 0)
    lp.sum().backward()
    assert w.grad.dtype == torch.float32 and (w.grad == 0).all() and h.grad.shape == (2, 0, 64)
    h = torch.randn(5, 64, device="cuda").t().contiguous().t().requires_grad_(True)       # column-major rows
    lab = torch.arange(5, device="cuda", dtype=torch.int32)
    got = VF.linear_log_probs(h, w, lab)
    want = VF.linear_log_probs(h.detach().contiguous().to(BF16), w.detach().to(BF16), lab.long())
    assert torch.equal(got, want)
    got.sum().backward()
    assert h.grad.dtype == torch.float32


def test_other_streams_and_repeatability():
    from spatialthinker_amd import ops
    T, H, V = 150, 256, 5003
    g, h, w, lab, gr = make(T, H, V, 41)

    def once():
        logp, lse = ops.linear_logprob_fwd(h, w, lab)
        dw = torch.empty(V, H, dtype=BF16, device="cuda")
        dh = ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw)
        return (logp, dh, dw) + ops.topk_logprob(dw.t().contiguous().t()[:7, :5].contiguous(), 3)
    base = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:                                              # three calls in flight at once
        with torch.cuda.stream(s):
            outs.append([once() for _ in range(3)])
    torch.cuda.synchronize()
    for per in outs:
        for r in per:
            assert all(torch.equal(x, y) for x, y in zip(base, r))


def test_captured_graphs_replay_with_eager_work_between():
    from spatialthinker_amd import ops
    T, H, V, K = 90, 128, 3000, 6
    g, h, w, lab, gr = make(T, H, V, 51)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g, dtype=torch.int32)
    a = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    z = torch.randn(3, 40000, device="cuda", generator=g).to(BF16)

    def labels():
        logp, lse = ops.linear_logprob_fwd(h, w, lab)
        dw = torch.empty(V, H, dtype=BF16, device="cuda")
        return logp, ops.linear_logprob_bwd(h, w, lab, logp, lse, gr, dweight=dw), dw

    def distill():
        kl, lse, logq = ops.linear_topk_kl_fwd(h, w, ids, a, 1.0, True)
        dw = torch.zeros(V, H, device="cuda")
        return (kl, ops.linear_topk_kl_bwd(h, w, ids, a, lse, logq, gr, 1.0, True, dweight_f32=dw, accumulate=True), dw) + ops.topk_logprob(z, 9)
    graphs = []
    for fn in (labels, distill):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            out = fn()
        graphs.append((fn, gph, out))
    for i in range(4):
        h.copy_(torch.randn(T, H, device="cuda", generator=g).to(BF16))            # new inputs in the captured buffers
        z.copy_(torch.randn(3, 40000, device="cuda", generator=g).to(BF16))
        wants = [[t.clone() for t in fn()] for fn, _, _ in graphs]
        torch.cuda.synchronize()
        for _, gph, _ in graphs:
            gph.replay()
        eager = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        assert torch.isfinite(eager).all()
        torch.cuda.synchronize()
        for (_, _, out), want in zip(graphs, wants):
            assert all(torch.equal(x, y) for x, y in zip(out, want)), i
