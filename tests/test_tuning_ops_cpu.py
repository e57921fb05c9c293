"""Expert selection, preference loss and AdamW with 8-bit moments on the CPU: definitions against independent forms, refusals."""
import math

import pytest
import torch

from shadowspill_b200.ops import functional as F, reference as R, routing


# ------------------------------------------------------------------------ expert selection
def _by_hand(row, k, scoring, bias, groups, keep, renorm, scale):
    s = [1 / (1 + math.exp(-v)) for v in row]
    if scoring == "softmax":
        top = max(row)
        e = [math.exp(v - top) for v in row]
        s = [v / sum(e) for v in e]
    key = [v + b for v, b in zip(s, bias)]
    size = len(row) // groups
    score = [sum(sorted(key[g * size:(g + 1) * size])[-2:]) for g in range(groups)]
    kept = sorted(range(groups), key=lambda g: (-score[g], g))[:keep]
    ids = sorted((e for e in range(len(row)) if e // size in kept), key=lambda e: (-key[e], e))[:k]
    total = sum(s[e] for e in ids) + 1e-20 if renorm else 1.0
    return ids, [s[e] / total * scale for e in ids]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2), (8, 8)])
@pytest.mark.parametrize("renorm", [True, False])
def test_selection_against_a_loop(scoring, groups, keep, renorm):
    g = torch.Generator().manual_seed(1)
    x, bias = torch.randn(20, 24, generator=g), torch.randn(24, generator=g) * 0.2
    ids, w, counts = routing.select_experts(x, 3, scoring=scoring, bias=bias, groups=groups, keep_groups=keep, renormalize=renorm, scale=1.5)
    for t in range(20):
        want, weights = _by_hand(x[t].tolist(), 3, scoring, bias.tolist(), groups, keep, renorm, 1.5)
        assert ids[t].tolist() == want
        assert w[t].tolist() == pytest.approx(weights, rel=2.0 ** -23)       # rounded once to fp32
    assert counts.tolist() == [int((ids == e).sum()) for e in range(24)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_selection_gradient_against_differences(scoring, renorm):
    g = torch.Generator().manual_seed(2)
    x, dw = torch.randn(6, 16, generator=g, dtype=torch.float64), torch.randn(6, 4, generator=g)
    ids, _, _ = R.select_experts(x, 4, scoring)
    got = R.select_experts_bwd(x, ids, dw, scoring, renorm, 2.0)

    def value(y):
        c = R.expert_scores(y, scoring).gather(1, ids.long())
        c = c / (c.sum(1, keepdim=True) + 1e-20) if renorm else c
        return (2.0 * c * dw).sum()
    want = torch.zeros_like(x)
    for i in range(6):
        for e in range(16):
            d = torch.zeros_like(x)
            d[i, e] = 1e-5
            want[i, e] = (value(x + d) - value(x - d)) / 2e-5
    # h^2 / 6 times a third derivative under 10, and 2^-52 of the value over h
    assert float((got - want).abs().max()) <= 1e-9


def test_selection_refuses():
    x = torch.zeros(3, 8)
    for bad in (dict(k=0), dict(k=9), dict(k=33), dict(k=5, groups=4, keep_groups=2), dict(k=1, groups=3), dict(k=1, groups=2, keep_groups=3),
                dict(k=1, groups=2, keep_groups=0), dict(k=1, scoring="tanh"), dict(k=1, bias=torch.zeros(7)),
                dict(k=1, bias=torch.zeros(8, dtype=torch.float64))):
        with pytest.raises(ValueError):
            routing.select_experts(x, **bad)
    with pytest.raises(TypeError):
        routing.select_experts(x.half(), 2)
    with pytest.raises(TypeError):
        routing.select_experts(x[0], 2)
    with pytest.raises(ValueError):
        routing.select_experts(torch.zeros(2, 513), 2)
    ids = torch.zeros(3, 2, dtype=torch.int32)
    for bad in ((ids.long(), torch.zeros(3, 2)), (ids, torch.zeros(3, 3)), (ids[:2], torch.zeros(2, 2))):
        with pytest.raises(ValueError):
            routing.select_experts_bwd(x, *bad)


# ------------------------------------------------------------------------ preference loss
def _pairs(R_rows=30, V=50, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, t = torch.randn(R_rows, V, generator=g), torch.randint(0, V, (R_rows,), generator=g)
    w = (torch.rand(R_rows, generator=g) + 0.2) * (torch.rand(R_rows, generator=g) < 0.8)
    return x, t, w, torch.tensor([0, 8, 15, 20, 28], dtype=torch.int32), torch.randn(R_rows, generator=g)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("average", [True, False])
def test_preference_against_autograd(kind, average):
    x, t, w, cu, ref = _pairs()
    x[3] = float("nan")
    w[3] = 0.0
    t[9] = -100
    logits, sums, loss = x.clone(), torch.empty(4), torch.full((1,), 2.0)
    smooth = 0.1 if kind == "sigmoid" else 0.0
    F.preference_(logits, t, w, cu, loss, beta=0.7, kind=kind, label_smoothing=smooth, average=average, ref_logp=ref, sums=sums, grad_scale=0.5)
    x64 = x.nan_to_num().double().requires_grad_(True)
    ok = (t >= 0) & (w != 0)
    lp = torch.log_softmax(x64, 1).gather(1, t.clamp(min=0)[:, None])[:, 0]
    s = []
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        ww = torch.where(ok, w, 0.0)[a:b].double()
        s.append((ww * (lp - ref.double())[a:b]).sum() / (ww.sum() if average else 1.0))
    want = torch.zeros((), dtype=torch.float64)
    for i in (0, 2):
        z = 0.7 * (s[i] - s[i + 1])
        want = want + (-0.9 * torch.log(torch.sigmoid(z)) - 0.1 * torch.log(1 - torch.sigmoid(z)) if kind == "sigmoid" else
                       torch.clamp(1 - z, min=0) if kind == "hinge" else (z / 0.7 - 1 / 1.4) ** 2)
    grad = torch.autograd.grad(want * 0.5, x64)[0]
    # fp32 log-probabilities of 50 words: a few roundings of numbers up to 8
    assert float(loss) - 2.0 == pytest.approx(float(want.detach()), rel=2e-5, abs=2e-5)
    assert torch.allclose(sums.double(), torch.stack(s).detach(), rtol=2e-5, atol=2e-5)
    assert torch.allclose(logits.double(), grad, rtol=2e-5, atol=2e-5)
    assert float(logits[28:].abs().sum()) == 0.0 and float(logits[3].abs().sum()) == 0.0


def test_preference_refuses():
    x, t, w, cu, ref = _pairs()
    loss = torch.zeros(1)
    good = dict(logits=x, targets=t, weights=w, cu_seqlens=cu, loss_sum=loss)
    for bad in (dict(kind="rank"), dict(beta=0.0), dict(label_smoothing=1.0), dict(kind="hinge", label_smoothing=0.1), dict(cu_seqlens=cu[:4]),
                dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:0]), dict(targets=t.int()), dict(targets=t[:5]), dict(weights=w.double()),
                dict(weights=w[:3]), dict(ref_logp=ref[:3]), dict(sums=torch.zeros(3)), dict(logp=torch.zeros(3)), dict(loss_sum=torch.zeros(2)),
                dict(grad=x.bfloat16()), dict(grad=x[:3])):
        with pytest.raises(ValueError):
            F.preference_(**{**good, **bad})
    assert float(loss) == 0.0


def test_preference_without_pairs():
    x, t, w, _, _ = _pairs()
    loss = torch.ones(1)
    F.preference_(x, t, w, torch.zeros(1, dtype=torch.int32), loss)
    assert float(loss) == 1.0 and float(x.abs().sum()) == 0.0


# ------------------------------------------------------------------------ 8-bit moments
def test_codes_and_exponents():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1000, generator=g) * torch.exp(4 * torch.randn(1000, generator=g))
    codes, e = R.moment_codes(x)
    assert codes.dtype == torch.float8_e4m3fn and e.tolist() == [_smallest(x[i:i + 256].abs().max().item()) for i in range(0, 1000, 256)]
    v = R.moment_values(codes, e)
    unit = torch.exp2(e.float() - 127).repeat_interleave(256)[:1000]
    assert bool(((v - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10)).all())     # half a step, normal or not
    zero, e = R.moment_codes(torch.zeros(300))
    assert e.tolist() == [0, 0] and float(R.moment_values(zero, e).abs().sum()) == 0.0
    for top in (448.0, 448.0 * (1 + 2 ** -20), 1.0, 1.75, 1.7500001, 3e38, 1e-38, 1e-45):
        assert R.moment_exponents(torch.tensor([top])).item() == _smallest(torch.tensor(top).item())


def _smallest(top):
    e = 1
    while top > 448.0 * 2.0 ** (e - 127):
        e += 1
    return e


def test_update_by_hand():
    t = (torch.tensor([1.0, -2.0]), torch.tensor([0.5, 0.0]), *F.moments8(2), 0)
    F.adamw8_many_([t], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.01, step=1)
    # first step: m / (1 - b1) = g, r / sqrt(1 - b2) = |g|: a step of lr where there is a gradient; then decay alone
    assert t[0].tolist() == pytest.approx([1.0 * 0.999 - 0.1, -2.0 * 0.999], rel=1e-6)
    assert R.moment_values(t[2], t[4]).tolist() == pytest.approx([0.05, 0.0], rel=2.0 ** -4)
    assert R.moment_values(t[3], t[5]).tolist() == pytest.approx([math.sqrt(0.05) * 0.5, 0.0], rel=2.0 ** -4)


def test_update_refuses_an_epsilon_that_single_precision_flushes():
    t = (torch.zeros(8), torch.zeros(8), *F.moments8(8), 0)
    for eps in (0.0, -1.0, 1e-20, float("nan")):
        with pytest.raises(ValueError):
            F.adamw8_many_([t], lr=0.1, eps=eps)
    F.adamw8_many_([t], lr=0.1, eps=1e-16)


def test_update_refuses():
    def lists(n=300):
        return [torch.zeros(n), torch.zeros(n), *F.moments8(n), 0]
    ok = dict(lr=0.1)
    for place, value, error in ((1, torch.zeros(299), ValueError), (2, torch.zeros(300), TypeError), (4, torch.zeros(1, dtype=torch.uint8), ValueError),
                                (5, torch.zeros(2), TypeError), (0, torch.zeros(300, dtype=torch.float64), TypeError), (6, 4, ValueError),
                                (6, -8, ValueError), (0, torch.zeros(600)[::2], ValueError), (1, torch.zeros(300, dtype=torch.float16), TypeError)):
        t = lists()
        t[place] = value
        with pytest.raises(error):
            F.adamw8_many_([tuple(t)], **ok)
    with pytest.raises(ValueError):
        F.adamw8_many_([tuple(lists())], step=0, **ok)
