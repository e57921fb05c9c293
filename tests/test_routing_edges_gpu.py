"""Selection of experts on the GPU where scores, sums or rows are far from ordinary, against the definition in 64 bits."""
import pytest
import torch

from shadowspill_b200.ops import reference as R, routing

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2.0 ** -23


def _rand(*shape, seed=0, std=1.0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * std


@pytest.mark.parametrize("low,high", [(-6.0, 6.0), (-20.0, -10.0), (10.0, 20.0), (-88.0, -60.0), (-100.0, -88.0)])
def test_sigmoid_weights_are_those_of_an_exact_exponential(low, high):
    """exp(-|x|) is off by 2 steps, 1 + it and the quotient by half a step each: 3 steps of 2^-23; denormal scores by half of 2^-149 twice.
    A gradient has two scores, their product's and its own factor's rounding."""
    x = low + (high - low) * torch.rand(2000, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    ids, w, _ = routing.select_experts(x, 8, scoring="sigmoid", renormalize=False)
    c = torch.sigmoid(x.double()).gather(1, ids.long())
    assert bool(((w - c).abs() <= 3 * STEP * c + 2.0 ** -149).all())
    dw = _rand(2000, 8, seed=2)
    got = routing.select_experts_bwd(x, ids, dw, scoring="sigmoid", renormalize=False).gather(1, ids.long())
    want = dw.double() * c * torch.sigmoid(-x.double()).gather(1, ids.long())
    assert bool(((got - want).abs() <= 7 * STEP * want.abs() + 2.0 ** -147).all())
    # renormalised: a sum of eight (three levels of half a step) and another quotient
    ids, w, _ = routing.select_experts(x, 8, scoring="sigmoid", scale=1.0)
    c = c / (c.sum(1, keepdim=True) + 1e-20)
    assert bool(((w - c).abs() <= 9 * STEP * c + 2.0 ** -149 * 1e20).all())


@pytest.mark.parametrize("renormalize", [True, False])
def test_softmax_weights_far_below_the_top(renormalize):
    """Scores of experts that a bias picks: x - top is rounded by half a step of up to 100, the exponential by 2, the row's sum and
    quotients by 16; denormal ones keep steps of 2^-149."""
    x = _rand(500, 32, seed=3)
    x[:, 0] = torch.linspace(5.0, 95.0, 500, device=DEV)
    bias = torch.zeros(32, device=DEV)
    bias[8:12] = 10.0
    ids, w, _ = routing.select_experts(x, 4, bias=bias, renormalize=renormalize)
    c = torch.softmax(x.double(), 1).gather(1, ids.long())
    assert bool((ids >= 8).all()) and bool((ids < 12).all())
    score, low = (x[:, :1].double() + 5) / 2 * STEP + 18 * STEP, 2.0 ** -148
    if renormalize:
        c = c / (c.sum(1, keepdim=True) + 1e-20)
        score, low = 2 * score, low * 1e20 * 5
    assert bool(((w - c).abs() <= score * c + low).all())


@pytest.mark.parametrize("gap", [0.0, 10.0, 18.0, 21.0, 40.0, 46.0, 50.0, 60.0, 90.0])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,k", [(16, 4), (64, 1), (65, 7), (512, 10)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_softmax_picks_far_below_the_top(gap, renormalize, E, k, dtype):
    """A bias picks experts whose scores are nothing beside the row's largest, which is not picked: the sum that the weights
    are divided by is then of the size of the 1e-20 beside it, and the others have gradients too."""
    x, dw, scale = _rand(50, E, seed=E), _rand(50, k, seed=8), 2.5
    x[:, 3] = x.amax(1) + gap
    x = x.to(dtype)
    bias = torch.zeros(E, device=DEV)
    bias[4:4 + k] = 10.0
    ids, w, _ = routing.select_experts(x, k, bias=bias, renormalize=renormalize, scale=scale)
    assert torch.equal(ids.sort(1).values, torch.arange(4, 4 + k, device=DEV, dtype=torch.int32).expand(50, k))
    got = routing.select_experts_bwd(x, ids, dw, renormalize=renormalize, scale=scale)
    x64 = x.double().requires_grad_(True)
    s = torch.softmax(x64, 1)
    c = s.gather(1, ids.long())
    want_w = scale * (c / (c.sum(1, keepdim=True) + 1e-20) if renormalize else c)
    want = torch.autograd.grad(want_w, x64, dw.double())[0]
    s, c, want_w = s.detach(), c.detach(), want_w.detach()
    # A score: its argument, a difference of up to gap + 8, is rounded by half a step of that, the exponential by 2 steps, its
    # row's sum by 16 together with the quotient. A weight has one above and one below the line; a gradient three such factors.
    score = (gap + 8) / 2 * STEP + 18 * STEP
    u = c / (c.sum(1, keepdim=True) + 1e-20) if renormalize else c
    mean = (dw.double().abs() * u).sum(1, keepdim=True)
    size = torch.zeros_like(s).scatter_(1, ids.long(), scale * u * (dw.double().abs() + (mean if renormalize else 0.0)))
    inner = scale * mean * (1e-20 / (c.sum(1, keepdim=True) + 1e-20) if renormalize else 1.0)
    size = size + s * inner
    # scores under fp32's normal range keep steps of 2^-149, times 1e20 where that is all they are divided by; and 1e-20 of a sum
    # that is 4e-12 or more (a pick within 20 of the top of 512) is below the rounding of the others and may be left out
    low = 2.0 ** -149 * (1e20 if renormalize else 1.0) * scale
    assert bool(((w - want_w).abs() <= 2 * score * want_w + 2 * k * low).all())
    left = 2.5e-9 * scale * mean * s if renormalize else 0.0
    # a gradient under the normal range is a multiple of the type's smallest step, half of which its rounding and that of a product that it
    # is formed from are off by, however small dw is
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    allowed = 4 * score * size + left + torch.finfo(dtype).eps / 2 * want.abs() + 4 * k * low * dw.abs().sum(1, keepdim=True) + 2 * least
    assert bool(((got.double() - want).abs() <= allowed).all())


@pytest.mark.parametrize("E,k,groups,keep", [(48, 3, 1, 1), (48, 8, 1, 1), (48, 6, 4, 2), (60, 6, 5, 2), (256, 5, 1, 1), (512, 10, 8, 3)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_rows_with_nan_or_inf_follow_the_definition(E, k, groups, keep, bias, scoring, renormalize):
    """A softmax with a NaN or +inf has no score that compares: the first experts are picked, with weights and gradients of NaN. Rows between
    such rows, some with keys a few units in the last place apart, are what they are without them."""
    nan, inf = float("nan"), float("inf")
    x = _rand(64, E, seed=E)
    x[1::4] = x[1::4, :1] + torch.randint(-4, 5, (16, E), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) * 2.0 ** -22
    x[0, 5] = x[2, 0] = nan
    x[4] = nan
    x[6, 7], x[8, 3:6] = inf, inf
    x[10], x[10, 9] = -inf, nan
    x[12], x[12, 11] = -inf, inf
    x[14, 1], x[14, 2] = nan, inf
    x[16, :5], x[16, E - 1] = -inf, nan
    bad = [0, 2, 4, 6, 8, 10, 12, 14, 16]
    b = _rand(E, seed=4) * 0.1 if bias else None
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        ids, w, counts = routing.select_experts(y, k, scoring=scoring, bias=b, groups=groups, keep_groups=keep, renormalize=renormalize)
        want = R.select_experts(y, k, scoring, b, groups, keep, renormalize)
        assert torch.equal(ids, want[0]) and torch.equal(counts, want[2])
        assert torch.equal(torch.isnan(w), torch.isnan(want[1]))
        dw = _rand(64, k, seed=5)
        got = routing.select_experts_bwd(y, ids, dw, scoring=scoring, renormalize=renormalize)
        ref = R.select_experts_bwd(y.double(), ids, dw, scoring, renormalize)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        if scoring == "softmax":
            if bias or groups > 1:
                assert torch.equal(ids[bad], torch.arange(k, dtype=torch.int32, device=DEV).expand(9, k))
            assert bool(torch.isnan(w[bad]).all()) and bool(torch.isnan(got[bad]).all())


# relative error of a weight of 33 to 512 picks: exponentials off by 2 steps and their argument's rounding (up to 16), twice; sums of 16 terms
# to a lane and five levels, twice; two quotients
MANY = (2 * (2 + 8) + 2 * 21 + 4) * STEP


@pytest.mark.parametrize("T,E,k,groups,keep", [(1, 33, 33, 1, 1), (50, 64, 40, 1, 1), (70, 512, 512, 1, 1), (9, 96, 48, 3, 2), (2500, 256, 33, 8, 5),
                                              (30, 511, 100, 1, 1), (0, 64, 40, 1, 1)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_picks_than_a_warp_has_lanes(T, E, k, groups, keep, bias, scoring, dtype):
    x, b = (_rand(T, E, seed=T) * 1.5).to(dtype), _rand(E, seed=3) * 0.1 if bias else None
    dw = _rand(T, k, seed=8)
    for renormalize in (True, False):
        ids, w, counts = routing.select_experts(x, k, scoring=scoring, bias=b, groups=groups, keep_groups=keep, renormalize=renormalize, scale=2.5)
        want = R.select_experts(x, k, scoring, b, groups, keep, renormalize, 2.5)
        assert torch.equal(ids, want[0]) and torch.equal(counts, want[2])
        assert bool(((w - want[1]).abs() <= STEP * want[1]).all())               # rounded once, in either
        got = routing.select_experts_bwd(x, ids, dw, scoring=scoring, renormalize=renormalize, scale=2.5)
        ref = R.select_experts_bwd(x.double(), ids, dw, scoring, renormalize, 2.5)
        s = R.expert_scores(x.double(), scoring)
        total = s.gather(1, ids.long()).sum(1, keepdim=True) if renormalize else 1.0
        most = 2.5 * dw.abs().amax(1, keepdim=True)                            # of the terms that may cancel
        size = most * s / total * (2 if renormalize else 1) + (0 if scoring == "sigmoid" else most * s / total)
        assert bool(((got - ref).abs() <= 2 * MANY * size + torch.finfo(dtype).eps / 2 * ref.abs()).all())


def test_many_picks_of_ties_masks_and_bad_rows():
    nan, inf = float("nan"), float("inf")
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randint(-2, 3, (64, 80), generator=g, device=DEV).float() * 0.5
    x[0], x[1, 3:], x[2, 5], x[3, 7], x[4] = -inf, -inf, nan, inf, nan
    for b in (None, torch.zeros(80, device=DEV)):
        for scoring in ("softmax", "sigmoid"):
            ids, w, counts = routing.select_experts(x, 50, scoring=scoring, bias=b)
            want = R.select_experts(x, 50, scoring, b)
            assert torch.equal(ids, want[0]) and torch.equal(counts, want[2]) and torch.equal(torch.isnan(w), torch.isnan(want[1]))
            got = routing.select_experts_bwd(x, ids, w.nan_to_num(), scoring=scoring)
            ref = R.select_experts_bwd(x.double(), ids, w.nan_to_num(), scoring)
            assert torch.equal(torch.isnan(got), torch.isnan(ref))


def test_many_picks_captured_and_on_another_stream():
    x, dw = _rand(600, 64, seed=1), _rand(600, 40, seed=2)
    routing.select_experts(x, 40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, w, counts = routing.select_experts(x, 40, scoring="sigmoid")
        grad = routing.select_experts_bwd(x, ids, dw, scoring="sigmoid")
    x.copy_(_rand(600, 64, seed=11))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = routing.select_experts(x, 40, scoring="sigmoid")
        want_grad = routing.select_experts_bwd(x, want[0], dw, scoring="sigmoid")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((ids, w, counts, grad), (*want, want_grad)))


def test_a_layer_of_more_picks_than_lanes():
    """Picks into the experts' products, forward and backward, against the tensor-operation form."""
    import shadowspill_b200.frontend.ops as ops
    T, D, Fw, E, k = 64, 128, 128, 48, 40
    h, w13, w2 = _rand(T, D, seed=1).bfloat16(), (_rand(E, 2 * Fw, D, seed=2) * 0.1).bfloat16(), (_rand(E, D, Fw, seed=3) * 0.1).bfloat16()
    logits, bias = _rand(T, E, seed=4), _rand(E, seed=5) * 0.1
    ids, w = torch.ops.ss.select_experts(logits, bias, k, True, 1, 1, True, 2.5)
    out, up = torch.ops.ss.moe_experts_routed(h, ids, w, w13, w2), _rand(T, D, seed=6).bfloat16()
    grads = torch.ops.ss.moe_experts_routed_bwd(h, ids, w, w13, w2, up, True)        # as exported stages call it
    ref = [t.double().requires_grad_(True) for t in (h, w, w13, w2)]
    want = ops._moe_routed_torch(ref[0], ids, *ref[1:])
    want.backward(up.double())
    # activations, products and their gradients are stored in bf16, four of them in a chain, each off by 2^-8 of its value
    for got, exact in ((out, want), *((a, b.grad) for a, b in zip(grads, ref))):
        assert float((got.double() - exact.detach()).norm()) <= 4 * 2.0 ** -8 * float(exact.detach().norm())


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (700, 3, 512), (8192, 8, 64), (0, 4, 8), (33, 40, 48)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint8])
def test_picks_made_elsewhere_are_counted(T, k, E, dtype):
    from shadowspill_b200.ops import _lib, moe
    ids = torch.randint(0, min(E, 256), (T, k), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    picks, counts = moe.counted(ids, E)
    assert torch.equal(picks, ids.int()) and torch.equal(counts.long(), torch.bincount(ids.reshape(-1).long(), minlength=E))
    _lib.check_status()


@pytest.mark.parametrize("bad", [-1, 8, 513, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_a_pick_of_no_expert_is_reported(bad, dtype):
    import shadowspill_b200.frontend.ops  # noqa: F401
    from shadowspill_b200.ops import _lib
    T, D, Fw, E, k = 40, 128, 128, 8, 2
    h, w13, w2 = _rand(T, D, seed=1).bfloat16(), (_rand(E, 2 * Fw, D, seed=2) * 0.1).bfloat16(), (_rand(E, D, Fw, seed=3) * 0.1).bfloat16()
    ids = torch.randint(0, E, (T, k), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(dtype)
    w = torch.rand(T, k, device=DEV)
    want = torch.ops.ss.moe_experts_routed(h, ids, w, w13, w2)
    _lib.check_status()
    wrong = ids.clone()
    wrong[3, 1] = bad
    torch.ops.ss.moe_experts_routed(h, wrong, w, w13, w2)
    with pytest.raises(RuntimeError, match="bad argument"):
        _lib.check_status()
    assert torch.equal(torch.ops.ss.moe_experts_routed(h, ids, w, w13, w2), want)
    _lib.check_status()


# lanes to a token and experts to a lane by the launcher's rule: 16 and 16 by logits alone and with a bias, 32 and 4, 32 and 8
@pytest.mark.parametrize("E,k,bias,groups,keep", [(256, 8, False, 1, 1), (129, 8, False, 1, 1), (200, 1, False, 1, 1), (256, 5, True, 1, 1),
                                                  (131, 3, True, 1, 1), (256, 2, True, 8, 8), (128, 9, False, 1, 1), (66, 32, False, 1, 1),
                                                  (256, 9, False, 1, 1), (129, 32, False, 1, 1), (240, 20, False, 1, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_picks_of_every_kernel(E, k, bias, groups, keep, scoring, dtype):
    g = torch.Generator(device=DEV).manual_seed(E + k)
    rough = torch.randint(-3, 4, (300, E), generator=g, device=DEV).float() * 0.5           # ties
    near = _rand(300, 1, seed=1) + torch.randint(-4, 5, (300, E), generator=g, device=DEV) * 2.0 ** -22
    b = _rand(E, seed=3) * 0.1 if bias else None
    for x in (_rand(1003, E, seed=2) * 1.5, rough, near):
        x = x.to(dtype)
        for renormalize in (True, False):
            ids, w, counts = routing.select_experts(x, k, scoring=scoring, bias=b, groups=groups, keep_groups=keep, renormalize=renormalize)
            want = R.select_experts(x, k, scoring, b, groups, keep, renormalize)
            assert torch.equal(ids, want[0]) and torch.equal(counts, want[2])
            # as in the tests of softmax and sigmoid weights, arguments up to 16; sums of up to 32 renormalised
            assert bool(((w - want[1]).abs() <= 2 * (8 + 18) * STEP * want[1]).all())


def test_an_eager_backward_pass_that_would_wait_for_itself_is_refused():
    import shadowspill_b200.frontend.ops  # noqa: F401
    T, D, Fw, E, k = 16, 128, 128, 8, 2
    h, w13, w2 = _rand(T, D, seed=1).bfloat16(), (_rand(E, 2 * Fw, D, seed=2) * 0.1).bfloat16(), (_rand(E, D, Fw, seed=3) * 0.1).bfloat16()
    ids, w = torch.ops.ss.select_experts(_rand(T, E, seed=4), _rand(E, seed=5), k, True, 1, 1, True, 1.0)
    for leaf in (h, w, w13):
        leaf.requires_grad_(True)
    out = torch.ops.ss.moe_experts_routed(h, ids, w, w13, w2)
    with pytest.raises(RuntimeError, match="exported stages"):
        out.sum().backward()
    with torch.autograd.set_multithreading_enabled(False):       # in the caller's thread: the helper has the device's to itself
        torch.ops.ss.moe_experts_routed(h, ids, w, w13, w2).sum().backward()
    assert bool(torch.isfinite(h.grad).all()) and float(h.grad.abs().max()) > 0
    assert len(torch.ops.ss.moe_experts_routed_bwd(h.detach(), ids, w.detach(), w13.detach(), w2, torch.ones_like(h), True)) == 4
