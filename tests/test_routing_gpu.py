"""Selection of experts on the GPU: the picks of keys in 64 bits, weights and gradients against the definition."""
import pytest
import torch

from shadowspill_b200.ops import reference as R, routing

pytestmark = pytest.mark.gpu
DEV = "cuda"
# relative error of a weight: __expf of an argument up to 16 has at most 2 + 1.173 * 16 = 21 steps of 2^-23, numerator and
# denominator each; two quotients of 2 and a sum of up to 32 terms (5 levels) of 1, rounded up
TOL = (2 * 21 + 12) * 2.0 ** -23


def _logits(T, E, dtype=torch.float32, seed=0, std=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(T, E, generator=g, device=DEV) * std).to(dtype)


def _compare(x, k, **kw):
    got = routing.select_experts(x, k, **kw)
    kw2 = {**dict(scoring="softmax", bias=None, groups=1, keep_groups=1, renormalize=True, scale=1.0), **kw}
    want = R.select_experts(x, k, kw2["scoring"], kw2["bias"], kw2["groups"], kw2["keep_groups"], kw2["renormalize"], kw2["scale"])
    assert got[0].dtype == got[2].dtype == torch.int32 and got[1].dtype == torch.float32
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[2], want[2])
    assert bool(((got[1] - want[1]).abs() <= TOL * want[1].abs() + 1e-37).all())
    return got


SHAPES = [(1, 8, 2, 1, 1), (7, 64, 8, 1, 1), (33, 65, 5, 1, 1), (1000, 256, 8, 8, 4), (130, 512, 32, 1, 1), (257, 512, 10, 8, 3),
          (64, 96, 7, 3, 2), (50, 40, 16, 5, 4), (9, 1, 1, 1, 1), (77, 32, 4, 32, 9), (20, 12, 12, 2, 2), (3001, 128, 8, 1, 1)]


@pytest.mark.parametrize("T,E,k,groups,keep", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_picks_weights_and_counts(T, E, k, groups, keep, scoring, bias, dtype):
    x = _logits(T, E, dtype, seed=T + E)
    b = _logits(1, E, seed=3)[0] * 0.1 if bias else None
    for renormalize in (True, False):
        _compare(x, k, scoring=scoring, bias=b, groups=groups, keep_groups=keep, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
@pytest.mark.parametrize("bias", [None, "zero", "coarse"])
def test_ties_go_to_the_lowest_index(scoring, groups, keep, bias):
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randint(-2, 3, (300, 64), generator=g, device=DEV).float() * 0.5     # few values: most picks tie
    x[0] = 0.0                                                                     # all of them
    x[1] = torch.where(torch.arange(64, device=DEV) % 2 == 0, 0.0, -0.0)           # equal under either sign
    b = {None: None, "zero": torch.zeros(64, device=DEV),
         "coarse": torch.randint(0, 2, (64,), generator=g, device=DEV).float() * 0.25}[bias]
    _compare(x, 8, scoring=scoring, bias=b, groups=groups, keep_groups=keep)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3)])
def test_keys_closer_than_single_precision_resolves(scoring, groups, keep):
    """Neighbouring experts' logits and biases differ by a few units in the last place: the order is that of 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(500, 1, generator=g, device=DEV) + torch.randint(-4, 5, (500, 128), generator=g, device=DEV) * 2.0 ** -22
    b = 0.1 + torch.randint(-4, 5, (128,), generator=g, device=DEV) * 2.0 ** -24
    _compare(x, 8, scoring=scoring, bias=b, groups=groups, keep_groups=keep)
    _compare(x * 1e-3, 8, scoring=scoring, bias=b, groups=groups, keep_groups=keep)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_masked_experts_come_last(scoring, bias, groups, keep):
    inf, low = float("-inf"), torch.finfo(torch.float32).min
    x = _logits(40, 32, seed=1)
    x[0, :] = inf                              # nothing is left
    x[1, 3:] = inf                             # fewer than k are
    x[2, :] = low
    x[3, ::2] = low
    x[4, 1:] = inf
    x[5, 5] = 300.0
    b = _logits(1, 32, seed=2)[0] * 0.1 if bias else None
    if bias:
        b[7] = inf                             # an expert that is never picked
    ids, w, _ = _compare(x, 6, scoring=scoring, bias=b, groups=groups, keep_groups=keep)
    assert bool(torch.isfinite(w).all())
    assert bool((ids.sort(1).values.diff(dim=1) > 0).all())
    if scoring == "softmax":
        assert float(w[0].abs().sum()) == 0.0
    d = torch.ones_like(w)
    grad = routing.select_experts_bwd(x, ids, d, scoring=scoring)
    assert bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_bad_logits_leave_different_experts_in_range(value, scoring, bias):
    x = _logits(30, 48, seed=4)
    x[::3, 5] = value
    x[1] = value
    b = torch.zeros(48, device=DEV) if bias else None
    for groups, keep in ((1, 1), (4, 2)):
        ids, w, counts = routing.select_experts(x, 8, scoring=scoring, bias=b, groups=groups, keep_groups=keep)
        assert int(ids.min()) >= 0 and int(ids.max()) < 48 and int(counts.sum()) == 240
        assert bool((ids.sort(1).values.diff(dim=1) > 0).all())
        bad = torch.zeros(30, dtype=torch.bool, device=DEV)
        bad[::3] = True
        bad[1] = True
        assert bool(torch.isfinite(w[~bad]).all())
        if scoring == "softmax":
            assert bool(torch.isnan(w[bad]).all())


@pytest.mark.parametrize("E,k", [(16, 4), (64, 8), (512, 10)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_biases_of_any_value(E, k, scoring):
    """Experts forced in or out by a bias without end, one that is no number, and ones beside which scores vanish."""
    x = _logits(300, E, seed=E)
    for values in ((float("inf"),) * 3, (float("inf"),) * (k + 2), (float("nan"), float("-inf")), (3e38, 3e38, -3e38), (1e6,) * k,
                   (float("inf"), float("nan"), 3e38, float("-inf"), 1e6)):
        b = torch.zeros(E, device=DEV)
        b[torch.randperm(E, generator=torch.Generator().manual_seed(k))[:len(values)].to(DEV)] = torch.tensor(values, device=DEV)
        ids, _, _ = _compare(x, k, scoring=scoring, bias=b)
        assert bool((ids.sort(1).values.diff(dim=1) > 0).all())


@pytest.mark.parametrize("E,groups", [(64, 8), (512, 8), (96, 3), (40, 5)])
def test_group_sums_past_single_precision(E, groups):
    """Two keys of a group add up to more than fp32 holds: the groups are told apart in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(E)
    x = _logits(100, E, seed=3)
    b = (1.55 + 0.3 * torch.rand(E, generator=g, device=DEV)) * 1e38
    b[torch.rand(E, generator=g, device=DEV) < 0.3] *= -1.0
    _compare(x, 6, scoring="sigmoid", bias=b, groups=groups, keep_groups=2)
    _compare(x, 6, scoring="sigmoid", bias=-b.abs(), groups=groups, keep_groups=2)


@pytest.mark.parametrize("E,groups", [(16, 8), (64, 8), (96, 3)])
def test_a_group_with_an_expert_forced_in_and_the_rest_forced_out(E, groups):
    """inf - inf is no sum: such a group comes last, with those of -inf."""
    x = _logits(50, E, seed=E)
    b = torch.zeros(E, device=DEV)
    b[:E // groups] = float("-inf")
    b[1] = float("inf")
    b[-1] = float("inf")
    for keep in (1, 2, groups):
        _compare(x, 2, scoring="sigmoid", bias=b, groups=groups, keep_groups=keep)


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (100, 64, 8), (33, 65, 5), (515, 256, 8), (20, 512, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients(T, E, k, scoring, renormalize, dtype):
    x, dw = _logits(T, E, dtype, seed=T), _logits(T, k, seed=8)
    ids, _, _ = routing.select_experts(x, k, scoring=scoring, renormalize=renormalize, scale=2.5)
    got = routing.select_experts_bwd(x, ids, dw, scoring=scoring, renormalize=renormalize, scale=2.5)
    assert got.dtype == dtype and got.is_contiguous()
    want = R.select_experts_bwd(x.double(), ids, dw, scoring, renormalize, 2.5)
    s = R.expert_scores(x.double(), scoring)
    total = s.gather(1, ids.long()).sum(1, keepdim=True) if renormalize else 1.0
    size = 2.5 * dw.abs().sum(1, keepdim=True) * s / total                    # of the terms that may cancel
    half = torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= 4 * TOL * size + half * want.abs() + 1e-37).all())


def test_strided_rows_empty_batches_and_other_streams():
    wide = _logits(200, 100, seed=6)
    for x in (wide[:, 3:67], wide[::2, :64], wide.t().contiguous().t()[:, :64], wide[:1].expand(9, 100)[:, :64]):
        ids, w, counts = _compare(x, 4, scoring="sigmoid", bias=torch.zeros(64, device=DEV))
        grad = routing.select_experts_bwd(x, ids, torch.ones_like(w), scoring="sigmoid")
        assert torch.equal(grad, routing.select_experts_bwd(x.contiguous(), ids, torch.ones_like(w), scoring="sigmoid"))
    ids, w, counts = routing.select_experts(wide[:0], 4)
    assert ids.shape == w.shape == (0, 4) and float(counts.abs().sum()) == 0
    assert routing.select_experts_bwd(wide[:0], ids, w).shape == (0, 100)
    want = routing.select_experts(wide, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = routing.select_experts(wide, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed_on_new_logits():
    x = _logits(600, 64, seed=1)
    dw = _logits(600, 4, seed=2)
    graph = torch.cuda.CUDAGraph()
    routing.select_experts(x, 4)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ids, w, counts = routing.select_experts(x, 4, renormalize=False)
        grad = routing.select_experts_bwd(x, ids, dw, renormalize=False)
    for seed in (11, 12):
        x.copy_(_logits(600, 64, seed=seed))
        graph.replay()
        want = routing.select_experts(x, 4, renormalize=False)
        assert torch.equal(ids, want[0]) and torch.equal(w, want[1]) and torch.equal(counts, want[2])
        assert torch.equal(grad, routing.select_experts_bwd(x, want[0], dw, renormalize=False))
