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
