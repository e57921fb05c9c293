"""AdamW with 8-bit moments on the GPU: the bits of its definition where everything is rounded to nearest, unbiased and
repeatable where not."""
import pytest
import torch

from shadowspill_b200.ops import functional as F, reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3, grad_scale=0.5)
NEAREST = dict(stochastic_param=False, stochastic_state=False)
EDGES = [1, 7, 8, 9, 255, 256, 257, 2047, 2048, 2049, 4096, 100003]


def _tensor(n, seed, dtype=torch.bfloat16, g_dtype=torch.bfloat16, offset=0, warm=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda s: torch.randn(n, generator=g, device=DEV) * s
    size = torch.exp(r(2.0) - 5.0)                        # magnitudes over six decades
    p, grad = r(0.1).to(dtype), (r(1.0) * size).to(g_dtype)
    state = F.moments8(n, DEV)
    if warm and n:
        for codes, exps, x, floor in ((state[0], state[2], r(1.0) * size, False), (state[1], state[3], r(1.0).abs() * size, True)):
            c, e = R.moment_codes(x, floor)
            codes.copy_(c)
            exps.copy_(e)
    return (p, grad, *state, offset)


def _copy(t):
    return tuple(x.clone() if isinstance(x, torch.Tensor) else x for x in t)


def _bits(t):
    return [x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x for x in t if isinstance(x, torch.Tensor)]


def _same_moments(a, b):
    return all(torch.equal(x, y) for x, y in zip(_bits(a)[2:], _bits(b)[2:]))


def _against_definition(tensors, **hyper):
    h = {**HYPER, **hyper}
    want = [_copy(t) for t in tensors]
    F.adamw8_many_(tensors, **h, **NEAREST)
    for got, ref in zip(tensors, want):
        p32 = ref[0].float().clone()
        R.adamw8_(p32, *ref[1:6], **h)
        assert _same_moments(got, (p32, *ref[1:]))
        # the step in fp32: a quotient of 2 steps (of 2^-23) and six roundings, on p' and the step's own size
        step = (p32 - ref[0].float()).abs()
        half = torch.finfo(got[0].dtype).eps / 2 if got[0].dtype == torch.bfloat16 else 0.0
        assert bool(((got[0].float() - p32).abs() <= half * p32.abs() + 2.0 ** -22 * (p32.abs() + 6 * step) + 1e-37).all())


@pytest.mark.parametrize("p_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("g_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes", [EDGES, [257] * 47, [65] * 48, [513] * 49, [4100] * 97, [0, 5, 0, 24], [0], [], [1_000_003, 3]],
                         ids=["edges", "47", "48", "49", "97", "empty", "one empty", "none", "large"])
def test_moments_have_the_bits_of_the_definition(sizes, p_dtype, g_dtype):
    _against_definition([_tensor(n, i, p_dtype, g_dtype) for i, n in enumerate(sizes)])


@pytest.mark.parametrize("hyper", [dict(step=1), dict(step=100_000), dict(beta1=0.0, beta2=0.0), dict(beta2=0.999, grad_scale=1.0),
                                   dict(weight_decay=0.0, lr=1e-5)])
def test_settings_and_a_first_step(hyper):
    _against_definition([_tensor(3001, 1, warm=False), _tensor(700, 2)], **hyper)


def test_special_values():
    t = _tensor(256 * 8, 5, torch.float32, torch.float32)
    grad = t[1]
    grad[:256] = 0.0                                      # a block without gradients
    for x in t[2:4]:
        x[:256].view(torch.uint8).zero_()
    grad[256:512] = 1e-30
    grad[512:768] = 1e30
    grad[768] = 3e38
    grad[769:1024] = 1e-38
    grad[1024:1280] = 448.0 * 2.0 ** -12                  # on the border of two exponents, and next to it
    grad[1280:1536] = 448.0 * 2.0 ** -12 * (1 + 2.0 ** -20)
    for h in (dict(), dict(beta1=0.0, beta2=0.0, grad_scale=1.0)):
        _against_definition([_copy(t)], **h)
    bad = _tensor(600, 6)
    bad[1][3], bad[1][300] = float("nan"), float("inf")
    F.adamw8_many_([bad], **HYPER, **NEAREST)
    m, r = R.moment_values(bad[2], bad[4]), R.moment_values(bad[3], bad[5])
    assert bool(torch.isnan(m[3])) and bool(torch.isnan(r[3])) and bool(torch.isinf(m[300])) and bool(torch.isnan(bad[0][3]))
    keep = torch.arange(600, device=DEV)
    assert bool(torch.isfinite(m[(keep != 3) & (keep // 256 != 1)]).all())   # a NaN stays with its element


def test_a_root_that_is_not_zero_keeps_a_code():
    t = _tensor(256, 7, torch.float32, torch.float32, warm=False)
    t[1].copy_(torch.cat([torch.full((1,), 1e6, device=DEV), torch.full((255,), 1e-6, device=DEV)]))
    for sr in (False, True):
        u = _copy(t)
        F.adamw8_many_([u], **HYPER, stochastic_param=False, stochastic_state=sr)
        assert int((u[3].view(torch.uint8) == 0).sum()) == 0


@pytest.mark.parametrize("shift", [1, 4])
def test_unaligned_views(shift):
    whole = _tensor(5000 + shift, 8)
    view = tuple(x[shift:].clone()[:5000] for x in whole[:4])
    padded = [torch.empty(5000 + shift, dtype=x.dtype, device=DEV)[shift:] for x in whole[:4]]
    for a, b in zip(padded, view):
        a.copy_(b)
    exps = [x[:20].clone() for x in whole[4:6]]
    a = (*padded, *[e.clone() for e in exps], 0)
    b = (*view, *[e.clone() for e in exps], 0)
    for sr in (False, True):
        F.adamw8_many_([a], **HYPER, stochastic_param=sr, stochastic_state=sr, seed=4)
        F.adamw8_many_([b], **HYPER, stochastic_param=sr, stochastic_state=sr, seed=4)
        assert all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))


def test_stochastic_rounding_is_unbiased_and_between_the_neighbours():
    n = 256 * 4096
    p, grad, m, r, m_exp, r_exp, _ = _tensor(n, 9, warm=False)
    g = torch.Generator(device=DEV).manual_seed(3)
    grad.copy_(torch.rand(n, generator=g, device=DEV) + 0.5)
    p.fill_(1.0)
    exact = [p.float().clone(), grad, *F.moments8(n, DEV), 0]
    F.adamw8_many_([(p, grad, m, r, m_exp, r_exp, 0)], **HYPER, seed=11)
    gf = grad.float() * 0.5
    first, root = 0.1 * gf, (0.05 * gf * gf).sqrt()
    R.adamw8_(*exact[:6], **HYPER)
    for codes, exps, x in ((m, m_exp, first), (r, r_exp, root)):
        v = R.moment_values(codes, exps)
        step = torch.exp2(torch.floor(torch.log2(x)) - 3)                # of e4m3's three stored bits
        assert bool(((v - x).abs() <= step * (1 + 2.0 ** -10)).all())
        lower = (x / step).floor() * step
        assert bool(((v == lower) | ((v - lower - step).abs() <= step * 2.0 ** -10)).all())
        # the mean error in steps: deviation at most 1/2 each; eight random bits move a mean by at most 2^-8
        assert abs(float(((v - x) / step).double().mean())) <= 5 * 0.5 / n ** 0.5 + 2.0 ** -8
    err = (p.float() - exact[0]).double()
    ulp = torch.where(exact[0] < 1, 2.0 ** -8, 2.0 ** -7)                # bf16 around 1
    assert bool((err.abs() <= ulp * 1.01).all()) and abs(float((err / ulp).mean())) <= 5 * 0.5 / n ** 0.5 + 2.0 ** -15


def test_random_bits_go_by_seed_step_and_global_element():
    def run(cuts, seed=5, **h):
        t = _tensor(256 * 40, 10)
        parts = []
        for a, b in zip(cuts[:-1], cuts[1:]):
            parts.append((t[0][a:b], t[1][a:b], t[2][a:b], t[3][a:b], t[4][a // 256:-(-b // 256)], t[5][a // 256:-(-b // 256)], a))
        F.adamw8_many_(parts, **{**HYPER, **h}, seed=seed)
        return _bits(t)
    whole = run([0, 10240])
    assert all(torch.equal(a, b) for a, b in zip(whole, run([0, 10240])))
    assert all(torch.equal(a, b) for a, b in zip(whole, run([0, 256, 5120, 10240])))
    assert not torch.equal(whole[2], run([0, 10240], seed=6)[2])
    m, r = whole[2].float(), whole[3].float()
    assert not torch.equal(whole[0], run([0, 10240], seed=6)[0])


def test_a_parameter_listed_twice_is_updated_twice():
    def lists():
        a = [_tensor(n, i) for i, n in enumerate([300, 40, 9])]
        return a, [a[0], a[1], a[0], a[2], a[0]]
    one, order = lists()
    for t in order:
        F.adamw8_many_([t], **HYPER)
    many, order = lists()
    F.adamw8_many_(order, **HYPER)
    for a, b in zip(one, many):
        assert all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))


def test_mixed_types_share_a_call():
    kinds = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)]
    _against_definition([_tensor(900 + i, i, *kinds[i % 4]) for i in range(9)])


def test_other_stream_and_replayed_graph():
    a, b = _tensor(5000, 1), _tensor(5000, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.adamw8_many_([a], **HYPER, seed=2)
    torch.cuda.current_stream().wait_stream(side)
    F.adamw8_many_([b], **HYPER, seed=2)
    assert all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.adamw8_many_([a], **HYPER, seed=2)
    for _ in range(2):
        graph.replay()
        F.adamw8_many_([b], **HYPER, seed=2)
    assert all(torch.equal(x, y) for x, y in zip(_bits(a), _bits(b)))


def test_a_long_run_follows_adamw_with_fp32_moments():
    """200 noisy steps towards a target: with stochastic rounding the distance left is that of unrounded moments, within
    the noise that a code's step (2^-3 of a moment at most) puts on each of the last steps."""
    n = 4096
    g = torch.Generator(device=DEV).manual_seed(1)
    target = torch.randn(n, generator=g, device=DEV)
    p8, p32 = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    m32, v32, state = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), F.moments8(n, DEV)
    h = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    for step in range(1, 201):
        noise = 0.3 * torch.randn(n, generator=g, device=DEV)
        F.adamw8_many_([(p8, p8 - target + noise, *state, 0)], step=step, seed=3, **h)
        F.adamw_(p32, p32 - target + noise, m32, v32, step=step, **h)
    # an Adam step is at most lr / sqrt(1 - beta2) = 0.09 an element; a window of 1 / (1 - beta1) = 10 steps, each off by at most 2^-3
    # of its size in the numerator and 2^-3 in the denominator, moves an element by at most 10 * 0.25 * 0.09 = 0.23
    assert float((p8 - p32).abs().max()) <= 0.23 + float((p32 - target).abs().max())
    assert float((p8 - target).square().mean().sqrt()) <= float((p32 - target).square().mean().sqrt()) + 0.23
