"""Preference loss and 8-bit AdamW on the GPU: launches, types and sizes that choose their paths."""
import pytest
import torch

from shadowspill_b200.ops import _lib, functional as F, reference as R, routing

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3, grad_scale=0.5)
NEAREST = dict(stochastic_param=False, stochastic_state=False)


class _Refuses:
    """Stands in for the native module: every call goes on in Python."""

    def launched(self):
        return {}

    def __getattr__(self, name):
        return lambda *a: NotImplemented


def _shifted(x, shift):
    """A copy of a flat tensor that starts ``shift`` elements into an allocation."""
    out = torch.zeros(x.numel() + shift, dtype=x.dtype, device=x.device)[shift:]
    out.view(torch.uint8).copy_(x.view(torch.uint8)) if x.element_size() == 1 else out.copy_(x)
    return out


def _tensor(n, seed, dtype=torch.bfloat16, g_dtype=torch.bfloat16, shift=0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda: torch.randn(n, generator=g, device=DEV)
    size = torch.exp(2.0 * r() - 5.0)
    (m, m_exp), (root, r_exp) = R.moment_codes(r() * size), R.moment_codes(r().abs() * size, True)
    return (*(_shifted(x, shift) for x in ((r() * 0.1).to(dtype), (r() * size).to(g_dtype), m, root)), m_exp, r_exp, offset)


def _launched(entry, call):
    before = _lib.launch_counts().get(entry, 0)
    call()
    return _lib.launch_counts().get(entry, 0) - before


@pytest.mark.parametrize("native", [True, False])
def test_launches_are_counted_as_they_are_made(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_host", _Refuses())
    def update(tensors):
        return _launched("ss_adamw8_many", lambda: F.adamw8_many_(tensors, **HYPER))
    assert [update([_tensor(40, i) for i in range(n)]) for n in (1, 48, 49, 97)] == [1, 1, 2, 3]
    assert update([_tensor(40, i, shift=i % 2) for i in range(10)]) == 2            # those off their boundaries go by themselves
    assert update([_tensor(40, i, shift=1) for i in range(49)]) == 2
    assert update([_tensor(0, 1)]) == 0
    x = torch.randn(6, 16, device=DEV)
    ids, w, _ = routing.select_experts(x, 2)
    for rows, n in ((6, 1), (0, 0)):
        assert _launched("ss_select_experts_bwd", lambda: routing.select_experts_bwd(x[:rows], ids[:rows], w[:rows])) == n
    loss, targets = torch.zeros(1, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV)
    name = "ss_preference with its gradient"
    assert _launched(name, lambda: F.preference_(x.clone(), targets, None, cu, loss)) == 2
    assert _launched(name, lambda: F.preference_(x[:0], targets[:0], None, cu[:1], loss)) == 1


def _against_definition(tensors, **hyper):
    want = [tuple(x.clone() if isinstance(x, torch.Tensor) else x for x in t) for t in tensors]
    F.adamw8_many_(tensors, **{**HYPER, **hyper}, **NEAREST)
    for got, ref in zip(tensors, want):
        p32 = ref[0].float().clone()
        R.adamw8_(p32, *ref[1:6], **{**HYPER, **hyper})
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[2:6], ref[2:6]))
        # the step in fp32: a quotient of 2 steps (of 2^-23) and six roundings, on p' and the step's own size
        step = (p32 - ref[0].float()).abs()
        half = 2.0 ** -8 if got[0].dtype == torch.bfloat16 else 0.0
        assert bool(((got[0].float() - p32).abs() <= half * p32.abs() + 2.0 ** -22 * (p32.abs() + 6 * step) + 1e-37).all())


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float32)]


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "bf16 by fp32", "fp32 by bf16", "fp32"])
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_tensors_off_their_boundaries_of_every_type(types, shift):
    sizes = [1, 7, 255, 256, 257, 2048, 2049, 40_003]
    _against_definition([_tensor(n, i, *types, shift=shift) for i, n in enumerate(sizes)])
    for sr in ((True, True), (True, False), (False, True)):
        on, off = ([_tensor(n, 40 + i, *types, shift=s, offset=8 * i) for i, n in enumerate(sizes)] for s in (0, shift))
        for tensors in (on, off):
            F.adamw8_many_(tensors, **HYPER, seed=4, stochastic_param=sr[0], stochastic_state=sr[1])
        for a, b in zip(on, off):
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[2:6], b[2:6])) and torch.equal(a[0], b[0])


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "bf16 by fp32", "fp32 by bf16", "fp32"])
def test_a_hundred_tensors_on_and_off_their_boundaries(types):
    _against_definition([_tensor(200 + 77 * i, i, *types, shift=i % 3) for i in range(100)])
    mixed = [_tensor(500 + i, i, *TYPES[i % 4], shift=i // 4 % 2) for i in range(110)]
    _against_definition(mixed)


def test_a_step_moves_parameters_as_the_definition_does():
    """Routing, experts, head, preference loss and update: the four updated matrices against the definition on the step's own gradients."""
    from test_tuning_step_gpu import _step
    T, D, E, Fw, V = 256, 128, 8, 128, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).bfloat16()
    names = ("router", "w13", "w2", "head")
    params = [r(E, D, std=0.2), r(E, 2 * Fw, D, std=0.1), r(E, D, Fw, std=0.1), r(V, D, std=0.1)]
    x, targets = r(T, D), torch.randint(0, V, (T,), generator=g, device=DEV)
    weights, ref = (torch.rand(T, generator=g, device=DEV) < 0.7).float(), torch.randn(T, generator=g, device=DEV) * 0.1 - 7.0
    cu = torch.tensor([0, 60, 128, 190, 250], dtype=torch.int32, device=DEV)
    state = {n: F.moments8(p.numel(), DEV) for n, p in zip(names, params)}
    state["bias"] = torch.randn(E, generator=g, device=DEV) * 0.05
    for step in (1, 2):
        before = [p.float().reshape(-1) for p in params]
        moments = {n: [t.clone() for t in state[n]] for n in names}
        _, grads = _step(*params, state, x, targets, weights, cu, ref, step, True)
        for n, p, old in zip(names, params, before):
            want = old.clone()
            R.adamw8_(want, grads[n].reshape(-1), *moments[n], lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=step)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state[n], moments[n]))
            # stored in bf16, half a step of 2^-7; the step itself (1e-3 and less) within 2^-20 of its size
            assert bool(((p.float().reshape(-1) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * ((want - old).abs() + want.abs())).all())
            assert float((want - old).abs().mean()) > 1e-4


def test_a_long_run_stays_by_adamw_with_fp32_moments():
    """200 noisy steps towards a target, the same noise for both. A code is off by a deviation of at most half its step, 2^-4 of its value; the
    first moment keeps what 1 / (1 - 0.9^2) = 5.3 such roundings add up to in square (0.14 of its value), the root 1 / (1 - 0.95^2) = 10.3
    (0.2), so a step's error is 0.25 of it in the root mean square, alike over some 20 steps. Steps are lr = 0.02 and less; the target
    draws parameters back over r / lr = 25 steps where the noise of 0.3 and the distance make roots of about 0.5. A walk of such errors
    held by that has a deviation of 0.02 * 0.25 * sqrt(2 * 20 * 25) = 0.16."""
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
    assert float((p8 - p32).square().mean().sqrt()) <= 0.16


# rows and words that the rows kernel takes with teams of 256 and of 512 threads (by the places on the GPU and the pieces to a thread)
@pytest.mark.parametrize("rows,V", [(600, 8192), (445, 8201), (740, 9000), (300, 16384), (444, 17000), (100, 50257)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["sigmoid", "ipo"])
def test_preference_teams_of_more_than_a_warp(rows, V, dtype, kind):
    from test_preference_gpu import _case, _compare
    cuts = [0, rows // 5, rows // 2, rows // 2, rows // 2 + 1, rows - 40, rows - 3]
    x, t, w, cu, ref = _case(V, cuts, rows, dtype, seed=rows + V)
    _compare(x, t, w, cu, ref_logp=ref, kind=kind, average=kind == "ipo", beta=0.2)


def test_preference_of_two_million_logits_captured():
    """Its counters are cleared by a kernel: captured, replayed on other data, and twice in one graph."""
    from test_preference_gpu import _case
    x, t, w, cu, ref = _case(4096, [0, 200, 430, 500, 590], 600, seed=20)
    loss, grad, sums = torch.zeros(1, device=DEV), torch.empty_like(x), torch.empty(4, device=DEV)
    again = torch.zeros(1, device=DEV)
    F.preference_(x, t, w, cu, loss, grad=grad, sums=sums, ref_logp=ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss.zero_()
        again.zero_()
        F.preference_(x, t, w, cu, loss, grad=grad, sums=sums, ref_logp=ref)
        F.preference_(x, t, w, cu, again, write_grad=False, ref_logp=ref)
    for seed, bounds in ((21, [0, 200, 430, 500, 590]), (22, [0, 1, 300, 301, 600]), (23, [10, 10, 10, 300, 550])):
        new = _case(4096, bounds, 600, seed=seed)
        for a, b in zip((x, t, w, cu, ref), new):
            a.copy_(b)
        graph.replay()
        want, want_grad, want_sums = torch.zeros(1, device=DEV), torch.empty_like(x), torch.empty(4, device=DEV)
        F.preference_(x, t, w, cu, want, grad=want_grad, sums=want_sums, ref_logp=ref)
        assert torch.equal(loss, want) and torch.equal(again, want) and torch.equal(grad, want_grad) and torch.equal(sums, want_sums)
