"""Expert selection, preference loss and 8-bit AdamW as one training step uses them, and through either of their host paths."""
import pytest
import torch

from shadowspill_b200.ops import _lib, functional as F, moe, reference as R, routing

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Refuses:
    def __getattr__(self, name):
        return lambda *a: NotImplemented


def _everything():
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(70, 96, generator=g, device=DEV)
    bias = torch.randn(96, generator=g, device=DEV) * 0.1
    out = list(routing.select_experts(x, 6, scoring="sigmoid", bias=bias, groups=4, keep_groups=2, scale=2.5))
    out.append(routing.select_experts_bwd(x, out[0], out[1], scoring="sigmoid", scale=2.5))
    logits = torch.randn(40, 1000, generator=g, device=DEV).bfloat16()
    targets = torch.randint(0, 1000, (40,), generator=g, device=DEV)
    weights, ref = torch.rand(40, generator=g, device=DEV), -torch.rand(40, generator=g, device=DEV)
    cu = torch.tensor([0, 9, 17, 30, 38], dtype=torch.int32, device=DEV)
    loss, sums, logp = torch.zeros(1, device=DEV), torch.empty(4, device=DEV), torch.empty(40, device=DEV)
    assert F.preference_(logits, targets, weights, cu, loss, ref_logp=ref, sums=sums, logp=logp, label_smoothing=0.1) is loss
    out += [logits, loss, sums, logp]
    tensors = []
    for i, n in enumerate((300, 5000, 7)):
        p, grad = torch.randn(n, generator=g, device=DEV).bfloat16(), torch.randn(n, generator=g, device=DEV).bfloat16()
        tensors.append((p, grad, *F.moments8(n, DEV), 8 * i))
    F.adamw8_many_(tensors, lr=0.01, seed=7, step=2)
    return out + [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for item in tensors for t in item[:6]]


def test_the_native_module_gives_the_bits_of_the_python_path(monkeypatch):
    before = _lib.launch_counts()
    got = _everything()
    after = _lib.launch_counts()
    for entry, n in (("ss_select_experts", 1), ("ss_select_experts_bwd", 1), ("ss_preference with its gradient", 2), ("ss_adamw8_many", 1)):
        assert after.get(entry, 0) - before.get(entry, 0) == n, entry
    with monkeypatch.context() as m:
        m.setattr(_lib, "_host", _Refuses())
        want = _everything()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_native_module_leaves_other_operands_to_python():
    h = _lib.host()
    x = torch.randn(8, 16, device=DEV)
    for bad in ((x.half(), 2, 0, None, 1, 1, True, 1.0), (x, 17, 0, None, 1, 1, True, 1.0), (x, 2, 2, None, 1, 1, True, 1.0),
                (x, 2, 0, torch.zeros(16), 1, 1, True, 1.0), (x.t(), 2, 0, None, 1, 1, True, 1.0), (x, 2, 0, None, 3, 1, True, 1.0)):
        assert h.select_experts(*bad) is NotImplemented
    state = F.moments8(64, DEV)
    p, g = torch.zeros(64, device=DEV), torch.zeros(64, device=DEV)
    hyper = (0.1, 0.9, 0.95, 1e-8, 0.0, 1.0)
    for tensors in ([], [(p, g, *state, 4)], [(p, g[:63], *state, 0)], [(p, g, *state, 0), (p, g, *state, 0)], [(p.half(), g, *state, 0)],
                    [(p, g, state[0].view(torch.uint8), *state[1:], 0)], [(p, g, *state, 0), (p.bfloat16(), g, *F.moments8(64, DEV), 0)]):
        assert h.adamw8_many(tensors, hyper, 1, 0, True, True) is NotImplemented
    with pytest.raises(TypeError):
        h.preference(x)


def _step(router, w13, w2, head, state, x, targets, weights, cu, ref, step, cuda):
    """A routed layer, a head and a preference loss, forward and backward by hand, and the update of all four matrices."""
    T, E, k = x.shape[0], router.shape[0], 2
    logits_r = x.float() @ router.float().t()
    ids, wts, counts = routing.select_experts(logits_r, k, scoring="sigmoid", bias=state["bias"], groups=2, keep_groups=2, scale=2.0)
    lay = moe.Layout(ids, counts)
    xs = lay.gather(x)
    gu, act = moe.grouped_swiglu(xs, w13, lay)
    y = lay.combine(moe.grouped_linear(act, w2, lay), wts)
    h = x + y
    logits = F.linear_fwd(h, head)
    loss = torch.zeros(1, device=x.device)
    F.preference_(logits, targets, weights, cu, loss, beta=0.5, ref_logp=ref)
    d_head = F.linear_wgrad(logits, h)
    dh = F.linear_dgrad(logits, head)
    dos = lay.gather(dh)
    dgu, hw, dw = lay.act_bwd(gu, moe.grouped_linear(dos, w2, lay, transpose=True), wts)
    d_w2, d_w13 = torch.zeros_like(w2), torch.zeros_like(w13)
    moe.grouped_wgrad(dos, hw, lay, d_w2, False)
    moe.grouped_wgrad(dgu, xs, lay, d_w13, False)
    d_logits = routing.select_experts_bwd(logits_r, ids, dw, scoring="sigmoid", scale=2.0)
    d_router = (d_logits.t() @ x.float())
    grads = dict(router=d_router, w13=d_w13, w2=d_w2, head=d_head)
    tensors, offset = [], 0
    for name, p in (("router", router), ("w13", w13), ("w2", w2), ("head", head)):
        tensors.append((p.view(-1), grads[name].reshape(-1), *state[name], offset))
        offset += (p.numel() + 255) // 256 * 256
    F.adamw8_many_(tensors, lr=1e-3, step=step, seed=5, stochastic_param=False, stochastic_state=False)
    return loss, grads


def test_a_step_of_all_three_against_autograd():
    """The gradients that reach the update are those of one loss: the same step in fp64 by autograd with the picks held."""
    T, D, E, Fw, V = 256, 128, 8, 128, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).bfloat16()
    router, w13, w2, head, x = r(E, D, std=0.2), r(E, 2 * Fw, D, std=0.1), r(E, D, Fw, std=0.1), r(V, D, std=0.1), r(T, D)
    targets = torch.randint(0, V, (T,), generator=g, device=DEV)
    weights = (torch.rand(T, generator=g, device=DEV) < 0.7).float()
    cu = torch.tensor([0, 60, 128, 190, 250], dtype=torch.int32, device=DEV)
    ref = torch.randn(T, generator=g, device=DEV) * 0.1 - 7.0
    state = {n: F.moments8(p.numel(), DEV) for n, p in (("router", router), ("w13", w13), ("w2", w2), ("head", head))}
    state["bias"] = torch.randn(E, generator=g, device=DEV) * 0.05
    before = [t.double().clone().requires_grad_(True) for t in (router, w13, w2, head)]
    loss, grads = _step(router, w13, w2, head, state, x, targets, weights, cu, ref, 1, True)
    _lib.check_status()
    R64, W13, W2, H = before
    xd = x.double()
    lr_ = xd @ R64.t()
    ids, _, _ = R.select_experts((x.float() @ router_before(before).t()), 2, "sigmoid", state["bias"], 2, 2, True, 2.0)
    c = torch.sigmoid(lr_).gather(1, ids.long())
    c = 2.0 * c / c.sum(1, keepdim=True)
    out = xd.clone()
    for j in range(2):
        a = torch.einsum("td,tfd->tf", xd, W13[ids[:, j].long()])
        act = torch.nn.functional.silu(a[:, :Fw]) * a[:, Fw:]
        out = out + c[:, j:j + 1] * torch.einsum("tf,tdf->td", act, W2[ids[:, j].long()])
    lp = torch.log_softmax(out @ H.t(), 1).gather(1, targets[:, None])[:, 0] - ref.double()
    s = [(weights.double() * lp)[a:b].sum() for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:])]
    want = sum(torch.nn.functional.softplus(-0.5 * (s[i] - s[i + 1])) for i in (0, 2))
    exact = torch.autograd.grad(want, before)
    # each of the chain's seven bf16 stores (logits, their gradient, rows in and out, activations and theirs, the result) rounds by
    # 2^-8 of its value, and errors of a chain add; the margin itself sums 40 rows' logits, each off by 2^-8 of a few units
    assert abs(float(loss) - float(want)) <= 0.5 * 40 ** 0.5 * 2.0 ** -8 * 4 * 2
    for name, e in zip(("router", "w13", "w2", "head"), exact):
        rel = float((grads[name].double() - e).norm() / e.norm())
        assert rel <= 7 * 2.0 ** -8 + 0.5 * 40 ** 0.5 * 2.0 ** -8 * 4, (name, rel)
    # and the update is the definition's for these gradients: a first step moves every element by lr where it has a gradient
    moved = (head.double() - H.detach()).abs()
    assert float(moved.max()) <= 1e-3 * 1.01 + float(H.detach().abs().max()) * 2.0 ** -8
    m = R.moment_values(state["head"][0], state["head"][2])
    assert float((m - 0.1 * grads["head"].float().reshape(-1)).abs().max()) <= 0.1 * float(grads["head"].abs().max()) * 2.0 ** -4


def router_before(before):
    return before[0].detach().float()


def test_calls_one_behind_the_other_see_what_came_before():
    """Kernels of these operators start beside the one before them: inputs written and buffers reused just ahead of every call."""
    g = torch.Generator(device=DEV).manual_seed(30)
    logits = [torch.randn(3000, 64, generator=g, device=DEV) for _ in range(30)]
    words = [torch.randn(700, 4000, generator=g, device=DEV).bfloat16() for _ in range(30)]
    t = torch.randint(0, 4000, (700,), generator=g, device=DEV)
    cu = torch.arange(0, 701, 35, dtype=torch.int32, device=DEV)
    x, y = torch.empty_like(logits[0]), torch.empty_like(words[0])
    results = []
    for wait in (True, False):
        p = torch.ones(300_001, device=DEV, dtype=torch.bfloat16)
        state = F.moments8(p.numel(), DEV)
        kept = []
        torch.cuda.synchronize()
        for i in range(30):
            steps = []

            def done(*tensors):
                steps.extend(v.clone() for v in tensors)
                if wait:
                    torch.cuda.synchronize()
            x.copy_(logits[i])
            ids, w, counts = routing.select_experts(x, 6, scoring="sigmoid")
            done(ids, w, counts)
            done(routing.select_experts_bwd(x, ids, w, scoring="sigmoid"))
            del ids, w, counts
            y.copy_(words[i])
            loss = torch.zeros(1, device=DEV)
            F.preference_(y, t, None, cu, loss)
            done(y, loss)
            F.adamw8_many_([(p, y.view(-1)[:300_001], *state, 0)], lr=1e-2, step=i + 1)
            done(p, *(v.view(torch.uint8) for v in state))
            x.zero_()
            y.zero_()
            kept.append(steps)
        torch.cuda.synchronize()
        results.append(kept)
    assert all(torch.equal(a, b) for one, other in zip(*results) for a, b in zip(one, other))
