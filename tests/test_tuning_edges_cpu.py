"""Expert selection, preference objective and 8-bit AdamW on the CPU: calls at the edges of what they take."""
import pytest
import torch

from shadowspill_b200.ops import reference as R


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("E,k", [(600, 3), (600, 40), (64, 33), (40, 40)])
@pytest.mark.parametrize("sigmoid", [True, False])
def test_layers_of_any_number_of_experts_route_on_the_cpu(E, k, sigmoid):
    import shadowspill_b200.frontend.ops  # noqa: F401
    x, bias, up = _rand(9, E).requires_grad_(True), _rand(E, seed=1) * 0.1, _rand(9, k, seed=2)
    ids, w = torch.ops.ss.select_experts(x, bias, k, sigmoid, 1, 1, True, 1.5)
    y = x.detach().double().requires_grad_(True)
    s = torch.sigmoid(y) if sigmoid else torch.softmax(y, 1)
    assert torch.equal(ids.long(), torch.sort(s + bias.double(), dim=1, descending=True, stable=True).indices[:, :k])
    c = s.gather(1, ids.long())
    want = 1.5 * c / (c.sum(1, keepdim=True) + 1e-20)
    (w * up).sum().backward()
    (want * up.double()).sum().backward()
    # weights and gradients are formed in 64 bits and rounded once, but for fp32 weights in the sum above, which no gradient sees
    assert bool(((w.double() - want).abs() <= 2.0 ** -24 * want).all())
    assert bool(((x.grad.double() - y.grad).abs() <= 2.0 ** -23 * y.grad.abs() + 1e-12).all())


def test_more_picks_than_experts_are_refused_on_the_cpu():
    import shadowspill_b200.frontend.ops  # noqa: F401
    for k, groups, keep in ((9, 1, 1), (0, 1, 1), (5, 4, 2), (1, 3, 1), (1, 2, 3), (1, 2, 0)):
        with pytest.raises(ValueError):
            torch.ops.ss.select_experts(_rand(3, 8), torch.zeros(8), k, True, groups, keep, True, 1.0)
    assert R.select_experts(_rand(3, 8), 8)[0].shape == (3, 8)


def test_a_sum_keeps_its_heads_settings():
    from shadowspill_b200.models.objectives import Objective
    settings = dict(preference_loss="ipo", preference_beta=0.5, average_logprobs=True, reference_free=True)
    got = Objective.from_component("shadowspill/sum@1", head="shadowspill/preference@1", head_config=settings, moe_balance=0.01)
    assert got == Objective("preference", moe_balance_coef=0.01, **settings) and got.extra_fields == ()
    got = Objective.from_component("shadowspill/sum@1", head="shadowspill/clipped_policy@1", head_config={"clip_ratio": 0.1, "reference_beta": 0.3})
    assert got == Objective("clipped_policy", clip_ratio=0.1, reference_beta=0.3)


def test_the_graph_only_family_names_the_objective_that_it_does_not_cover():
    from shadowspill_b200.frontend.capture import BatchGeometry, StepDataOrdering, build_step
    from shadowspill_b200.models.config import preset
    from shadowspill_b200.models.objectives import Objective
    geo = BatchGeometry(microbatch_tokens=256, n_microbatches=2, slots=16, mean_seqlen=64)
    for ob, match in ((Objective("preference"), "the preference objective"), (Objective("clipped_policy"), "the clipped_policy objective"),
                      (Objective(moe_balance_coef=0.01), "router-balance")):
        with pytest.raises(ValueError, match=match):
            build_step(preset("glm53-tiny"), geo, StepDataOrdering(), dtype=torch.float32, objective=ob)


def test_an_update_that_is_refused_leaves_every_tensor_as_it_was():
    from shadowspill_b200.ops import functional as F
    good = [(torch.ones(300), torch.ones(300), *F.moments8(300), 0) for _ in range(2)]
    for bad in ((torch.ones(8), torch.ones(7), *F.moments8(8), 0), (torch.ones(8), torch.ones(8), *F.moments8(8), 4),
                (torch.ones(8, dtype=torch.float64), torch.ones(8), *F.moments8(8), 0)):
        with pytest.raises((ValueError, TypeError)):
            F.adamw8_many_([*good, bad], lr=0.1)
        for p, _, m, r, m_exp, r_exp, _ in good:
            assert float((p - 1).abs().max()) == 0.0 and not any(int(x.view(torch.uint8).sum()) for x in (m, r, m_exp, r_exp))
