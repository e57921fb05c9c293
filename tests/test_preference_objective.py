"""The preference objective in the output head: planned execution against the resident trainer and against autograd on whole
logits; the routed layers' selection operator in exported stages."""
import numpy as np
import pytest
import torch

from shadowspill_b200.communication.info import CommunicationInfo
from shadowspill_b200.data.synthetic import make_batch, to_device
from shadowspill_b200.execution.executor import Executor, Hyperparameters
from shadowspill_b200.execution.resident import ResidentTrainer
from shadowspill_b200.frontend.capture import BatchGeometry, StepDataOrdering, build_step
from shadowspill_b200.models.config import preset
from shadowspill_b200.models.decoder import build_stages
from shadowspill_b200.models.objectives import Objective
from shadowspill_b200.ops import functional as F
from shadowspill_b200.planning.plan import MemoryBudgets, SearchOptions, plan_program

OB = Objective("preference", preference_beta=0.3, label_smoothing=0.1)


def _batch(cfg, seed=0, n=1, slots=16):
    host = make_batch(seed, vocab=cfg.vocab_size, tokens_per_step=256 * n, microbatch_tokens=256, median=40, min_len=8,
                      max_len=80, slots=slots)
    rng = np.random.default_rng(seed)
    for mb in host:
        mb.extras["reference_logprobs"] = (rng.standard_normal(256) * 0.3 - 6.0).astype(np.float32)
    return host


def _loss(logits, meta, ob):
    """By hand, differentiable, in 64 bits."""
    ok = (meta.targets >= 0) & (meta.weights != 0)
    lp = torch.log_softmax(logits.double(), 1).gather(1, meta.targets.clamp(min=0)[:, None])[:, 0]
    ratio = torch.where(ok, meta.weights.double() * (lp - meta.extras["reference_logprobs"].double()), 0.0)
    cu, total = meta.cu_seqlens.tolist(), 0.0
    for i in range((len(cu) - 1) // 2):
        a, b, c = cu[2 * i:2 * i + 3]
        if bool(ok[a:b].any()) and bool(ok[b:c].any()):
            z = ob.preference_beta * (ratio[a:b].sum() - ratio[b:c].sum())
            soft = torch.nn.functional.softplus
            total = total + (1 - ob.label_smoothing) * soft(-z) + ob.label_smoothing * soft(z)
    return total


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("slots", [16, 17])
def test_the_head_against_autograd(device, slots):
    cfg = preset("llama3-tiny")
    head = build_stages(cfg, objective=OB)[-1]
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    g = torch.Generator().manual_seed(2)
    P = {"final_norm": torch.ones(cfg.d_model, dtype=dtype, device=device),
         "head": (torch.randn(cfg.vocab_size, cfg.d_model, generator=g) * 0.2).to(device, dtype)}
    G = {"final_norm": torch.zeros(cfg.d_model, device=device), "head": torch.zeros(cfg.vocab_size, cfg.d_model, dtype=dtype, device=device)}
    meta = to_device(_batch(cfg, 3, slots=slots)[0], device)
    x = torch.randn(256, cfg.d_model, generator=g).to(device, dtype)
    loss = torch.zeros(1, device=device)
    dx = head.loss_and_backward(P, G, x, meta, loss, True)
    x64 = x.double().requires_grad_(True)
    W = P["head"].double().requires_grad_(True)
    h = x64 * torch.rsqrt(x64.square().mean(1, keepdim=True) + cfg.norm_epsilon)
    want = _loss(h @ W.t(), meta, OB)
    want.backward()
    # fp32: roundings of a few hundred products; bf16: hidden rows, logits, their gradients and both products are stored with 2^-8 each,
    # and a margin sums forty logits of a few units
    tol = 1e-4 if device == "cpu" else 5 * 2.0 ** -8 + 0.3 * 40 ** 0.5 * 2.0 ** -8 * 4
    assert abs(float(loss) - float(want.detach())) <= tol * max(1.0, float(want.detach()))
    for got, ref in ((dx, x64.grad), (G["head"], W.grad)):
        assert float((got.double() - ref).norm()) <= tol * float(ref.norm())
    again = torch.zeros(1, device=device)
    assert head.loss_and_backward(P, None, x, meta, again, True, train=False) is None
    assert torch.equal(again, loss)


def test_through_the_planned_executor():
    cfg = preset("llama3-tiny")
    assert OB.extra_fields == ("reference_logprobs",) and Objective("preference", reference_free=True).extra_fields == ()
    geo = BatchGeometry(microbatch_tokens=256, n_microbatches=2, slots=16, mean_seqlen=64)
    prog, desc = build_step(cfg, geo, StepDataOrdering(), dtype=torch.float32, objective=OB)
    total = sum(o.bytes for o in prog.objects) + max(t.workspace_bytes for t in prog.tasks)
    plan = plan_program(prog, MemoryBudgets(total, 64 << 20, headroom_bytes=0), CommunicationInfo(),
                        SearchOptions(minimum_object_bytes_evict_eligible=1024, workers=1))
    ex = Executor(plan, desc, device="cpu", seed=5, hyper=Hyperparameters(lr=1e-3))
    ex.initialize()
    tr = ResidentTrainer(cfg, device="cpu", dtype=torch.float32, seed=5, lr=1e-3, objective=OB)
    for step in range(2):
        host = _batch(cfg, step, n=2)
        got = ex.run(host).loss
        want = tr.step([to_device(m, "cpu") for m in host])
        assert abs(got - want) < 1e-5 * max(1.0, abs(want)), (step, got, want)
    ex.close()


def test_the_head_forms_all_logits_of_a_pair():
    cfg = preset("llama3-8b")
    plain, pairs = build_stages(cfg)[-1], build_stages(cfg, objective=OB)[-1]
    assert pairs.workspace_bytes(8192) - plain.workspace_bytes(8192) == (8192 - plain.block_rows) * cfg.vocab_size * 2
    assert pairs.workspace_bytes(1000) == plain.workspace_bytes(1000)


def test_records_and_refusals():
    assert Objective.from_json(OB.to_json()) == OB and OB.component_id == "shadowspill/preference@1"
    assert Objective.from_json({"kind": "clipped_policy", "clip_ratio": 0.1, "reference_beta": 0.0, "moe_balance_coef": 0.0}).clip_ratio == 0.1
    for bad in (dict(preference_loss="rank"), dict(preference_beta=0.0), dict(label_smoothing=1.0),
                dict(preference_loss="hinge", label_smoothing=0.1)):
        with pytest.raises(ValueError):
            Objective("preference", **bad)
    from shadowspill_b200.training.components import _objective_record
    for rec in ({"id": "shadowspill/preference@1"}, {"id": "shadowspill/sum@1", "terms": [{"id": "shadowspill/preference@1"}]}):
        with pytest.raises(ValueError, match="adjacent"):
            _objective_record(rec)


def _selection(device, dtype):
    import shadowspill_b200.frontend.ops  # noqa: F401
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(50, 16, generator=g).to(device, dtype)
    return logits, (torch.randn(16, generator=g) * 0.1).to(device), torch.randn(50, 3, generator=g).to(device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("sigmoid", [True, False])
def test_the_selection_operator_differentiates(device, sigmoid):
    logits, bias, up = _selection(device, torch.float32)
    x = logits.clone().requires_grad_(True)
    ids, wts = torch.ops.ss.select_experts(x, bias, 3, sigmoid, 4, 2, True, 2.5)
    (wts * up).sum().backward()
    y = logits.double().requires_grad_(True)
    s = torch.sigmoid(y) if sigmoid else torch.softmax(y, 1)
    c = s.gather(1, ids.long())
    w = 2.5 * c / (c.sum(1, keepdim=True) + 1e-20)
    (w * up.double()).sum().backward()
    # exponentials of arguments up to 4 (6 steps of 2^-23), a dozen roundings, of terms that cancel: their sizes' sum is under 2.5 * 8
    assert float((wts.double() - w.detach()).abs().max()) <= 2.5 * 30 * 2.0 ** -23
    assert float((x.grad.double() - y.grad).abs().max()) <= 20 * 30 * 2.0 ** -23
    torch.library.opcheck(torch.ops.ss.select_experts.default, (logits, bias, 3, sigmoid, 4, 2, True, 2.5),
                          test_utils=("test_schema", "test_faketensor"))


def test_routed_stages_of_the_latent_attention_family_select_by_the_operator():
    from shadowspill_b200.frontend.export import op_name
    cfg = preset("glm53-tiny")
    geo = BatchGeometry(microbatch_tokens=256, n_microbatches=2, slots=16, mean_seqlen=64)
    _, desc = build_step(cfg, geo, StepDataOrdering(), dtype=torch.float32)
    names = [op_name(n) for n in desc.stages()[2].graph.gm.graph.nodes]
    assert names.count("ss.select_experts") == 2 and not any(n.startswith("aten.topk") for n in names)
