"""Measured cases of three operators of a routed model's preference tuning: the selection of experts (``ops/routing.py``),
the preference loss over a block of logits and the AdamW update with 8-bit moments (``ops/functional.py``).

``listed()`` names the cases and ``draw(rng)`` gives one more of the same ranges; ``prepare(case, seed)`` makes a case's inputs on the GPU,
``run(state)`` makes one pass, in plain tensor operations or (``own``) by the framework's calls, ``exact(case, seed)`` is the
same from the definitions in 64 bits, and ``work(case)`` counts what a pass has to move and to compute."""
import math
import random

import torch

own = False
DEV = "cuda"
BLOCK = 256                                   # elements that share a moment's exponent
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------ the cases
def listed():
    route = dict(op="route", scoring="softmax", bias=False, groups=1, keep=1, renorm=True, scale=1.0, dtype="fp32", train=True)
    pref = dict(op="preference", kind="sigmoid", smoothing=0.0, average=False, dtype="bf16", prompt=0.3, beta=0.1, empty=False)
    adam = dict(op="adamw8", dtype="bf16", grads="bf16", step=10)
    return [
        # one token through a sigmoid-scored router with groups: nothing but latency
        dict(route, name="route_one_token", T=1, E=256, k=8, scoring="sigmoid", bias=True, groups=8, keep=4, scale=2.5, train=False),
        # a training step's microbatch, softmax over 64 experts, weights as they are (olmoe-7b-a1b's router)
        dict(route, name="route_softmax_64", T=8192, E=64, k=8, renorm=False),
        # the same microbatch with sigmoid scores, a balance bias and scaled weights (glm53-published's router)
        dict(route, name="route_sigmoid_256", T=8192, E=256, k=8, scoring="sigmoid", bias=True, scale=2.5),
        # a long microbatch of odd length, many experts in groups, logits in bf16
        dict(route, name="route_grouped_long", T=65537, E=512, k=10, bias=True, groups=8, keep=3, dtype="bf16"),
        # one short pair on a small model's vocabulary (llama3-plumbing): launches
        dict(pref, name="preference_small", P=1, R=24, V=4096),
        # a handful of pairs, olmoe-7b-a1b's vocabulary, smoothed labels
        dict(pref, name="preference_pairs_50k", P=4, R=1021, V=50304, smoothing=0.1),
        # a microbatch of pairs on llama3-8b's vocabulary
        dict(pref, name="preference_llama3_8b", P=8, R=4096, V=128256),
        # one pair of long answers, hardly any prompt
        dict(pref, name="preference_long_pair", P=1, R=5000, V=50304, prompt=0.05),
        # fp32 logits of an odd vocabulary, mean log ratios, the squared loss
        dict(pref, name="preference_ragged_fp32", P=3, R=333, V=32003, kind="ipo", average=True, dtype="fp32"),
        # every tensor of a small model (llama3-plumbing) in one call
        dict(adam, name="adamw8_small_model", shapes="plumbing"),
        # one decoder layer of llama3-8b
        dict(adam, name="adamw8_layer_8b", shapes="layer8b"),
        # fp32 parameters and gradients, sizes off every boundary
        dict(adam, name="adamw8_odd_fp32", shapes="1000003,77777,511,257,255,9,1", dtype="fp32", grads="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "preference", "adamw8"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * rng.choice([8, 12, 16, 32, 40, 64])
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, keep * E // groups))
        return dict(op="route", T=_log(rng, 1, 65537), E=E, k=k, scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6,
                    groups=groups, keep=keep, renorm=k > 1 and rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["fp32", "bf16"]), train=rng.random() < 0.8)
    if op == "preference":
        kind = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        V = _log(rng, 1000, 152000)
        R = min(_log(rng, 8, 8192), 500_000_000 // V)
        return dict(op="preference", P=min(_log(rng, 1, 16), max(1, R // 4)), R=R, V=V, kind=kind,
                    smoothing=rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0, average=kind == "ipo" or rng.random() < 0.3,
                    dtype=rng.choice(["bf16", "bf16", "fp32"]), prompt=rng.choice([0.0, 0.3, 0.6]), beta=rng.choice([0.05, 0.1, 0.5]),
                    empty=rng.random() < 0.3)
    dtype = rng.choice(["bf16", "fp32"])
    sizes = [_log(rng, 1, 20_000_000) for _ in range(rng.randint(1, 12))]
    return dict(op="adamw8", shapes=",".join(map(str, sizes)), dtype=dtype, grads=rng.choice([dtype, "fp32"]), step=_log(rng, 1, 2000))


def _sizes(case):
    if case["shapes"] == "plumbing":          # d 256, ff 688, 4 layers, kv width 128, vocabulary 4,096
        layer = [256, 512 * 256, 256 * 256, 256, 1376 * 256, 256 * 688]
        return [4096 * 256] + layer * 4 + [256, 4096 * 256]
    if case["shapes"] == "layer8b":           # d 4,096, ff 14,336, q/k/v widths 4,096 + 2 x 1,024
        return [4096, 6144 * 4096, 4096 * 4096, 4096, 28672 * 4096, 4096 * 14336]
    return [int(s) for s in case["shapes"].split(",")]


def _bounds(case):
    """Row bounds of the 2 P sequences; a few rows stay behind the last one."""
    rng = random.Random(case["R"] * 31 + case["P"])
    S, used = 2 * case["P"], case["R"] - min(case["R"] // 50, 7)
    cuts = [(i + rng.uniform(-0.3, 0.3)) / S for i in range(1, S)]
    at = [0] + [int(c * used) for c in cuts] + [used]
    if case["empty"]:
        at[1] = 0                             # the first pair has no chosen sequence
    return at


def _scored(case):
    """For every row: does it carry weight?"""
    at, out = _bounds(case), [False] * case["R"]
    for a, b in zip(at[:-1], at[1:]):
        for r in range(a + int((b - a) * case["prompt"]), b):
            out[r] = True
    return out


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    with torch.no_grad():
        return {"route": _prepare_route, "preference": _prepare_preference, "adamw8": _prepare_adamw8}[case["op"]](case, g, rand)


def _prepare_route(case, g, rand):
    T, E = case["T"], case["E"]
    state = dict(case=case, logits=(rand(T, E) * 1.5).to(DTYPES[case["dtype"]]), bias=rand(E) * 0.05 if case["bias"] else None)
    if case["train"]:
        state["dweights"] = rand(T, case["k"])
    return state


def _prepare_preference(case, g, rand):
    R, V = case["R"], case["V"]
    dtype = DTYPES[case["dtype"]]
    wide = (V + 7) // 8 * 8                    # rows start on 16 bytes
    logits = torch.empty(R, wide, dtype=dtype, device=DEV)[:, :V]
    targets = torch.randint(0, V, (R,), generator=g, device=DEV)
    logp = torch.empty(R, device=DEV)
    rows = max(1, 40_000_000 // V)
    for a in range(0, R, rows):                # the target's logit stands out, as a trained model's does
        x, t = rand(min(rows, R - a), V) * 2.0, targets[a:a + rows, None]
        x.scatter_add_(1, t, 5.0 + 2.0 * rand(x.shape[0], 1))
        logits[a:a + rows] = x.to(dtype)
        logp[a:a + rows] = x.gather(1, t)[:, 0] - torch.logsumexp(x, 1)
    scored = torch.tensor(_scored(case), device=DEV)
    targets = torch.where(scored | (torch.rand(R, generator=g, device=DEV) < 0.5), targets, -100)
    return dict(case=case, logits=logits, targets=targets, weights=scored.float(), ref_logp=logp + 0.3 * rand(R),
                cu_seqlens=torch.tensor(_bounds(case), dtype=torch.int32, device=DEV),
                grad=torch.empty(R, wide, dtype=dtype, device=DEV)[:, :V], sums=torch.empty(2 * case["P"], device=DEV))


def _prepare_adamw8(case, g, rand):
    sizes, places, at = _sizes(case), [], 0
    for n in sizes:                            # views of flat buffers, each on its own blocks, as a stage holds them
        places.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    p, grad = torch.zeros(at, device=DEV, dtype=DTYPES[case["dtype"]]), torch.zeros(at, device=DEV, dtype=DTYPES[case["grads"]])
    m, r = (torch.zeros(at, device=DEV, dtype=torch.float8_e4m3fn) for _ in range(2))
    m_exp, r_exp = (torch.zeros(at // BLOCK, device=DEV, dtype=torch.uint8) for _ in range(2))
    tensors = []
    for n, a in zip(sizes, places):
        blocks = slice(a // BLOCK, a // BLOCK + (n + BLOCK - 1) // BLOCK)
        k = blocks.stop - blocks.start
        size = torch.exp(1.5 * rand(k, 1) - 7.0)                          # gradients of a size per block
        fill = lambda x: x.reshape(-1)[:n]
        p[a:a + n] = fill(rand(k, BLOCK) * 0.02).to(p.dtype)
        grad[a:a + n] = fill(rand(k, BLOCK) * size).to(grad.dtype)
        for codes, exps, x in ((m, m_exp, rand(k, BLOCK) * size * 0.3), (r, r_exp, (rand(k, BLOCK).abs() + 0.1) * size)):
            x.reshape(-1)[n:] = 0.0
            e = _exponent(x.abs().amax(1))
            codes[a:a + n] = fill(x * torch.exp2(127.0 - e[:, None])).to(codes.dtype)
            exps[blocks] = e.to(torch.uint8)
        tensors.append((p[a:a + n], grad[a:a + n], m[a:a + n], r[a:a + n], m_exp[blocks], r_exp[blocks], a))
    return dict(case=case, tensors=tensors, flat=(p, grad, m, r, m_exp, r_exp))


def _hyper(case):
    return dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=case["step"], grad_scale=0.5)


def _exponent(top):
    """Biased exponent e of the smallest power of two with top <= 448 * 2^(e - 127); 0 for a block of zeros."""
    fraction, e = torch.frexp(top)             # top = fraction * 2^e with fraction in [0.5, 1)
    e = e + torch.where(fraction > 0.875, -8, -9) + 127
    return torch.where(top > 0, e.clamp(min=1), 0).float()


# ------------------------------------------------------------------------ one pass
def run(state):
    return {"route": _run_route, "preference": _run_preference, "adamw8": _run_adamw8}[state["case"]["op"]](state)


def _run_route(state):
    c, x, bias = state["case"], state["logits"], state["bias"]
    if own:
        from shadowspill_b200.ops import routing
        ids, weights, counts = routing.select_experts(x, c["k"], scoring=c["scoring"], bias=bias, groups=c["groups"], keep_groups=c["keep"],
                                                      renormalize=c["renorm"], scale=c["scale"])
        out = dict(ids=ids, weights=weights, counts=counts)
        if c["train"]:
            out["dlogits"] = routing.select_experts_bwd(x, ids, state["dweights"], scoring=c["scoring"], renormalize=c["renorm"], scale=c["scale"])
        return out
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    x64 = x.double()                           # keys next to each other: 64 bits
    if c["scoring"] == "sigmoid":
        s = 1 / (1 + torch.exp(-x64))
    else:
        s = torch.exp(x64 - x64.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    key = s if bias is None else s + bias.double()
    if bias is None and G == 1:
        key = x64
    if G > 1:
        best = torch.sort(key.view(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        off = torch.ones(T, G, dtype=torch.bool, device=x.device).scatter(1, kept, False)
        key = key.masked_fill(off[:, :, None].expand(T, G, E // G).reshape(T, E), -math.inf)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    s = s.float()
    picked = s.gather(1, ids)
    total = picked.sum(1, keepdim=True) + 1e-20
    weights = picked / total * c["scale"] if c["renorm"] else picked * c["scale"]
    counts = torch.zeros(E, dtype=torch.int32, device=x.device)
    counts.index_add_(0, ids.reshape(-1), torch.ones(T * k, dtype=torch.int32, device=x.device))
    out = dict(ids=ids.to(torch.int32), weights=weights, counts=counts)
    if c["train"]:
        d = state["dweights"]
        d = c["scale"] / total * (d - (d * picked / total).sum(1, keepdim=True)) if c["renorm"] else c["scale"] * d
        wide = torch.zeros(T, E, device=x.device).scatter(1, ids, d)
        dx = wide * s * (1 - s) if c["scoring"] == "sigmoid" else s * (wide - (d * picked).sum(1, keepdim=True))
        out["dlogits"] = dx.to(x.dtype)
    return out


def _run_preference(state):
    c, x, targets, weights, cu = state["case"], state["logits"], state["targets"], state["weights"], state["cu_seqlens"]
    if own:
        from shadowspill_b200.ops import functional as F
        loss = torch.zeros(1, device=x.device)
        F.preference_(x, targets, weights, cu, loss, beta=c["beta"], kind=c["kind"], label_smoothing=c["smoothing"], average=c["average"],
                      ref_logp=state["ref_logp"], grad=state["grad"], sums=state["sums"])
        return dict(loss=loss, sums=state["sums"], grad=state["grad"])
    R, V = x.shape
    f = x.float()
    f = f - f.amax(1, keepdim=True)
    valid = (targets >= 0) & (targets < V) & (weights != 0)
    t = torch.where(valid, targets, 0)[:, None]
    picked = f.gather(1, t)[:, 0]
    e = torch.exp(f)
    del f
    total = e.sum(1, keepdim=True)
    ratio = torch.where(valid, weights * (picked - torch.log(total[:, 0]) - state["ref_logp"]), 0)
    rows = torch.arange(R, device=x.device)
    member = ((rows >= cu[:-1, None]) & (rows < cu[1:, None])).double()       # long sums of log ratios: 64 bits
    sums, mass = member @ ratio.double(), member @ (valid * weights).double()
    if c["average"]:
        sums = sums / torch.where(mass > 0, mass, 1)
    sums, mass = sums.float(), mass.float()
    z = c["beta"] * (sums[0::2] - sums[1::2])
    live = ((member @ valid.double()) > 0).view(-1, 2).all(1)
    if c["kind"] == "sigmoid":
        soft = lambda a: torch.clamp(a, min=0) + torch.log(1 + torch.exp(-a.abs()))
        loss = (1 - c["smoothing"]) * soft(-z) + c["smoothing"] * soft(z)
        slope = c["smoothing"] - 1 / (1 + torch.exp(z))
    elif c["kind"] == "hinge":
        loss, slope = torch.clamp(1 - z, min=0), torch.where(z < 1, -1.0, 0.0)
    else:
        gap = z / c["beta"] - 1 / (2 * c["beta"])
        loss, slope = gap * gap, 2 * gap / c["beta"]
    pull = torch.where(live, c["beta"] * slope, 0)
    pull = torch.stack((pull, -pull), 1).view(-1)
    if c["average"]:
        pull = pull / torch.where(mass > 0, mass, 1)
    coef = torch.where(valid, -weights * (member.float().t() @ pull[:, None])[:, 0], 0)
    grad = e / total
    del e
    grad.scatter_add_(1, t, torch.full((R, 1), -1.0, device=x.device))
    grad *= coef[:, None]
    return dict(loss=torch.where(live, loss, 0).sum().reshape(1), sums=sums, grad=grad.to(x.dtype))


def _run_adamw8(state):
    c, h = state["case"], _hyper(state["case"])
    p, g, m, r, m_exp, r_exp = state["flat"]
    if own:
        from shadowspill_b200.ops import functional as F
        F.adamw8_many_(state["tensors"], **h, stochastic_param=False, stochastic_state=False)
        return dict(p=p, m=m, r=r, m_exp=m_exp, r_exp=r_exp)
    unit = lambda e: torch.exp2(e.float() - 127.0)[:, None]
    gf = (g.float() * h["grad_scale"]).view(-1, BLOCK)
    mf = h["beta1"] * (m.float().view(-1, BLOCK) * unit(m_exp)) + (1 - h["beta1"]) * gf
    rf = r.float().view(-1, BLOCK) * unit(r_exp)
    rf = torch.sqrt(h["beta2"] * (rf * rf) + (1 - h["beta2"]) * gf * gf)
    del gf
    bias1, bias2 = 1 - h["beta1"] ** h["step"], math.sqrt(1 - h["beta2"] ** h["step"])
    pf = p.float().view(-1, BLOCK)
    pf = pf * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * (mf / bias1) / (rf / bias2 + h["eps"])
    p.copy_(pf.reshape(-1))
    del pf
    e = _exponent(mf.abs().amax(1))
    m.copy_((mf * torch.exp2(127.0 - e)[:, None]).reshape(-1))
    m_exp.copy_(e)
    e = _exponent(rf.amax(1))
    y = rf * torch.exp2(127.0 - e)[:, None]
    r.copy_(torch.where(rf > 0, torch.clamp(y, min=2.0 ** -9), 0.0).reshape(-1))
    r_exp.copy_(e)
    return dict(p=p, m=m, r=r, m_exp=m_exp, r_exp=r_exp)


# ------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "preference": _exact_preference, "adamw8": _exact_adamw8}[case["op"]](case, state)


def _exact_route(case, state):
    x = state["logits"].double().requires_grad_(True)
    E, G, k = case["E"], case["groups"], case["k"]
    s = torch.sigmoid(x) if case["scoring"] == "sigmoid" else torch.softmax(x, 1)
    with torch.no_grad():
        key = s + (0 if state["bias"] is None else state["bias"].double())
        if G == 1 and state["bias"] is None:
            key = x.detach()
        if G > 1:
            group = key.unflatten(1, (G, E // G))
            best = group.topk(min(2, E // G), 2).values.sum(2)
            # the place of a group: how many are better, or as good and before it
            order = torch.arange(G, device=x.device)
            ahead = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) & (order[None, :] < order[:, None]))
            group = torch.where((ahead.sum(2) < case["keep"])[:, :, None], group, -math.inf)
            key = group.flatten(1)
        ids = torch.argsort(key, dim=1, descending=True, stable=True)[:, :k]
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = w * case["scale"]
    out = dict(ids=ids.int(), weights=w.detach(), counts=torch.bincount(ids.flatten(), minlength=E).int())
    if case["train"]:
        out["dlogits"] = torch.autograd.grad(w, x, state["dweights"].double())[0]
    return out


def _exact_preference(case, state):
    R, V = state["logits"].shape
    at, beta, rows = _bounds(case), case["beta"], max(1, 60_000_000 // V)
    w, t = state["weights"].double(), state["targets"].clamp(0, V - 1)
    w = torch.where((state["targets"] >= 0) & (state["targets"] < V), w, 0.0)
    logp = torch.cat([torch.log_softmax(state["logits"][a:a + rows].double(), 1).gather(1, t[a:a + rows, None])[:, 0] for a in range(0, R, rows)])
    ratio = w * (logp - state["ref_logp"].double())
    share = [w[a:b].sum().item() if case["average"] else 1.0 for a, b in zip(at[:-1], at[1:])]
    sums = torch.stack([ratio[a:b].sum() / (n or 1.0) for (a, b), n in zip(zip(at[:-1], at[1:]), share)]).requires_grad_(True)
    loss = sums.sum() * 0
    for i in range(case["P"]):
        if not all(bool((w[at[j]:at[j + 1]] != 0).any()) for j in (2 * i, 2 * i + 1)):
            continue
        z = beta * (sums[2 * i] - sums[2 * i + 1])
        if case["kind"] == "sigmoid":
            up, down = torch.nn.functional.logsigmoid(z), torch.nn.functional.logsigmoid(-z)
            loss = loss - (1 - case["smoothing"]) * up - case["smoothing"] * down
        elif case["kind"] == "hinge":
            loss = loss + torch.relu(1 - z)
        else:
            loss = loss + (z / beta - 1 / (2 * beta)) ** 2
    pull = torch.autograd.grad(loss, sums)[0]
    up = torch.zeros(R, dtype=torch.float64, device=w.device)
    for j, (a, b) in enumerate(zip(at[:-1], at[1:])):
        up[a:b] = pull[j] * w[a:b] / (share[j] or 1.0)
    grad = torch.empty(R, V, dtype=torch.float64, device=w.device)
    for a in range(0, R, rows):
        part = -torch.softmax(state["logits"][a:a + rows].double(), 1)
        part.scatter_add_(1, t[a:a + rows, None], torch.ones(part.shape[0], 1, dtype=torch.float64, device=w.device))
        grad[a:a + rows] = part * up[a:a + rows, None]
    return dict(loss=loss.detach().reshape(1), sums=sums.detach(), grad=grad)


def _exact_adamw8(case, state):
    h = _hyper(case)
    p, g, m, r, m_exp, r_exp = state["flat"]
    spread = lambda e: torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.int() - 127).repeat_interleave(BLOCK)
    grad = g.double() * h["grad_scale"]
    first = torch.lerp(grad, m.double() * spread(m_exp), h["beta1"])
    second = torch.lerp(grad.square(), (r.double() * spread(r_exp)).square(), h["beta2"])
    root = second.sqrt()
    step = first / (1 - h["beta1"] ** h["step"]) / ((second / (1 - h["beta2"] ** h["step"])).sqrt() + h["eps"])
    new = p.double() - h["lr"] * (step + h["weight_decay"] * p.double())
    units = []
    for x in (first, root):                    # by the logarithm: the smallest power of two that holds the block
        top = x.abs().view(-1, BLOCK).amax(1)
        e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)).clamp(min=-126), -127)
        units.append(torch.ldexp(x.view(-1, BLOCK), -e.int()[:, None]).reshape(-1))
    return dict(p=new, m=units[0], r=units[1], m_exp=None, r_exp=None)


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        b = size[case["dtype"]]
        moved = T * E * b + 8 * T * k + 4 * E * (2 if case["bias"] else 1)
        return {"bytes": moved + (T * E * b + 4 * T * k if case["train"] else 0), "flops": T * E * (8 if case["train"] else 4)}
    if case["op"] == "preference":
        R, V, b = case["R"], case["V"], size[case["dtype"]]
        scored = sum(_scored(case))
        return {"bytes": (scored + R) * V * b + 16 * R, "flops": 7 * scored * V}
    n = sum(_sizes(case))
    return {"bytes": n * (2 * size[case["dtype"]] + size[case["grads"]] + 4) + 4 * sum(-(-s // BLOCK) for s in _sizes(case)), "flops": 20 * n}
