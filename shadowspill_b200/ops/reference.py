"""Plain-PyTorch definitions of every model op.

These are the numerical oracles for the CUDA kernels and the execution path on
CPU. They restate the semantics of the reference's pure-PyTorch decoders
(packages/workloads/src/shadowspill_workloads/models/shared/decoder.py:18-330 and
models/qwen35/implementations/pytorch/delta_rule/reference.py:8-132) and run in
fp32 internally, casting at the same points the kernels do.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def gemm(a: torch.Tensor, b: torch.Tensor, *, a_mn: bool, b_mn: bool, out: torch.Tensor | None,
         accumulate: bool, alpha: float, out_dtype: torch.dtype) -> torch.Tensor:
    am = a.float().t() if a_mn else a.float()          # [M, K]
    bm = b.float() if b_mn else b.float().t()          # [K, N]
    res = (am @ bm) * alpha
    if out is None:
        return res.to(out_dtype)
    if accumulate:
        res = res + out.float()
    out.copy_(res.to(out.dtype))
    return out


def rmsnorm_fwd(x, w, eps, zero_centered=False, delta=None):
    """Returns (y, rstd); folds ``delta`` into ``x`` in place first when given."""
    if delta is not None:
        x.copy_((x.float() + delta.float()).to(x.dtype))
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(dim=-1) + eps)
    scale = (1.0 + w.float()) if zero_centered else w.float()
    y = (xf * rstd[:, None] * scale).to(x.dtype)
    return y, rstd


def rmsnorm_bwd(x, w, gy, rstd, zero_centered=False):
    """Returns (dx fp32, dw fp32)."""
    xf, gf = x.float(), gy.float()
    scale = (1.0 + w.float()) if zero_centered else w.float()
    xh = xf * rstd[:, None]
    gw = gf * scale
    mean = (gw * xh).mean(dim=-1, keepdim=True)
    dx = rstd[:, None] * (gw - xh * mean)
    dw = (gf * xh).sum(dim=0)
    return dx, dw


def rope_(buf, positions, col0, heads, dh, rot, theta, inverse=False):
    """In-place half-split rotary on columns [col0, col0 + heads*dh) of ``buf`` [T, C]."""
    T = buf.shape[0]
    half = rot // 2
    inv = theta ** (-torch.arange(0, half, dtype=torch.float32, device=buf.device) * 2.0 / rot)
    ang = positions.float()[:, None] * inv[None, :]
    cos, sin = ang.cos()[:, None, :], ang.sin()[:, None, :]
    if inverse:
        sin = -sin
    view = buf[:, col0:col0 + heads * dh].reshape(T, heads, dh)
    a = view[..., :half].float()
    b = view[..., half:rot].float()
    oa = a * cos - b * sin
    ob = b * cos + a * sin
    view = view.clone()
    view[..., :half] = oa.to(buf.dtype)
    view[..., half:rot] = ob.to(buf.dtype)
    buf[:, col0:col0 + heads * dh] = view.reshape(T, heads * dh)
    return buf


def swiglu_fwd(gu):
    F_ = gu.shape[-1] // 2
    g, u = gu[..., :F_], gu[..., F_:]
    return (F.silu(g.float()).to(gu.dtype).float() * u.float()).to(gu.dtype)


def swiglu_bwd(gu, dh):
    F_ = gu.shape[-1] // 2
    g, u, d = gu[..., :F_].float(), gu[..., F_:].float(), dh.float()
    sig = torch.sigmoid(g)
    dg = d * u * (sig * (1 + g * (1 - sig)))
    du = d * g * sig
    return torch.cat([dg, du], dim=-1).to(gu.dtype)


def embedding_fwd(ids, W):
    return W[ids.clamp(0, W.shape[0] - 1)]


def embedding_bwd(ids, g, dW):
    dW.index_add_(0, ids, g.to(dW.dtype))
    return dW


def cross_entropy_(logits, targets, weights, grad_scale=1.0, write_grad=True):
    """Weighted-sum cross entropy over a logits block; rewrites ``logits`` with
    its gradient when asked. Returns (loss_sum fp32 scalar, lse fp32[R])."""
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    V = logits.shape[-1]
    valid = (targets >= 0) & (targets < V)
    w = torch.ones_like(lse) if weights is None else weights.float()
    w = torch.where(valid, w, torch.zeros_like(w))
    tgt = targets.clamp(0, V - 1)
    picked = lf.gather(1, tgt[:, None])[:, 0]
    loss = (w * (lse - picked)).sum()
    if write_grad:
        p = torch.exp(lf - lse[:, None])
        p.scatter_add_(1, tgt[:, None], -torch.ones_like(picked)[:, None])
        logits.copy_((p * (w * grad_scale)[:, None]).to(logits.dtype))
    return loss, lse


def clipped_policy_(logits, targets, weights, old_logp, advantage, clip, ref_logp=None,
                    ref_beta=0.0, grad_scale=1.0, write_grad=True):
    """Weighted-sum clipped policy objective over a logits block (autograd-derived
    gradient written in place). Returns (loss_sum, logp[R])."""
    lf = logits.float().detach().requires_grad_(write_grad)
    V = logits.shape[-1]
    valid = (targets >= 0) & (targets < V)
    w = torch.ones(logits.shape[0], device=logits.device) if weights is None else weights.float()
    w = torch.where(valid, w, torch.zeros_like(w))
    tgt = targets.clamp(0, V - 1)
    logp = lf.gather(1, tgt[:, None])[:, 0] - torch.logsumexp(lf, dim=-1)
    r = torch.exp(logp - old_logp.float())
    A = advantage.float()
    per = -torch.minimum(r * A, r.clamp(1 - clip, 1 + clip) * A)
    if ref_logp is not None:
        d = ref_logp.float() - logp
        per = per + ref_beta * (torch.exp(d) - d - 1)
    loss = (w * per).sum()
    if write_grad:
        (g,) = torch.autograd.grad(loss * grad_scale, lf)
        logits.copy_(g.to(logits.dtype))
    return loss.detach(), logp.detach()


def adamw_(p, g, m, v, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """Round-to-nearest AdamW in fp32 math on tensors of any dtype (in place)."""
    gf = g.float() * grad_scale
    mf = beta1 * m.float() + (1 - beta1) * gf
    vf = beta2 * v.float() + (1 - beta2) * gf * gf
    b1 = 1 - beta1 ** step
    b2 = 1 - beta2 ** step
    pf = p.float() * (1 - lr * weight_decay)
    pf = pf - lr * (mf / b1) / ((vf / b2).sqrt() + eps)
    p.copy_(pf.to(p.dtype)); m.copy_(mf.to(m.dtype)); v.copy_(vf.to(v.dtype))


RULES = ("adamw", "sgd", "lion")


def update_rule_(rule, p, g, m, v, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """The update rules other than AdamW, in fp32 math with round-to-nearest stores, on tensors of
    any dtype and device (plain tensor operations: these are not hot paths).

    ``sgd``: momentum ``m <- beta1 m + g``, ``p <- p - lr (m + wd p)`` (``torch.optim.SGD`` with
    momentum ``beta1``, no dampening; the decay is added to the step, not to the gradient).
    ``lion``: ``u = sign(beta1 m + (1 - beta1) g)``, ``p <- p - lr (u + wd p)``,
    ``m <- beta2 m + (1 - beta2) g`` (Chen et al. 2023). ``v`` is not used by either."""
    if hasattr(rule, "apply"):
        # the update of a torch.optim optimizer captured as a graph (frontend/optimizer_capture.py);
        # its own hyperparameters are constants of that graph, the learning rate follows the run
        return rule.apply(p, g, m, v, lr=lr, step=step, grad_scale=grad_scale)
    if rule == "adamw":
        return adamw_(p, g, m, v, lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=weight_decay,
                      step=step, grad_scale=grad_scale)
    gf = g.float() * grad_scale
    pf, mf = p.float(), m.float()
    if rule == "sgd":
        mf = beta1 * mf + gf
        pf = pf - lr * (mf + weight_decay * pf)
    elif rule == "lion":
        u = torch.sign(beta1 * mf + (1 - beta1) * gf)
        pf = pf - lr * (u + weight_decay * pf)
        mf = beta2 * mf + (1 - beta2) * gf
    else:
        raise ValueError(f"unknown update rule {rule!r}; known: {RULES}")
    p.copy_(pf.to(p.dtype)); m.copy_(mf.to(m.dtype))


def attention_varlen(q, k, v, cu_seqlens, scale=None):
    """Packed causal GQA: q [T,Hq,dh], k/v [T,Hkv,dh]; each [cu[i],cu[i+1]) is its
    own causal sequence. Returns (out [T,Hq,dh], lse fp32 [Hq,T])."""
    T, Hq, dh = q.shape
    Hkv = k.shape[1]
    rep = Hq // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(dh)
    out = torch.zeros_like(q)
    lse = torch.full((Hq, T), float("-inf"), dtype=torch.float32, device=q.device)
    bounds = cu_seqlens.tolist()
    for s, e in zip(bounds[:-1], bounds[1:]):
        if e <= s:
            continue
        qs = q[s:e].float().transpose(0, 1)                               # [Hq, L, dh]
        ks = k[s:e].float().transpose(0, 1).repeat_interleave(rep, dim=0)
        vs = v[s:e].float().transpose(0, 1).repeat_interleave(rep, dim=0)
        sc = (qs @ ks.transpose(1, 2)) * scale
        L = e - s
        mask = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
        sc = sc.masked_fill(~mask, float("-inf"))
        lse[:, s:e] = torch.logsumexp(sc, dim=-1)
        out[s:e] = (torch.softmax(sc, dim=-1) @ vs).transpose(0, 1).to(q.dtype)
    return out, lse


def attention_varlen_bwd(q, k, v, out, lse, dout, cu_seqlens, scale=None):
    """Returns (dq, dk, dv) in the input dtypes."""
    T, Hq, dh = q.shape
    Hkv = k.shape[1]
    rep = Hq // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(dh)
    dq = torch.zeros_like(q); dk = torch.zeros_like(k); dv = torch.zeros_like(v)
    bounds = cu_seqlens.tolist()
    for s, e in zip(bounds[:-1], bounds[1:]):
        if e <= s:
            continue
        L = e - s
        qs = q[s:e].float().transpose(0, 1)
        ks = k[s:e].float().transpose(0, 1).repeat_interleave(rep, dim=0)
        vs = v[s:e].float().transpose(0, 1).repeat_interleave(rep, dim=0)
        do = dout[s:e].float().transpose(0, 1)
        o = out[s:e].float().transpose(0, 1)
        sc = (qs @ ks.transpose(1, 2)) * scale
        mask = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
        sc = sc.masked_fill(~mask, float("-inf"))
        p = torch.exp(sc - lse[:, s:e, None])
        dvs = p.transpose(1, 2) @ do
        dp = do @ vs.transpose(1, 2)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        dqs = ds @ ks
        dks = ds.transpose(1, 2) @ qs
        dq[s:e] = dqs.transpose(0, 1).to(q.dtype)
        dk[s:e] = dks.reshape(Hkv, rep, L, dh).sum(1).transpose(0, 1).to(k.dtype)
        dv[s:e] = dvs.reshape(Hkv, rep, L, dh).sum(1).transpose(0, 1).to(v.dtype)
    return dq, dk, dv


def l2_normalize(x, eps=1e-6):
    xf = x.float()
    return (xf * torch.rsqrt(xf.square().sum(-1, keepdim=True) + eps)).to(x.dtype)


def gated_delta_rule(q, k, v, beta, g, cu_seqlens):
    """Token-by-token gated delta rule (the recurrence the chunked kernel must
    match). q,k [T,Hk,dk] (already L2-normalised), v [T,Hv,dv], beta,g [T,Hv];
    g is the log-decay (<= 0). QK heads are repeat-interleaved to V heads.
    Returns out [T,Hv,dv] in v.dtype."""
    T, Hk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    rep = Hv // Hk
    qf = q.float().repeat_interleave(rep, dim=1) * dk ** -0.5
    kf = k.float().repeat_interleave(rep, dim=1)
    vf, bf, gf = v.float(), beta.float(), g.float()
    out = torch.zeros(T, Hv, dv, dtype=torch.float32, device=q.device)
    bounds = cu_seqlens.tolist()
    for s, e in zip(bounds[:-1], bounds[1:]):
        S = torch.zeros(Hv, dk, dv, dtype=torch.float32, device=q.device)
        for t in range(s, e):
            S = S * torch.exp(gf[t])[:, None, None]
            u = bf[t][:, None] * (vf[t] - torch.einsum("hk,hkv->hv", kf[t], S))
            S = S + kf[t][:, :, None] * u[:, None, :]
            out[t] = torch.einsum("hk,hkv->hv", qf[t], S)
    return out.to(v.dtype)


def causal_conv_silu(x, w, cu_seqlens):
    """Depthwise causal conv1d (kernel K) + SiLU over packed sequences.
    x [T,C], w [C,K]; the window never crosses a sequence boundary."""
    T, C = x.shape
    K = w.shape[1]
    out = torch.zeros_like(x)
    bounds = cu_seqlens.tolist()
    for s, e in zip(bounds[:-1], bounds[1:]):
        if e <= s:
            continue
        seg = x[s:e].float().t()[None]                       # [1, C, L]
        y = F.conv1d(F.pad(seg, (K - 1, 0)), w.float()[:, None, :], groups=C)[0].t()
        out[s:e] = F.silu(y).to(x.dtype)
    return out


def router_topk(logits, top_k, renormalize=True):
    """top-k then softmax over the selected logits (Qwen-MoE convention).
    Returns (weights fp32 [T,k], ids int64 [T,k], counts int64 [E])."""
    vals, ids = torch.topk(logits.float(), top_k, dim=-1)
    if renormalize:
        w = torch.softmax(vals, dim=-1)
    else:
        w = torch.softmax(logits.float(), dim=-1).gather(1, ids)
    counts = torch.bincount(ids.reshape(-1), minlength=logits.shape[-1])
    return w, ids, counts


def expert_scores(logits, scoring):
    """Scores in the logits' precision: ``sigmoid``, or a softmax in which a row of -inf has scores of zero."""
    if scoring == "sigmoid":
        return torch.sigmoid(logits)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    return e / e.sum(-1, keepdim=True).clamp(min=1.0)


def select_experts(logits, k, scoring="softmax", bias=None, groups=1, keep_groups=1, renormalize=True, scale=1.0):
    """Definition of :func:`..routing.select_experts`: keys in 64 bits, ties to the lowest index, experts without a
    comparable key last. Returns (ids int32 [T,k], weights fp32 [T,k], counts int32 [E])."""
    T, E = logits.shape
    x = logits.double()
    s = expert_scores(x, scoring)
    key = x if bias is None and groups == 1 else s if bias is None else s + bias.double()
    key = torch.where(torch.isnan(key), torch.full_like(key, float("-inf")), key)
    if groups > 1:
        g = key.view(T, groups, E // groups)
        best = torch.sort(g, dim=-1, descending=True).values[..., :2].sum(-1)
        best = torch.where(torch.isnan(best), torch.full_like(best, float("-inf")), best)        # inf - inf
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :keep_groups]
        drop = torch.ones(T, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, False)
        key = g.masked_fill(drop[..., None], float("-inf")).reshape(T, E)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if renormalize:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    counts = torch.zeros(E, dtype=torch.int32, device=x.device)
    counts.index_add_(0, ids.reshape(-1), torch.ones(T * k, dtype=torch.int32, device=x.device))
    return ids.to(torch.int32), (w * scale).float(), counts


def select_experts_bwd(logits, ids, dweights, scoring="softmax", renormalize=True, scale=1.0):
    """Gradient of the weights of :func:`select_experts` with respect to the logits, the picks held fixed."""
    s = expert_scores(logits.double(), scoring)
    at = ids.long()
    c, dw = s.gather(1, at), dweights.double()
    dc = scale * dw
    if renormalize:
        total = c.sum(-1, keepdim=True) + 1e-20
        dc = (dc - (dc * c / total).sum(-1, keepdim=True)) / total
    wide = torch.zeros_like(s).scatter_(1, at, dc * c * (1 - c) if scoring == "sigmoid" else dc)
    dx = wide if scoring == "sigmoid" else s * (wide - (dc * c).sum(-1, keepdim=True))
    return dx.to(logits.dtype)


PREFERENCE_KINDS = ("sigmoid", "hinge", "ipo")


def preference_terms(sums, beta, kind, label_smoothing):
    """Loss of each pair and its derivative by ``sums[2i]`` (that by ``sums[2i + 1]`` is the negative), from the
    sequences' log ratios."""
    z = beta * (sums[0::2] - sums[1::2])
    if kind == "sigmoid":
        loss = (1 - label_smoothing) * F.softplus(-z) + label_smoothing * F.softplus(z)
        slope = beta * (label_smoothing - torch.sigmoid(-z))
    elif kind == "hinge":
        loss, slope = torch.relu(1 - z), torch.where(z < 1, -beta, 0.0).to(z.dtype)
    else:
        gap = sums[0::2] - sums[1::2] - 1 / (2 * beta)
        loss, slope = gap * gap, 2 * gap
    return loss, slope


def preference_(logits, targets, weights, cu_seqlens, beta, kind, label_smoothing, average, ref_logp, grad_scale, grad):
    """Paired preference loss over a logits block, sums and coefficients in 64 bits; ``grad`` (when given) receives the
    gradient. Returns (loss fp32 scalar, sums fp32[S], logp fp32[R])."""
    R, V = logits.shape
    f = logits.float()
    w = torch.ones(R, device=f.device) if weights is None else weights.float()
    valid = (targets >= 0) & (targets < V) & (w != 0)
    t = torch.where(valid, targets, torch.zeros_like(targets))[:, None]
    logp = torch.where(valid, f.gather(1, t)[:, 0] - torch.logsumexp(f, -1), torch.zeros_like(w))
    ratio = logp if ref_logp is None else logp - ref_logp.float()
    ratio = torch.where(valid, w * ratio, torch.zeros_like(w)).double()
    bounds = [min(max(int(c), 0), R) for c in cu_seqlens.tolist()]
    spans = [(a, max(a, b)) for a, b in zip(bounds[:-1], bounds[1:])]
    sums = torch.stack([ratio[a:b].sum() for a, b in spans]) if spans else ratio.new_zeros(0)
    mass = torch.stack([torch.where(valid, w, 0.0)[a:b].double().sum() for a, b in spans]) if spans else ratio.new_zeros(0)
    some = torch.tensor([bool(valid[a:b].any()) for a, b in spans], dtype=torch.bool, device=f.device)
    if average:
        sums = torch.where(mass != 0, sums / mass, torch.zeros_like(sums))
    loss, slope = preference_terms(sums, beta, kind, label_smoothing)
    live = some[0::2] & some[1::2]
    loss = torch.where(live, loss, torch.zeros_like(loss)).sum()
    if grad is not None:
        slope = torch.where(live, slope, torch.zeros_like(slope))
        coef = torch.zeros(R, dtype=torch.float64, device=f.device)
        for i, (a, b) in enumerate(spans):
            each = slope[i // 2] * (1 - 2 * (i % 2))
            if average:
                each = torch.where(mass[i] != 0, each / mass[i], torch.zeros_like(each))
            coef[a:b] = torch.where(valid[a:b], w[a:b].double() * each, 0.0)
        coef = (coef * grad_scale).float()
        onehot = torch.zeros_like(f).scatter_(1, t, 1.0)
        full = (onehot - torch.softmax(f, -1)) * coef[:, None]
        grad.copy_(torch.where(valid[:, None], full, torch.zeros_like(full)).to(grad.dtype))
    return loss.float(), sums.float(), logp


MOMENT_BLOCK = 256        # elements that share the exponent of an 8-bit moment


def moment_exponents(top):
    """Biased exponents of the smallest powers of two with ``top <= 448 * 2^(e - 127)``, 0 for blocks of zeros."""
    bits = top.contiguous().view(torch.int32)
    e = (bits >> 23) - torch.where((bits & 0x7fffff) > 0x600000, 7, 8)
    return torch.where(top > 0, e.clamp(1, 254), torch.zeros_like(e)).to(torch.uint8)


def moment_values(codes, exponents):
    """What 8-bit moments stand for, in fp32."""
    unit = torch.exp2(exponents.float() - 127.0).repeat_interleave(MOMENT_BLOCK)[:codes.numel()]
    return codes.float() * unit


def moment_codes(x, floor=False):
    """fp32 values -> (e4m3 codes, exponents); with ``floor`` a value that is not zero keeps a code that is not."""
    n = x.numel()
    blocks = F.pad(x, (0, -n % MOMENT_BLOCK)).view(-1, MOMENT_BLOCK)
    e = moment_exponents(torch.where(torch.isnan(blocks), 0.0, blocks.abs()).amax(1) if n else x.new_zeros(0))
    y = (blocks * torch.exp2(127.0 - e.float())[:, None]).reshape(-1)[:n]
    if floor:
        y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), e


def adamw8_(p, g, m, r, m_exp, r_exp, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """Round-to-nearest AdamW with 8-bit moments (in place): ``m`` and ``r``, the root of the second moment, as e4m3
    codes with an exponent per block. The moments' arithmetic is fp32, one rounding to an operation."""
    gf = g.float() * grad_scale
    mf = beta1 * moment_values(m, m_exp) + (1 - beta1) * gf
    old = moment_values(r, r_exp)
    rf = torch.sqrt(beta2 * (old * old) + (1 - beta2) * gf * gf)
    pf = p.float() * (1 - lr * weight_decay)
    pf = pf - lr * (mf / (1 - beta1 ** step)) / (rf / math.sqrt(1 - beta2 ** step) + eps)
    p.copy_(pf.to(p.dtype))
    for codes, exps, x, floor in ((m, m_exp, mf, False), (r, r_exp, rf, True)):
        c, e = moment_codes(x, floor)
        codes.copy_(c)
        exps.copy_(e)
