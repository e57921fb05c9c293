"""The paired preference loss on the GPU against its definition in 64 bits."""
import pytest
import torch

from shadowspill_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _case(V, bounds, rows, dtype=torch.bfloat16, seed=0, masked=0.3, wide=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, V, generator=g, device=DEV) * 2
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    x.scatter_add_(1, t[:, None], torch.full((rows, 1), 4.0, device=DEV))
    full = torch.empty(rows, V + wide, dtype=dtype, device=DEV)
    full[:, :V] = x
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    w[torch.rand(rows, generator=g, device=DEV) < masked] = 0.0
    ref = torch.randn(rows, generator=g, device=DEV) - 3.0
    return full[:, :V], t, w, torch.tensor(bounds, dtype=torch.int32, device=DEV), ref


def _exact(x, t, w, cu, beta=0.1, kind="sigmoid", label_smoothing=0.0, average=False, ref_logp=None, grad_scale=1.0):
    """(loss, sums, softmax, dloss / dlogp per row, masses of the sums' errors) in 64 bits, derivatives by autograd."""
    V = x.shape[1]
    w = torch.ones(x.shape[0], device=DEV) if w is None else w
    ok = (t >= 0) & (t < V) & (w != 0)
    p = torch.log_softmax(torch.where(ok[:, None], x.double(), 0.0), 1)      # what is masked may hold anything
    lp = p.gather(1, torch.where(ok, t, 0)[:, None])[:, 0].requires_grad_(True)
    ratio = lp if ref_logp is None else lp - torch.where(ok, ref_logp, 0.0).double()
    wd = torch.where(ok, w.double(), 0.0)
    sums, sizes, some = [], [], []
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        m = wd[a:b].sum() if average and bool(ok[a:b].any()) else 1.0
        sums.append((wd * ratio)[a:b].sum() / m)
        sizes.append(float(wd[a:b].abs().sum() / m))
        some.append(bool(ok[a:b].any()))
    loss = lp.sum() * 0
    for i in range(len(sums) // 2):
        if some[2 * i] and some[2 * i + 1]:
            d = sums[2 * i] - sums[2 * i + 1]
            if kind == "sigmoid":
                soft = torch.nn.functional.softplus
                loss = loss + (1 - label_smoothing) * soft(-beta * d) + label_smoothing * soft(beta * d)
            elif kind == "hinge":
                loss = loss + torch.relu(1 - beta * d)
            else:
                loss = loss + (d - 1 / (2 * beta)) ** 2
    slope = torch.autograd.grad(loss * grad_scale, lp)[0]
    return (loss.detach(), torch.stack(sums).detach() if sums else torch.zeros(0, device=DEV, dtype=torch.float64), p.exp(), slope,
            torch.tensor(sizes, device=DEV, dtype=torch.float64))


def _compare(x, t, w, cu, **kw):
    V, R = x.shape[1], x.shape[0]
    before = x.clone()
    loss, sums, grad = torch.full((1,), 0.25, device=DEV), torch.full((cu.numel() - 1,), 9.0, device=DEV), torch.full_like(x, 7.0)
    F.preference_(x, t, w, cu, loss, grad=grad, sums=sums, **kw)
    want_loss, want_sums, p, slope, sizes = _exact(before, t, w, cu, **kw)
    onehot = torch.zeros_like(p).scatter_(1, torch.where((t >= 0) & (t < V), t, 0)[:, None], 1.0)
    want = slope[:, None] * (onehot - p)
    # A row's log-probability: __expf of -y has at most 2 + 1.173 y steps of 2 U, and its share of the sum falls as e^-y, so the sum is
    # off by at most 2 + 1.173 * 24 of them and e^-24 V; a thread adds V / 512 + 16 terms, 9 levels follow; logarithm and two
    # differences round values up to the largest finite logit and log V + 24 once each.
    finite = torch.where(torch.isfinite(before.float()), before.float().abs(), 0.0)
    big = float(finite.max()) + 24 + 12 if R else 0.0
    row = (2 * (2 + 1.173 * 24) + V / 512 + 25 + 3 * big) * U
    refs = 0.0 if kw.get("ref_logp") is None else float(kw["ref_logp"].nan_to_num(0, 0, 0).abs().max())
    off = sizes * (row + 3 * U * (refs + big)) + 2 * U * want_sums.abs()
    assert bool(((sums - want_sums).abs() <= off).all())
    beta, kind = kw.get("beta", 0.1), kw.get("kind", "sigmoid")
    d = want_sums[0::2] - want_sums[1::2]
    pair = off[0::2] + off[1::2]
    # |f'| and, relative to f', |f''| by the margin
    steep, bend = (2 * (d - 0.5 / beta).abs() + pair, 1 / (d - 0.5 / beta).abs()) if kind == "ipo" else (beta, beta)
    assert abs(float(loss) - 0.25 - float(want_loss)) <= float((steep * pair).sum()) + 4 * U * (float(want_loss) + 0.25)
    rel = float((pair * bend).max()) + 8 * U if pair.numel() else 0.0
    share = (2 * (2 + 1.173 * (2 * big)) + 4) * U + row          # of a probability: its own __expf, and the lse's error
    half = torch.finfo(x.dtype).eps / 2
    allowed = (rel + half) * want.abs() + slope.abs()[:, None] * (p * share + 4 * U) + 1e-37
    assert bool(((grad.double() - want).abs() <= allowed).all())
    x2, loss2 = before.clone(), torch.full((1,), 0.25, device=DEV)
    F.preference_(x2, t, w, cu, loss2, **kw)                      # over the logits: the same bits
    assert torch.equal(x2, grad) and torch.equal(loss2, loss)
    loss3, logp = torch.full((1,), 0.25, device=DEV), torch.empty(R, device=DEV)
    F.preference_(x, t, w, cu, loss3, write_grad=False, logp=logp, **kw)
    assert torch.equal(loss3, loss) and torch.equal(x.view(torch.int32 if x.dtype == torch.float32 else torch.int16),
                                                    before.view(torch.int32 if x.dtype == torch.float32 else torch.int16))
    return loss, sums, grad, logp


@pytest.mark.parametrize("V", [1, 7, 1000, 4096, 32003])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("sigmoid", True), ("hinge", False), ("ipo", True)])
def test_loss_sums_and_gradient(V, dtype, kind, average):
    x, t, w, cu, ref = _case(V, [0, 11, 30, 31, 45], 50, dtype, seed=V)
    _compare(x, t, w, cu, kind=kind, average=average, ref_logp=ref, beta=0.3)


@pytest.mark.parametrize("options", [dict(label_smoothing=0.2), dict(beta=2.5), dict(grad_scale=0.125), dict(ref_logp=None)])
def test_options(options):
    x, t, w, cu, ref = _case(512, [0, 20, 33, 70, 100, 101, 120], 120, seed=1)
    _compare(x, t, w, cu, **{"ref_logp": ref, **options})
    _compare(x, t, None, cu, **{"ref_logp": ref, **options})


@pytest.mark.parametrize("bounds", [[0], [0, 0, 0], [0, 0, 9], [0, 9, 9], [3, 9, 20], [0, 1, 2], [0, 5, 5, 5, 5, 5, 30], [40, 40, 40],
                                    [0, 40, 40, 40, 40]])
def test_empty_sides_and_rows_of_no_sequence(bounds):
    x, t, w, cu, ref = _case(300, bounds, 40, seed=2, masked=0.0)
    loss, sums, grad, _ = _compare(x, t, w, cu, ref_logp=ref)
    covered = torch.zeros(40, dtype=torch.bool, device=DEV)
    for i in range((len(bounds) - 1) // 2):
        a, b, c = bounds[2 * i:2 * i + 3]
        if b > a and c > b:
            covered[a:c] = True
    assert float(grad[~covered].float().abs().sum()) == 0.0
    assert bool((grad[covered].float().abs().sum(1) > 0).all())
    if not bool(covered.any()):
        assert float(loss) == 0.25


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("by", ["weight", "target", "beyond"])
def test_masked_rows_may_hold_anything(bad, by):
    x, t, w, cu, ref = _case(1000, [0, 20, 44], 50, seed=3, masked=0.0)
    rows = torch.tensor([0, 7, 25, 49], device=DEV)
    x[rows] = bad
    ref[rows] = bad
    if by == "weight":
        w[rows] = 0.0
    else:
        t[rows] = -100 if by == "target" else 1000
    _, _, grad, logp = _compare(x, t, w, cu, ref_logp=ref)
    assert float(grad[rows].float().abs().sum()) == 0.0 and float(logp[rows].abs().sum()) == 0.0


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.bfloat16).min])
def test_masked_vocabulary(low):
    x, t, w, cu, ref = _case(1024, [0, 20, 44], 44, seed=4, masked=0.0)
    keep = torch.zeros_like(x, dtype=torch.bool).scatter_(1, t[:, None], True)
    keep[:, 900:930] = True
    x[~keep] = low
    x[5] = low
    x[5, t[5]] = 1.0                                              # one word is left
    loss, _, grad, logp = _compare(x, t, w, cu, ref_logp=ref)
    # its probability is one exponential over itself: the exponential is off by at most 2^-22.7, quotient, logarithm and product by
    # less than 2^-23 together, and its coefficient is at most 0.1 (beta) * 1.5 (its weight)
    assert abs(float(logp[5])) <= 2.0 ** -21 and float(grad[5].float().abs().max()) <= 0.15 * 2.0 ** -21
    assert float(grad[~keep].float().abs().sum()) == 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [-3e38, -1e30, -1e5, -65000.0, 65000.0, 1e5, 1e30, 3e38])
def test_logits_far_from_zero(shift, dtype):
    """Rows around any level, in range of the type: few values, so that words tie at the top."""
    x, t, w, cu, ref = _case(5000, [0, 20, 44], 44, torch.float32, seed=12, masked=0.0)
    step = abs(shift) * 2.0 ** -7
    x = (shift + torch.round(x) * step * (x.abs() > 7)).to(dtype)
    _compare(x, t, w, cu, ref_logp=ref * 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wide,skip", [(8, 0), (5, 0), (8, 3), (5, 1)])
def test_strided_and_unaligned_logits(dtype, wide, skip):
    x, t, w, cu, ref = _case(1000 + skip, [0, 20, 44], 50, dtype, seed=5, wide=wide)
    x, t = x[:, skip:], t.clamp(max=999)
    want = x.contiguous().clone()
    _compare(x, t, w, cu, ref_logp=ref)
    a, b = torch.zeros(1, device=DEV), torch.zeros(1, device=DEV)
    F.preference_(x, t, w, cu, a, ref_logp=ref)
    F.preference_(want, t, w, cu, b, ref_logp=ref)
    assert float(a) == pytest.approx(float(b), rel=1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [3, 9, 17, 130, 1001, 4110, 50257])
def test_bits_do_not_depend_on_where_rows_lie(V, dtype):
    x, t, w, cu, ref = _case(V, [0, 9, 20], 21, dtype, seed=V, masked=0.1)
    t[:8] = torch.tensor([0, V - 1, min(7, V - 1), min(8, V - 1), max(V - 2, 0), V // 2, min(1, V - 1), max(V - 9, 0)], device=DEV)
    rows = []
    pitch = -(-V // 8) * 8
    for skip in range(8):
        buffer = torch.full((21 * pitch + 24,), 5.0, dtype=dtype, device=DEV)
        for wide in (V, pitch):
            at = torch.as_strided(buffer, (21, V), (wide, 1), skip)
            at.copy_(x)
            loss, logp = torch.zeros(1, device=DEV), torch.empty(21, device=DEV)
            other = torch.empty(21, V, dtype=dtype, device=DEV)
            F.preference_(at, t, w, cu, loss, ref_logp=ref, logp=logp, grad=other)
            F.preference_(at, t, w, cu, loss, ref_logp=ref, logp=logp)
            rows.append((loss, logp, at.clone(), other))
            around = torch.ones_like(buffer, dtype=torch.bool)
            torch.as_strided(around, (21, V), (wide, 1), skip).fill_(False)
            assert bool((buffer[around] == 5.0).all())            # what lies between and around the rows is left as it was
            buffer.fill_(5.0)
    for got in rows:
        assert all(torch.equal(a, b) for a, b in zip(got, rows[0])) and torch.equal(got[2], got[3])


def test_saturated_margins_and_hinge_without_loss():
    x, t, w, cu, _ = _case(600, [0, 30, 60, 90, 120], 120, torch.float32, seed=6, masked=0.0)
    for far in (-60.0, 60.0):                                    # the reference far off: z near +-100
        ref = torch.where(torch.arange(120, device=DEV) % 60 < 30, far, 0.0)
        for kind in ("sigmoid", "hinge", "ipo"):
            loss, _, grad, _ = _compare(x, t, w, cu, kind=kind, ref_logp=ref, beta=0.05)
            assert bool(torch.isfinite(grad).all()) and bool(torch.isfinite(loss).all())


def test_many_pairs_one_long_sequence_and_repeatable_bits():
    bounds = list(range(0, 601, 1))                              # 300 pairs of single tokens
    x, t, w, cu, ref = _case(256, bounds, 600, seed=7, masked=0.1)
    first = _compare(x, t, w, cu, ref_logp=ref)
    again = _compare(x, t, w, cu, ref_logp=ref)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    x, t, w, cu, ref = _case(64, [0, 9000, 9001], 9001, seed=8, masked=0.0)
    _compare(x, t, w, cu, ref_logp=ref, average=True)


@pytest.mark.parametrize("V", [40, 3000])
@pytest.mark.parametrize("pairs,most", [(16, 3), (513, 4), (5000, 2), (1, 40)])
def test_pairs_by_the_hundred_with_empty_sides(pairs, most, V):
    g = torch.Generator().manual_seed(pairs)
    lengths = torch.randint(0, most + 1, (2 * pairs,), generator=g)
    lengths[2:4] = 0                                              # a pair without rows
    bounds = [0, *lengths.cumsum(0).tolist()]
    x, t, w, cu, ref = _case(V, bounds, bounds[-1] + 3, seed=14, masked=0.1)
    _compare(x, t, w, cu, ref_logp=ref, average=True)


def test_rows_that_overlap_are_refused():
    x, t, w, cu, ref = _case(64, [0, 4, 8], 8, seed=15)
    loss = torch.zeros(1, device=DEV)
    for bad in (dict(logits=x[:1].expand(8, 64)), dict(grad=x[:1].expand(8, 64)), dict(logits=x.t().contiguous().t())):
        with pytest.raises(ValueError):
            F.preference_(**{**dict(logits=x, targets=t, weights=w, cu_seqlens=cu, loss_sum=loss), **bad})
    assert float(loss) == 0.0


def test_two_streams_at_once():
    cases = [_case(2000, [0, 300, 640], 640, seed=s) for s in (16, 17)]
    want = [_compare(x, t, w, cu, ref_logp=ref) for x, t, w, cu, ref in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[] for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (x, t, w, cu, ref) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                loss, grad = torch.full((1,), 0.25, device=DEV), torch.empty_like(x)
                F.preference_(x, t, w, cu, loss, grad=grad, ref_logp=ref)
                got[i].append((loss, grad))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(loss, want[i][0]) and torch.equal(grad, want[i][2]) for loss, grad in got[i])


def test_gradient_against_differences():
    x, t, w, cu, ref = _case(40, [0, 5, 9, 12, 20], 20, torch.float32, seed=9)
    grad = torch.empty_like(x)
    F.preference_(x, t, w, cu, torch.zeros(1, device=DEV), grad=grad, ref_logp=ref, beta=0.4, label_smoothing=0.1)
    g = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(5):
        d = torch.randn(x.shape, generator=g, device=DEV, dtype=torch.float64)
        up, down = (_exact(x.double() + s * 1e-5 * d, t, w, cu, beta=0.4, label_smoothing=0.1, ref_logp=ref)[0] for s in (1, -1))
        # central differences of a smooth loss: h^2 / 6 times a third derivative of a few units along d, far under the fp32
        # rounding of 800 products (2^-22 of their sum of magnitudes)
        assert abs(float((grad.double() * d).sum()) - float(up - down) / 2e-5) <= 2.0 ** -20 * float((grad.double() * d).abs().sum()) + 1e-7


def test_other_stream_and_replayed_graph():
    x, t, w, cu, ref = _case(2000, [0, 30, 64], 64, seed=10)
    loss, grad, sums = torch.zeros(1, device=DEV), torch.empty_like(x), torch.empty(2, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.preference_(x, t, w, cu, loss, grad=grad, sums=sums, ref_logp=ref)
    torch.cuda.current_stream().wait_stream(side)
    other, want = torch.zeros(1, device=DEV), torch.empty_like(x)
    F.preference_(x, t, w, cu, other, grad=want, ref_logp=ref)
    assert torch.equal(loss, other) and torch.equal(grad, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss.zero_()
        F.preference_(x, t, w, cu, loss, grad=grad, sums=sums, ref_logp=ref)
    x2 = _case(2000, [0, 30, 64], 64, seed=11)[0]
    x.copy_(x2)
    cu.copy_(torch.tensor([0, 10, 60], dtype=torch.int32))
    graph.replay()
    other.zero_()
    F.preference_(x, t, w, cu, other, grad=want, ref_logp=ref)
    assert torch.equal(loss, other) and torch.equal(grad, want)
