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
