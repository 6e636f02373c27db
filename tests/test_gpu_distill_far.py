"""GPU: the divergence from a teacher's best entries where numbers lie far apart or far from zero; bounds in distill_far.py."""
import numpy as np
import pytest

from distill_far import rows_of
from logits_cases import EPS, TINY, make_distill

pytestmark = pytest.mark.gpu

# G = 16 lanes, one wave, one wave with a longer row, several waves, split rows, rows beyond the registers
SHAPES = [(4, 64, 3), (5, 1003, 20), (5, 6001, 20), (260, 9001, 40), (3, 50001, 20), (257, 70001, 20)]


def _grads(z, ids, t, T, kind):
    """The gradient of the rows' sum and the rows' losses by value + gradient, value alone and autograd"""
    import torch
    import flowrl_hip as fh
    kw = dict(kind=kind, temperature=T, reduction="none")
    args = (torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda())
    zc = z.cuda()
    rows, grad = fh.logits.distill_loss(zc, *args, want_grad=True, **kw)
    value = fh.logits.distill_loss(zc, *args, **kw)
    leaf = zc.clone().requires_grad_(True)
    out = fh.autograd.distill_loss(leaf, *args, **kw)
    back, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    return (rows, value, out.detach()), (grad, back)


def _check_gradients(grads, pick, g, tolg):
    for got in grads:
        half, tiny = EPS[got.dtype], TINY[got.dtype]
        a = got[pick].double().cpu().numpy()
        bad = ~(np.abs(a - g) <= tolg + half * (np.abs(g) + tolg) + tiny)
        assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[:3].tolist()}: {a[bad][:3]} vs {g[bad][:3]}"


def _picked(N):
    return sorted({0, 1, 2, N // 2, N - 1})


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("fill", [-1e9, -1e10, -1e20, -1e30, -3.4e38, 1e10, 1e30])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_gradient_of_students_far_from_zero(N, V, K, fill, kind):
    """A row of one value throughout is uniform; a row with a level far below keeps its gradient on the others."""
    import torch
    rng = np.random.default_rng(V)
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, t = make_distill(rng, N, V, K, kind, dtype)
        level = torch.tensor(max(fill, torch.finfo(dtype).min)).to(dtype)       # -3.4e38 is no bfloat16 number but -inf
        z[0], z[1, ::2] = level, level
        pick = _picked(N)
        _, g, _, tolg = rows_of(z[pick], ids[pick], t[pick], kind, 1.0)
        losses, grads = _grads(z, ids, t, 1.0, kind)
        _check_gradients(grads, pick, g, tolg)


@pytest.mark.parametrize("kind", ["logits"])
@pytest.mark.parametrize("T", [1e-30, 1e-9, 1e-6, 1e-3, 1e6, 1e30])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_gradient_over_the_temperatures(N, V, K, T, kind):
    """From the argmax alone to the uniform distribution."""
    import torch
    rng = np.random.default_rng(V + 1)
    T = float(np.float32(T))
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, t = make_distill(rng, N, V, K, kind, dtype)
        pick = _picked(N)
        _, g, _, tolg = rows_of(z[pick], ids[pick], t[pick], kind, T)
        losses, grads = _grads(z, ids, t, T, kind)
        _check_gradients(grads, pick, g, tolg)
