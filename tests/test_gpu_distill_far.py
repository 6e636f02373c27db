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


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
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


def _check_losses(losses, pick, L, tolL):
    for got in losses:
        a = got[pick].double().cpu().numpy()
        assert (np.abs(a - L) <= tolL + 2.0 ** -24 * np.abs(L)).all(), f"{a} vs {L}, bounds {tolL}"


@pytest.mark.parametrize("fill", [-1e5, -1e9, -1e20, -3.4e38, 1e5, 1e10, 1e30])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_loss_of_students_far_from_zero(N, V, K, fill):
    """The divergence depends on differences of logits only: the same for a row of 1e30 as for a row of 0."""
    import torch
    rng = np.random.default_rng(V + 2)
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, t = make_distill(rng, N, V, K, "logits", dtype)
        level = torch.tensor(max(fill, torch.finfo(dtype).min)).to(dtype)
        z[0] = level
        z[1] = level
        z[1, ids[1]] = 2 * level if fill > 0 else level / 2      # named entries ahead of the others by more than an exponential spans
        pick = _picked(N)
        L, _, tolL, _ = rows_of(z[pick], ids[pick], t[pick], "logits", 1.0)
        losses, _ = _grads(z, ids, t, 1.0, "logits")
        _check_losses(losses, pick, L, tolL)
        # the rest as a class, of a row that its rules leave uniform
        u = torch.log_softmax(torch.from_numpy(t).double(), 1).add(np.log(0.7)).float().numpy()
        L, _, tolL, _ = rows_of(z[:1], ids[:1], u[:1], "logprobs", 1.0)
        losses, _ = _grads(z, ids, u, 1.0, "logprobs")
        _check_losses(losses, [0], L, tolL)


@pytest.mark.parametrize("T", [1e-30, 1e-9, 1e-6, 1e-3, 1e6, 1e30])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_loss_over_the_temperatures(N, V, K, T):
    """A teacher whose best entry is the student's: at small temperatures both are certain of it, and the divergence is what their doubts differ by."""
    import torch
    rng = np.random.default_rng(V + 3)
    T = float(np.float32(T))
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, t = make_distill(rng, N, V, K, "logits", dtype)
        best, mine = z.float().argmax(1).numpy(), t.argmax(1)
        keep = ~(ids == best[:, None]).any(1)
        ids[keep, mine[keep]] = best[keep]
        pick = _picked(N)
        L, _, tolL, _ = rows_of(z[pick], ids[pick], t[pick], "logits", T)
        losses, _ = _grads(z, ids, t, T, "logits")
        _check_losses(losses, pick, L, tolL)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("gap", [60.0, 100.0, 1e4])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_a_rest_far_below(N, V, K, gap, dtype):
    """The teacher's unnamed mass is a class of its own, of which a student that is sure of the named entries keeps e^-gap: its divergence is near
    P gap and the rest's gradient is minus the rest's own distribution times P, with numbers throughout."""
    import torch
    rng = np.random.default_rng(V + 4)
    z, ids, t = make_distill(rng, N, V, K, "logprobs", getattr(torch, dtype), ragged=True)
    r = np.arange(N)
    z[0, ids[0, 0]] += gap                               # one named entry is ahead
    named = np.zeros((N, V), bool)
    for k in range(K):
        ok = (ids[:, k] >= 0) & (ids[:, k] < V)
        named[r[ok], ids[ok, k]] = True
    z[1:][torch.from_numpy(named[1:])] += gap            # all of them are
    z[2][torch.from_numpy(~named[2])] = -gap             # the rest is one masked level
    z[N - 1][torch.from_numpy(~named[N - 1] & (rng.random(V) < 0.5))] = float("-inf")
    if N > 3:
        t[N // 2] += 1.0 - np.log(np.exp(t[N // 2].astype(np.float64)).sum())       # names more than all there is: no rest
    for T in (1.0, 0.5):
        pick = _picked(N)
        L, g, tolL, tolg = rows_of(z[pick], ids[pick], t[pick], "logprobs", T)
        assert np.isfinite(L).all()
        losses, grads = _grads(z, ids, t, T, "logprobs")
        _check_losses(losses, pick, L, tolL)
        _check_gradients(grads, pick, g, tolg)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_a_rest_of_nothing(N, V, K, dtype):
    """Mass that is left where the student has none, neither below nor beside what is named: an infinite divergence, gradients that are numbers, 0 at
    the entries that are ruled out."""
    import torch
    rng = np.random.default_rng(V + 5)
    z, ids, t = make_distill(rng, N, V, K, "logprobs", getattr(torch, dtype))
    named = torch.zeros((N, V), dtype=torch.bool).scatter_(1, torch.from_numpy(ids).long(), True)
    z[1][~named[1]] = float("-inf")
    pick = _picked(N)
    L, g, tolL, tolg = rows_of(z[pick], ids[pick], t[pick], "logprobs", 1.0)
    losses, grads = _grads(z, ids, t, 1.0, "logprobs")
    for got in losses:
        assert float(got[1]) == float("inf") and torch.isfinite(got[torch.arange(N, device="cuda") != 1]).all()
    _check_gradients(grads, pick, g, tolg)
    assert not any(got[1].cpu()[~named[1]].any() for got in grads)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("skip,gap", [(0, 0), (1, 2), (3, 1), (7, 4)])
@pytest.mark.parametrize("N,V", [(4, 61), (5, 1003), (260, 9001), (3, 50001), (257, 70001)])
def test_named_ends_and_repeats_far_above_the_rest(N, V, skip, gap, dtype):
    """Rows that start anywhere: the single entries before and behind the vectors are named, some of them twice, and lie far above the rest."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V + skip)
    K, dt = 24, getattr(torch, dtype)
    z, ids, t = make_distill(rng, N, V, K, "logprobs", dt, repeats=True)
    ids[:, :8] = np.arange(8)
    ids[:, 8:16] = V - 1 - np.arange(8)
    ids[:, 16:18] = [0, V - 1]
    t -= 1.0                                             # a token named several times counts as often: mass is left all the same
    z.scatter_(1, torch.from_numpy(ids).long(), torch.from_numpy((200.0 + rng.standard_normal((N, K))).astype(np.float32)).to(dt))
    buf = torch.zeros((N * (V + gap) + skip,), dtype=dt, device="cuda")
    view = buf[skip:].view(N, V + gap)[:, :V]
    view.copy_(z)
    pick = _picked(N)
    L, g, tolL, tolg = rows_of(z[pick], ids[pick], t[pick], "logprobs", 1.0)
    args = (torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda())
    kw = dict(kind="logprobs", reduction="none")
    rows, grad = fh.logits.distill_loss(view, *args, want_grad=True, **kw)
    value = fh.logits.distill_loss(view, *args, **kw)
    leaf = view.detach().requires_grad_(True)
    out = fh.autograd.distill_loss(leaf, *args, **kw)
    back, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    _check_losses((rows, value, out.detach()), pick, L, tolL)
    _check_gradients((grad, back), pick, g, tolg)
