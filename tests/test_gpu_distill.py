"""GPU: frl_distill_fwd / frl_distill_bwd against the float64 restatement (oracle/logits_oracle.py) and against differences.  PARITY UNPINNED:
the reference has no such operator.

Tolerances count roundings.  Every logarithm of a row is a sum of a few float32 terms of the size of |z| / T, ln V and |log p|, each off by a few
times 2^-24 of itself, the log of the sum of exponentials by 2^-22 of the mean distance from the maximum: below 2^-21 A with
A = max |z| / T + ln V + max |log p| + 4 in all, and the loss is their mean under p.  A probability p = exp(d) / sum with d = (t - max) / T comes
from three roundings of d (the difference, 1 / T, their product), each 2^-24 |d|, and at most eight more (exponential, sum, quotient): its relative error
is below 2^-24 (3 |d| + 8), and |d| <= |log p| because the sum is at least 1.  In the loss that weighs E_p |d| <= E_p |log p| <= ln K
times |log p - log q| <= A: 2^-24 (3 ln K + 8) A more.  An element of the gradient is f (k q - p) with q off by 2^-22 (4 + m - z) of itself,
k by 2^-21 (1 + P / Q), p as above, f by 2^-22, and is rounded once to its type."""
import numpy as np
import pytest

import logits_oracle as orc
from logits_cases import EPS, TINY, make_distill

pytestmark = pytest.mark.gpu


def _expected(z, ids, t, kind, T):
    zn = z.double().numpy()
    rows = [orc.distill_row(zn[r], ids[r], t[r].astype(np.float64), kind, T) for r in range(len(zn))]
    L, g, q = (np.stack([x[i] for x in rows]) for i in range(3))
    tolL, tolg = np.zeros(len(rows)), np.zeros_like(g)
    for r, (_, _, qr, more) in enumerate(rows):
        y = zn[r] / T
        fin = np.isfinite(y)
        lp = more["logp"][np.isfinite(more["logp"])]
        far = np.abs(lp).max() if lp.size else 0.0
        tolL[r] = (2.0 ** -21 + 2.0 ** -24 * (3 * np.log(max(lp.size, 1)) + 8)) * (np.abs(y[fin]).max() + np.log(y.size) + far + 4)
        ratio = more["P"] / more["Q"] if more["P"] > 0 else 0.0
        p = np.abs(T * g[r]) + qr * (1 + ratio)            # no less than p and k q
        tolg[r] = (qr * (1 + ratio) * 2.0 ** -21 * (4 + np.where(fin, y.max() - y, 0.0)) + p * (2.0 ** -24 * (3 * far + 8) + 2.0 ** -22)) / T
    return L, g, tolL, tolg


def _close(grad, want, tol, scale):
    half, tiny = EPS[grad.dtype], TINY[grad.dtype]
    got = grad.double().cpu().numpy()
    want, tol = want * scale, tol * np.abs(scale)
    bad = ~(np.abs(got - want) <= tol + half * (np.abs(want) + tol) + tiny)
    assert not bad.any(), f"{bad.sum()} of {bad.size} elements, first at {np.argwhere(bad)[:3].tolist()}: {got[bad][:3]} vs {want[bad][:3]}"


CASES = [
    # N, V, K, ragged, repeats, wide
    (1, 1, 1, False, False, False),
    (3, 2, 2, False, False, True),
    (9, 50, 8, True, False, False),
    (67, 64, 64, False, False, False),          # every entry of the vocabulary is named
    (5, 1000, 130, True, True, True),
    (6, 1025, 20, False, False, False),
    (7, 8191, 64, True, False, False),
    (4, 8193, 1024, False, True, False),         # few rows: split over their length
    (3, 50001, 33, True, False, True),
    (260, 8197, 40, True, False, False),         # workgroups of 1024 threads
]


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("N,V,K,ragged,repeats,wide", CASES, ids=[f"{c[0]}x{c[1]}-top{c[2]}" for c in CASES])
def test_value_and_gradient(N, V, K, ragged, repeats, wide, kind):
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(N * 1009 + V)
    for dtype, T in ((torch.float32, 1.0), (torch.bfloat16, 2.0), (torch.float16, 0.7)):
        z, ids, t = make_distill(rng, N, V, K, kind, dtype, ragged=ragged, repeats=repeats, wide=wide)
        L, g, tolL, tolg = _expected(z, ids, t, kind, T)
        full = kind == "logprobs" and K == V       # nothing is left for the rest: L is infinite
        w = rng.random(N).astype(np.float32)
        w[N // 2] = 0.0 if N > 1 else 0.5
        zc, ic, tc, wc = z.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda(), torch.from_numpy(w).cuda()
        kw = dict(kind=kind, temperature=T)
        rows = fh.logits.distill_loss(zc, ic, tc, reduction="none", **kw).double().cpu().numpy()
        if full:
            assert np.isinf(rows).all()
            continue
        assert (np.abs(rows - L) <= tolL).all(), f"{np.abs(rows - L).max()} > {tolL.min()}"
        loss, grad = fh.logits.distill_loss(zc, ic, tc, want_grad=True, **kw)
        assert abs(float(loss) - L.mean()) <= tolL.max() + 2.0 ** -24 * abs(L.mean())
        _close(grad, g, tolg, 1.0 / N)
        w64 = w.astype(np.float64)
        loss, grad = fh.logits.distill_loss(zc, ic, tc, weights=wc, want_grad=True, **kw)
        assert abs(float(loss) - (w64 * L).sum() / w64.sum()) <= tolL.max() * (1 + 2.0 ** -20) + 2.0 ** -23 * np.abs(L).max()
        _close(grad, g, tolg + np.abs(g) * 2.0 ** -22, w64[:, None] / w64.sum())
        assert not grad[w == 0].any()
        total, grad = fh.logits.distill_loss(zc, ic, tc, weights=wc, reduction="sum", want_grad=True, **kw)
        assert abs(float(total) - (w64 * L).sum()) <= (w64 * tolL).sum() + 2.0 ** -23 * np.abs(w64 * L).sum()
        _close(grad, g, tolg + np.abs(g) * 2.0 ** -22, w64[:, None])
        # the differentiable form: same value, a cotangent of its own
        for red, cot in (("mean", np.float32(1.7)), ("none", rng.standard_normal(N).astype(np.float32))):
            leaf = zc.clone().requires_grad_(True)
            out = fh.autograd.distill_loss(leaf, ic, tc, weights=wc, reduction=red, **kw)
            got, = torch.autograd.grad(out, leaf, torch.as_tensor(cot).cuda())
            f = w64 / w64.sum() * float(cot) if red == "mean" else w64 * cot.astype(np.float64)
            _close(got, g, tolg + np.abs(g) * 2.0 ** -22, f[:, None])
            again = fh.logits.distill_loss(zc, ic, tc, weights=wc, reduction=red, **kw)
            assert torch.equal(out.detach(), again)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("N,V,K", [(3, 40, 7), (2, 3000, 30), (2, 9000, 30)])
def test_gradient_against_differences(N, V, K, kind):
    """(L(z + h d) - L(z - h d)) / 2h along a direction of +-1.  Its own errors: the third derivative along d is at most a third cumulant of a
    variable in [-1, 1] / T^3, 0.77 for each of the two log-sum-exps (weights 1 and P <= 1), so h^2 / 6 * 1.54 / T^3 a row, and the float32
    losses' roundings over h."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    T, h = 1.3, 2.0 ** -5
    z, ids, t = make_distill(rng, N, V, K, kind, torch.float32)
    _, _, tolL, _ = _expected(z, ids, t, kind, T)
    args = (torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda())
    kw = dict(kind=kind, temperature=T, reduction="sum")
    for _ in range(3):
        d = torch.from_numpy(rng.choice([-1.0, 1.0], (N, V)).astype(np.float32)).cuda()
        zc = (z.cuda() / 2 ** -18).round() * 2 ** -18      # z +- h d is exact in float32
        up, down = (fh.logits.distill_loss(zc + s * h * d, *args, **kw).double() for s in (1, -1))
        _, g = fh.logits.distill_loss(zc, *args, want_grad=True, **kw)
        along = float((g.double() * d.double()).sum())
        bound = N * h * h / 6 * 1.54 / T ** 3 + (2 * tolL.sum() + 2.0 ** -23 * float(up.abs())) / (2 * h)
        assert abs(float(up - down) / (2 * h) - along) <= bound, (float(up - down) / (2 * h), along, bound)


@pytest.mark.parametrize("V", [40, 5000, 30000])
def test_rows_that_say_nothing(V):
    """Rows that name nothing or weigh nothing have loss 0 and gradient 0 whatever stands in them; -inf in the teacher is probability 0."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    N, K = 5, 6
    z, ids, t = make_distill(rng, N, V, K, "logits", torch.bfloat16)
    z[1] = float("nan")
    z[2] = float("nan")
    ids[1] = -1
    t[3, 2] = -np.inf
    w = np.array([1, 1, 0, 1, 1], np.float32)
    args = (z.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda())
    for kind in ("logits", "logprobs"):
        tt = args[2] if kind == "logits" else torch.log_softmax(args[2], -1) - 0.3
        if kind == "logprobs":
            z[1] = 0.5
            args = (z.cuda(), args[1], tt)
        rows = fh.logits.distill_loss(*args[:2], tt, kind=kind, weights=torch.from_numpy(w).cuda(), reduction="none")
        loss, grad = fh.logits.distill_loss(*args[:2], tt, kind=kind, weights=torch.from_numpy(w).cuda(), want_grad=True)
        assert rows[2] == 0 and not grad[2].any()
        if kind == "logits":
            assert rows[1] == 0 and not grad[1].any()
        else:
            # names nothing: the rest is everything on both sides
            assert abs(float(rows[1])) <= 2.0 ** -21 * (np.log(V) + 5) and float(grad[1].abs().max()) <= 2.0 ** -20
        for r in (0, 3, 4):
            want = orc.distill_row(z[r].double().numpy(), ids[r], tt[r].double().cpu().numpy(), kind, 1.0)[0]
            assert abs(float(rows[r]) - want) <= 2.0 ** -21 * (np.log(V) + 30)
        assert torch.isfinite(loss) and torch.isfinite(grad).all()
    nothing = fh.logits.distill_loss(*args, weights=torch.zeros(N, device="cuda"), want_grad=True)
    assert nothing[0] == 0 and not nothing[1].any()


def test_extremes_of_the_type():
    """The type's lowest value as a mask: those entries have probability 0 and gradient 0; a whole row of it is uniform."""
    import torch
    import flowrl_hip as fh
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        V, low = 300, torch.finfo(dtype).min
        z = torch.zeros((2, V), dtype=dtype)
        z[0, 100:] = low
        z[1] = low
        ids = torch.tensor([[0, 1], [0, 1]]).cuda()
        t = torch.zeros((2, 2)).cuda()
        loss, grad = fh.logits.distill_loss(z.cuda(), ids, t, reduction="none", want_grad=True)
        assert abs(float(loss[0]) - np.log(50.0)) <= 2.0 ** -20 and not grad[0, 100:].any()
        if dtype == torch.float16:           # |z| = 65504 leaves the row's logarithms 2^-24 * 65504 and no less
            assert abs(float(loss[1]) - np.log(150.0)) <= 2.0 ** -7
        assert torch.isfinite(grad).all() and abs(float(grad[1, 5]) - 1 / 300) <= EPS[dtype] / 300 + 2.0 ** -24


def test_strides_types_and_leading_dimensions():
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(2)
    for N, V, K in ((6, 77, 9), (3, 2501, 40), (4, 20003, 5), (300, 9001, 20)):
        z, ids, t = make_distill(rng, N, V, K, "logprobs", torch.bfloat16, ragged=True)
        zc, ic, tc = z.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
        kw = dict(kind="logprobs", want_grad=True)
        want = fh.logits.distill_loss(zc, ic, tc, **kw)
        same = [(zc, ic.long(), tc), (zc.t().contiguous().t(), ic.t().contiguous().t(), tc.t().contiguous().t()),
                (zc, torch.cat([ic, ic], 1)[:, :K], torch.cat([tc, tc], 1)[:, :K])]
        for a in same:
            got = fh.logits.distill_loss(*a, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # where a row starts decides how it is cut into vectors, so the order of its sum: against the formula
        L, g, tolL, tolg = _expected(z, ids, t, "logprobs", 1.0)
        for skip, gap in ((1, 3), (3, 0), (7, 8), (2, 1)):
            buf = torch.zeros((N * (V + gap) + skip,), dtype=torch.bfloat16, device="cuda")
            view = buf[skip:].view(N, V + gap)[:, :V]
            view.copy_(zc)
            loss, grad = fh.logits.distill_loss(view, ic, tc, **kw)
            assert abs(float(loss) - L.mean()) <= tolL.max() + 2.0 ** -24 * abs(L.mean())
            _close(grad, g, tolg, 1.0 / N)
            rows = fh.logits.distill_loss(view, ic, tc, kind="logprobs", reduction="none").double().cpu().numpy()
            assert (np.abs(rows - L) <= tolL).all()
            leaf = view.detach().requires_grad_(True)
            got, = torch.autograd.grad(fh.autograd.distill_loss(leaf, ic, tc, kind="logprobs"), leaf)
            _close(got, g, tolg, 1.0 / N)
        tc = torch.from_numpy(t - t.max() - 1).cuda()
        for dt in (torch.bfloat16, torch.float16):
            narrow = tc.to(dt)
            a, b = fh.logits.distill_loss(zc, ic, narrow), fh.logits.distill_loss(zc, ic, narrow.float())
            assert torch.equal(a, b)
    z3 = torch.randn((2, 3, 60), device="cuda")
    i3, t3 = torch.randint(0, 60, (2, 3, 4), device="cuda"), torch.randn((2, 3, 4), device="cuda")
    rows, grad = fh.logits.distill_loss(z3, i3, t3, reduction="none", want_grad=True)
    assert rows.shape == (2, 3) and grad.shape == z3.shape
    flat, gflat = fh.logits.distill_loss(z3.view(6, 60), i3.view(6, 4), t3.view(6, 4), reduction="none", want_grad=True)
    assert torch.equal(rows.view(6), flat) and torch.equal(grad.view(6, 60), gflat)
    e = torch.empty((0, 60), device="cuda")
    loss, grad = fh.logits.distill_loss(e, i3.view(6, 4)[:0], t3.view(6, 4)[:0], want_grad=True)
    assert float(loss) == 0.0 and grad.shape == (0, 60)


def test_autograd_rules():
    """Two backward passes through one node, a change in place in between, and what is not differentiated."""
    import torch
    import flowrl_hip as fh
    z = torch.randn((5, 333), device="cuda", requires_grad=True)
    ids, t = torch.randint(0, 333, (5, 7), device="cuda"), torch.randn((5, 7), device="cuda")
    loss = fh.autograd.distill_loss(z, ids, t)
    a, = torch.autograd.grad(loss, z, retain_graph=True)
    b, = torch.autograd.grad(loss, z)
    assert torch.equal(a, b)
    (3 * fh.autograd.distill_loss(z, ids, t)).backward()
    # f = cotangent / (N T), then f k / s, then the exponential: six roundings on either side of the comparison and one of 3 a, 13 in all, of f q
    # and (named entries) of f p, with f p <= 3 / 5 and f q <= |f (q - p)| + f p
    want = 3 * a
    named = torch.zeros((5, 333), dtype=torch.bool, device="cuda").scatter_(1, ids, True)
    assert ((z.grad - want).abs() <= 13 * 2.0 ** -24 * (want.abs() + torch.where(named, 2 * 3 / 5, 0.0))).all()
    loss = fh.autograd.distill_loss(z * 1, ids, t)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    with torch.no_grad():
        assert not fh.autograd.distill_loss(z, ids, t).requires_grad
    with pytest.raises(NotImplementedError, match="teacher"):
        fh.autograd.distill_loss(z, ids, t.clone().requires_grad_(True))
    with pytest.raises(NotImplementedError, match="autograd.distill_loss"):
        fh.logits.distill_loss(z, ids, t)
    (v, grads) = fh.autograd.value_and_grad(lambda p: fh.autograd.distill_loss(p["z"], ids, t), {"z": z.detach()})
    direct = fh.logits.distill_loss(z.detach(), ids, t, want_grad=True)
    # the two forms may sum a row's 333 exponentials in another order: less than 32 roundings of that sum, which the gradient's q share
    assert abs(float(v) - float(direct[0])) <= 2.0 ** -19 + 2.0 ** -23 * float(v)
    assert ((grads["z"] - direct[1]).abs() <= 2.0 ** -18 * (direct[1].abs() + torch.where(named, 1 / 5, 0.0))).all()


def test_captured_and_replayed():
    """Forward and backward in one graph, several replays on new inputs, eager work in between."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(11)
    for N, V in ((300, 9001), (4, 30011)):
        z, ids, t = make_distill(rng, N, V, 20, "logprobs", torch.bfloat16)
        zc = z.cuda().requires_grad_(True)
        ic, tc, wc = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda(), torch.rand(N, device="cuda")

        def step():
            loss = fh.autograd.distill_loss(zc, ic, tc, kind="logprobs", weights=wc)
            grad, = torch.autograd.grad(loss, zc)
            return loss.detach(), grad, *fh.logits.distill_loss(zc.detach(), ic, tc, kind="logprobs", weights=wc, want_grad=True)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            with torch.no_grad():
                zc.copy_(torch.randn((N, V), device="cuda"))
            wc.copy_(torch.rand(N, device="cuda"))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_far_rows():
    """Offsets beyond 2^31 elements: the last row of a batch of 2.2e9 logits, value and gradient."""
    import torch
    import flowrl_hip as fh
    N, V = 1100, 2_000_003
    z = torch.zeros((N, V), dtype=torch.bfloat16, device="cuda")
    z[-1, V - 2] = 4.0
    ids = torch.full((N, 1), V - 2, device="cuda")
    rows, grad = fh.logits.distill_loss(z, ids, torch.zeros((N, 1), device="cuda"), reduction="none", want_grad=True)
    tol = 2.0 ** -21 * (np.log(V) + 9)
    lse = np.log(V - 1 + np.exp(4.0))
    assert abs(float(rows[-1]) - (lse - 4.0)) <= tol and abs(float(rows[0]) - np.log(V)) <= tol
    q = np.exp(4.0 - lse)
    assert abs(float(grad[-1, V - 2]) - (q - 1)) <= 2.0 ** -8 and abs(float(grad[-1, 0]) - np.exp(-lse)) <= 2.0 ** -8 * np.exp(-lse) * 1.01
    assert grad[0, V - 2] == -1.0


def test_answer_teach_answer():
    """The operators as they are used together: a policy over tokens answers under its rules step by step, a teacher names its best entries for
    every answer, the policy's table of logits takes a gradient step, and answers again — against the same loop in float64."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(21)
    R, V, K, steps = 6, 700, 16, 5
    table = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32)).cuda()
    teacher = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32) * 2).cuda()
    history = torch.full((R, steps), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(R, dtype=torch.int32, device="cuda")
    allowed = torch.from_numpy(rng.random((R, V)) < 0.5).cuda()
    rules = fh.logits.Constraints(history=history, lengths=lengths, repetition=1.3, frequency=0.4, presence=0.6, allowed=allowed)
    t64, h64 = table.double().cpu().numpy(), np.full((R, steps), -1)
    for k in range(steps):
        token, logprob = fh.logits.choose(table, rules)
        ids = teacher.topk(K).indices
        loss, grad = fh.logits.distill_loss(table, ids, teacher.gather(1, ids), want_grad=True, reduction="sum")
        history[:, k] = token
        lengths += 1
        table = table - 0.5 * grad
        g64, L64 = np.zeros_like(t64), 0.0
        for r in range(R):
            x, _ = orc.constrain_row(t64, r, history=h64[:, :k], repetition=1.3, frequency=0.4, presence=0.6, allowed=allowed.cpu().numpy())
            v, lp = orc.choose_row(*orc.keys_of(x, 0.0, None))
            srt = np.sort(x)
            assert srt[-1] - srt[-2] > 1e-4, "the inputs hold a near tie"
            assert int(token[r]) == v and abs(float(logprob[r]) - lp) <= 2.0 ** -18
            h64[r, k] = v
            i = ids[r].cpu().numpy()
            L, g, _, _ = orc.distill_row(t64[r], i, teacher[r].double().cpu().numpy()[i], "logits", 1.0)
            L64, g64[r] = L64 + L, g
        assert abs(float(loss) - L64) <= R * 2.0 ** -17
        t64 = t64 - 0.5 * g64


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("V,dtype", [(32771, "float32"), (51207, "float32"), (60003, "float32"), (65543, "bfloat16"), (102417, "float16"), (140001, "bfloat16")])
def test_rows_longer_than_registers(V, dtype, kind):
    """A batch that is not split, of rows that registers hold but for a few entries, that LDS holds beside them, and that are read twice: named
    entries at the ends of each, steep rows, a row of weight 0."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    N, K, T, dt = 257, 12, 1.5, getattr(torch, dtype)
    held = 32768 if dt == torch.float32 else 65536
    z, ids, t = make_distill(rng, N, V, K, kind, dt)
    ids[:, :6] = [0, V - 1, held - 1, held, held + 2, V - 9]
    ids[:, 6:] = 100 + np.arange(6) * 1111
    z[3, held:] += 20.0                            # the maximum lies behind what is held
    z[4, :held] = float("-inf")
    z[5, held:] = float("-inf")
    zc, ic, tc = z.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    w = np.ones(N, np.float32)
    w[6] = 0.0
    wc = torch.from_numpy(w).cuda()
    kw = dict(kind=kind, temperature=T, weights=wc, reduction="none")
    rows, grad = fh.logits.distill_loss(zc, ic, tc, want_grad=True, **kw)
    value = fh.logits.distill_loss(zc, ic, tc, **kw)
    leaf = zc.clone().requires_grad_(True)
    out = fh.autograd.distill_loss(leaf, ic, tc, **kw)
    back, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    pick = [0, 1, 3, 128, 255, 256]
    L, g, tolL, tolg = _expected(z[pick], ids[pick], t[pick], kind, T)
    for got in (rows, value, out.detach()):
        assert (np.abs(got[pick].double().cpu().numpy() - L) <= tolL).all()
    for got in (grad, back):
        _close(got[pick], g, tolg + np.abs(g) * 2.0 ** -22, 1.0)
        assert not got[6].any()
    assert rows[6] == 0.0 and value[6] == 0.0
    for r in (4, 5):                               # -inf at a named entry: an infinite divergence, and gradients that stay numbers
        assert rows[r] == float("inf") and value[r] == float("inf")
        free = np.setdiff1d(np.flatnonzero(np.isneginf(z[r].float().numpy())), ids[r])
        assert not grad[r].cpu()[free].any()
    # every row against torch's float32 log sum exp (off by at most 2^-20 of itself and its largest argument, below 40 here)
    lse = torch.logsumexp(zc.float() / T, 1)
    assert torch.isfinite(lse).all()
    if kind == "logits":
        p = torch.softmax(tc.double() / T, 1)
        want = (p * (p.log() + lse.double()[:, None] - zc.gather(1, ic.long()).double() / T)).sum(1) * wc
        fine = torch.isfinite(want)
        assert ((rows.double() - want)[fine].abs() <= 2.0 ** -16 * (want[fine].abs() + 40)).all()
