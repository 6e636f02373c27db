"""GPU: frl_logits_constrain / frl_logits_choose against the float64 restatement (oracle/logits_oracle.py).  PARITY UNPINNED: the
reference has no such operators.

Tolerances count roundings.  A constrained element goes through at most 8 float32 operations plus one per bias listed for it, each off by
at most 2^-24 of the magnitudes that went in (`size`), then one rounding to the output type.  A key adds the reciprocal of the temperature (two
roundings), a product and a sum.  A choice is right if no other entry is ahead of it by more than both keys' errors.  The
log-probability inherits the errors of y (log sum exp moves by no more than its arguments) and adds the float32 exponentials': their
arguments are rounded (2^-23 of m - y), the hardware's exponential is off by 2^-23, the sum by its depth; weighted by the
softmax itself this is below 2^-21 (m - y[token] + ln V + 4)."""
import numpy as np
import pytest

import logits_oracle as orc
from logits_cases import EPS, TINY, make_rules, pack_words, rules_to_gpu

pytestmark = pytest.mark.gpu


def _logits(rng, R, V, dtype, pad=True):
    import torch
    z = (4 * rng.standard_normal((R, V))).astype(np.float32)
    if pad and V > 8:
        z[:, V - V // 50 - 1:] = -np.inf
    return torch.from_numpy(z).to(dtype)


def _check_constrained(out, z, c, K, rows=None):
    import torch
    zn, on = z.double().numpy(), out.double().cpu().numpy()
    half, tiny = EPS[out.dtype], TINY[out.dtype]
    for r in (range(z.shape[0]) if rows is None else rows):
        x, size = orc.constrain_row(zn, r, **c)
        fin = np.isfinite(x)
        np.testing.assert_array_equal(on[r][~fin], x[~fin])
        err = (8 + K) * 2.0 ** -24 * size[fin]
        if out.dtype == torch.float32:
            half = 0.0      # the last of the counted operations is the result
        bad = np.abs(on[r][fin] - x[fin]) > err + half * (np.abs(x[fin]) + err) + tiny
        assert not bad.any(), f"row {r}: {bad.sum()} of {fin.sum()} elements, first at {np.flatnonzero(fin)[bad][:3]}"


def _check_chosen(token, logprob, z, c, K, temperature, gumbel, rows=None):
    zn, V = z.double().numpy(), z.shape[1]
    token, logprob = token.cpu().numpy(), logprob.double().cpu().numpy()
    for r in (range(z.shape[0]) if rows is None else rows):
        x, size = orc.constrain_row(zn, r, **c)
        T = float(np.asarray(temperature).reshape(-1)[r]) if np.ndim(temperature) else float(temperature)
        y, key = orc.keys_of(x, T, None if gumbel is None else gumbel[r])
        if (y == -np.inf).all():
            assert token[r] == -1 and logprob[r] == -np.inf
            continue
        drawn = gumbel is not None and T > 0
        fin = np.isfinite(y)
        err = (8 + K) * 2.0 ** -24 * np.where(fin, size, 0.0) * (1.0 / (1e-6 + T) if drawn else 1.0) + (4 * 2.0 ** -24 * np.abs(np.where(fin, y, 0.0)) if drawn else 0.0)
        kerr = err + (2.0 ** -24 * np.abs(np.where(fin, key, 0.0)) if drawn else 0.0)
        v = int(token[r])
        assert 0 <= v < V and fin[v], f"row {r}: token {v}"
        assert key[v] + kerr[v] >= (key[fin] - kerr[fin]).max(), f"row {r}: token {v} at {key[v]}, best {key[fin].max()}"
        m = y[fin].max()
        lse = m + np.log(np.exp(y[fin] - m).sum())
        tol = err[v] + err[fin].max() + 2.0 ** -21 * (m - y[v] + np.log(V) + 4) + 2.0 ** -23 * abs(m)
        assert abs(logprob[r] - (y[v] - lse)) <= tol, f"row {r}: logprob {logprob[r]} vs {y[v] - lse}, tol {tol}"


CASES = [
    # R, V, rules, mask
    (1, 1, dict(), None),
    (2, 3, dict(hist=5, dense="shared"), "bool"),
    (5, 31, dict(hist=1, sparse=3), "words"),
    (7, 64, dict(), "bool"),
    (70, 65, dict(hist=40, prompt=True, sparse=9, dense="rows"), "words"),
    (6, 511, dict(hist=700, sparse=64, wide=True), "bool"),
    (5, 512, dict(hist=33), None),
    (5, 513, dict(hist=100, prompt=True, sparse=17), "words"),
    (4, 2047, dict(sparse=300, dense="rows"), "bool"),
    (4, 2049, dict(hist=257, prompt=True, tensors=False), "words"),
    (3, 4100, dict(hist=1000, sparse=2048), None),
    (9, 50001, dict(hist=513, prompt=True, sparse=40, dense="shared", wide=True), "words"),
    (300, 8195, dict(hist=130, prompt=True, sparse=33), "words"),          # workgroups of 1024 threads
    (520, 5003, dict(hist=64, dense="shared"), "bool"),
    (600, 4097, dict(), None),
    (600, 5003, dict(hist=16, sparse=2048), None),                          # the longest lists beside 1024 threads
    (2, 40, dict(hist=9, sparse=2048), "bool"),                             # lists far longer than the row
    (3, 70001, dict(hist=9000, prompt=True, sparse=600, wide=True), "bool"),   # a history that no group keeps in registers
    (560, 9001, dict(hist=5000, prompt=True), None),
    (5, 9001, dict(hist=1500, prompt=True, sparse=20, wide=True), "words"),  # beyond what 256 threads keep in registers
    (128, 70001, dict(hist=3000, prompt=True, sparse=50), "words"),         # several chunks to a workgroup of 1024 threads
    (4300, 4001, dict(hist=50, sparse=5), "words"),                         # and to one of 256
]
IDS = [f"{R}x{V}-{'-'.join(k for k in kw)}-{mask}" for R, V, kw, mask in CASES]


@pytest.mark.parametrize("R,V,kw,mask", CASES, ids=IDS)
def test_constrain(R, V, kw, mask):
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(R * 100003 + V)
    c = make_rules(rng, R, V, mask=mask, **kw)
    rules = rules_to_gpu(fh, c, mask)
    rows = range(R) if R <= 70 else sorted({0, 1, 2, 3, R - 1, *rng.integers(0, R, 20).tolist()})
    for dtype, out_dtype in ((torch.float32, None), (torch.bfloat16, None), (torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, None)):
        z = _logits(rng, R, V, dtype)
        out = fh.logits.constrain(z.cuda(), rules, out_dtype=out_dtype)
        assert out.dtype == (out_dtype or dtype) and out.shape == z.shape
        _check_constrained(out, z, c, kw.get("sparse", 0), rows)


@pytest.mark.parametrize("draw", ["greedy", "mixed", "number"])
@pytest.mark.parametrize("R,V,kw,mask", CASES, ids=IDS)
def test_choose(R, V, kw, mask, draw):
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(R * 100019 + V)
    c = make_rules(rng, R, V, mask=mask, **kw)
    rules = rules_to_gpu(fh, c, mask)
    rows = range(R) if R <= 70 else sorted({0, 1, 2, 3, R - 1, *rng.integers(0, R, 20).tolist()})
    gumbel = rng.gumbel(size=(R, V)).astype(np.float32) if draw != "greedy" else None
    temperature = (rng.random(R) * 1.5 * (rng.random(R) < 0.8)).astype(np.float32) if draw == "mixed" else 0.7 if draw == "number" else 0.0
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z = _logits(rng, R, V, dtype, pad=draw != "number")
        t = torch.from_numpy(temperature).cuda() if draw == "mixed" else temperature
        token, logprob = fh.logits.choose(z.cuda(), rules, temperature=t, gumbel=None if gumbel is None else torch.from_numpy(gumbel).cuda())
        assert token.dtype == torch.int32 and logprob.dtype == torch.float32 and token.shape == logprob.shape == (R,)
        _check_chosen(token, logprob, z, c, kw.get("sparse", 0), temperature, gumbel, rows)


@pytest.mark.parametrize("V", [5, 700, 40000])
def test_choose_is_the_argmax_of_constrain(V):
    """The two entry points apply the rules bit for bit alike: a greedy choice is the first argmax of the float32 constrained row."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    c = make_rules(rng, 6, V, hist=90, sparse=min(20, V), mask="words")
    rules = rules_to_gpu(fh, c, "words")
    z = _logits(rng, 6, V, torch.bfloat16).cuda()
    x = fh.logits.constrain(z, rules, out_dtype=torch.float32)
    token, _ = fh.logits.choose(z, rules)
    want = torch.where((x == -torch.inf).all(1), -1, x.argmax(1)).to(torch.int32)
    assert torch.equal(token, want)


@pytest.mark.parametrize("V", [3, 64, 600, 9000, 70000])
def test_ties_take_the_first(V):
    import torch
    import flowrl_hip as fh
    z = torch.zeros((4, V), device="cuda")
    z[1, V // 2:] = 1.0
    z[2] = -0.0
    z[2, V - 1] = 0.0                       # equal to -0
    z[3, V - 1] = 2.0
    token, logprob = fh.logits.choose(z)
    assert token.tolist() == [0, V // 2, 0, V - 1]
    # every exponential is exact and so are their sums up to 2^24: only the logarithm and one subtraction round
    assert abs(float(logprob[0]) + np.log(V)) <= 2.0 ** -22 * (1 + np.log(V))


@pytest.mark.parametrize("R,V", [(1, 5000), (40, 33000), (700, 9000)])
def test_extreme_temperatures(R, V):
    """From the argmax of the noise (infinite temperature, what is not allowed stays out) to that of the logits (tiny)."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    z = _logits(rng, R, V, torch.float32).cuda()
    g = torch.from_numpy(rng.gumbel(size=(R, V)).astype(np.float32)).cuda()
    allowed = torch.rand((R, V), device="cuda") < 0.5
    rules = fh.logits.Constraints(allowed=allowed)
    x = torch.where(allowed, z, -torch.inf)
    token, logprob = fh.logits.choose(z, rules, temperature=float("inf"), gumbel=g)
    assert torch.equal(token.long(), torch.where(x == -torch.inf, -torch.inf, g).argmax(1))
    n = (x > -torch.inf).sum(1).double().cpu().numpy()
    assert (np.abs(logprob.double().cpu().numpy() + np.log(n)) <= 2.0 ** -21 * (np.log(n) + 4)).all()
    # 1 / (1e-6 + 1e-30) = 1e6 scales the gaps of the logits past what the noise spans (a gap of 1e-4 is 100)
    top = x.topk(2, dim=1).values
    clear = top[:, 0] - top[:, 1] > 1e-4
    token, _ = fh.logits.choose(z, rules, temperature=1e-30, gumbel=g)
    assert clear.any() and torch.equal(token.long()[clear], x.argmax(1)[clear])


@pytest.mark.parametrize("V", [40, 3000, 33000])
def test_values_that_are_no_numbers(V):
    """NaN and infinities in masked places do nothing; an allowed NaN is the largest value; a row of nothing answers -1."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    z = torch.from_numpy(rng.standard_normal((7, V)).astype(np.float32))
    low = torch.finfo(torch.float32).min
    allowed = torch.ones((7, V), dtype=torch.bool)
    clean = z.clone()
    hit = torch.zeros(V, dtype=torch.bool)
    hit[torch.from_numpy(rng.choice(V, V // 4, replace=False))] = True
    for r, bad in ((0, float("nan")), (1, float("inf")), (2, -float("inf"))):
        z[r, hit] = bad
        allowed[r, hit] = False
        clean[r, hit] = low                  # the oracle's row, masked anyway
    z[3, V // 3] = float("nan")
    z[3, V // 2] = float("nan")
    z[4] = -float("inf")
    z[5] = low                               # the type's lowest value everywhere: a uniform row, not an empty one
    allowed[6] = False
    for mask in ("bool", "words"):
        a = (allowed if mask == "bool" else torch.from_numpy(pack_words(allowed.numpy()))).cuda()
        rules = fh.logits.Constraints(allowed=a)
        out = fh.logits.constrain(z.cuda(), rules).cpu()
        assert torch.equal(out[:3], torch.where(allowed[:3], z[:3], -torch.inf))
        assert torch.isnan(out[3, V // 3]) and int(torch.isnan(out).sum()) == 2
        assert (out[6] == -torch.inf).all() and (out[5] == low).all()
        token, logprob = fh.logits.choose(z.cuda(), rules)
        token, logprob = token.tolist(), logprob.tolist()
        assert token[3] == V // 3 and np.isnan(logprob[3])
        assert token[4] == token[6] == -1 and logprob[4] == logprob[6] == -np.inf
        assert token[5] == 0 and abs(logprob[5] + np.log(V)) <= 2.0 ** -22 * (1 + np.log(V))
        _check_chosen(torch.tensor(token[:3]), torch.tensor(logprob[:3]), clean[:3], dict(allowed=allowed.numpy()), 0, 0.0, None)


def test_strides_alignment_and_neighbours():
    """Rows anywhere: odd distances, odd starts, transposed and expanded inputs; what lies between the output's rows stays."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(5)
    for R, V, dtype in ((5, 77, torch.bfloat16), (3, 2501, torch.float16), (4, 9001, torch.float32), (600, 4099, torch.bfloat16)):
        c = make_rules(rng, R, V, hist=20, sparse=5, mask="bool")
        rules = rules_to_gpu(fh, c, "bool")
        z = _logits(rng, R, V, dtype)
        want = fh.logits.constrain(z.cuda(), rules)
        for skip, gap in ((1, 3), (3, 0), (0, 5)):
            buf = torch.full((skip + R * (V + gap),), 7.0, dtype=dtype, device="cuda")
            view = buf[skip:].view(R, V + gap)[:, :V]
            view.copy_(z)
            obuf = torch.full_like(buf, 9.0)
            out = obuf[skip:].view(R, V + gap)[:, :V]
            assert fh.logits.constrain(view, rules, out=out) is out
            assert torch.equal(out, want)
            assert (obuf[:skip] == 9).all() and (obuf[skip:].view(R, V + gap)[:, V:] == 9).all()
            assert torch.equal(fh.logits.constrain(view, rules, out=view), want)          # in place
            assert torch.equal(view, want) and (buf[skip:].view(R, V + gap)[:, V:] == 7).all()
        t = z.cuda().t().contiguous().t()
        assert t.stride(0) == 1 and torch.equal(fh.logits.constrain(t, rules), want)
        shifted = fh.logits.Constraints(**{k: (torch.cat([v, v], -1)[..., 1:v.shape[-1] + 1] if torch.is_tensor(v) and v.dim() == 2 else v)
                                           for k, v in rules.__dict__.items()})
        rolled = {k: (np.concatenate([v, v], -1)[..., 1:v.shape[-1] + 1] if isinstance(v, np.ndarray) and v.ndim == 2 else v) for k, v in c.items()}
        _check_constrained(fh.logits.constrain(z.cuda(), shifted), z, rolled, 5, range(min(R, 5)))
    one = torch.randn((1, 300), device="cuda").expand(4, 300)
    token, _ = fh.logits.choose(one)
    assert torch.equal(token, one.argmax(1).int())


def test_leading_dimensions_shared_rules_and_no_rows():
    import torch
    import flowrl_hip as fh
    z = torch.randn((2, 3, 50), device="cuda")
    allowed = torch.rand(50, device="cuda") < 0.5
    bias = torch.randn(50, device="cuda")
    tokens, values = torch.tensor([3, 3, 49, -1, 50], device="cuda"), torch.tensor([1.0, 2.0, 4.0, 8.0, 16.0], device="cuda")
    rules = fh.logits.Constraints(allowed=allowed, bias=bias, bias_tokens=tokens, bias_values=values)
    want = z + bias
    want[..., 3] += 3.0
    want[..., 49] += 4.0
    want = torch.where(allowed, want, -torch.inf)
    out = fh.logits.constrain(z, rules)
    assert out.shape == z.shape and torch.equal(out, want)
    token, logprob = fh.logits.choose(z, rules)
    assert token.shape == logprob.shape == (2, 3) and torch.equal(token.long(), want.argmax(-1))
    assert torch.equal(fh.logits.constrain(z), z)
    v, _ = fh.logits.choose(z[0, 0])
    assert v.shape == () and int(v) == int(z[0, 0].argmax())
    empty = torch.empty((0, 50), device="cuda", dtype=torch.bfloat16)
    assert fh.logits.constrain(empty, rules).shape == (0, 50) and fh.logits.choose(empty, rules)[0].shape == (0,)
    none = fh.logits.Constraints(history=torch.empty((6, 0), dtype=torch.int32, device="cuda"), bias_tokens=torch.empty((0,), dtype=torch.int64, device="cuda"),
                                 bias_values=torch.empty((0,), device="cuda"), repetition=2.0)
    assert torch.equal(fh.logits.constrain(z, none), z)


def test_lengths_beyond_the_history_and_repeated_biases():
    """lengths / prompt_lengths are clamped; a token listed many times gets its biases in the order of the list, at every position."""
    import torch
    import flowrl_hip as fh
    V = 2100
    z = torch.zeros((3, V), device="cuda")
    h = torch.tensor([[4, 4, 9], [4, 4, 9], [4, 4, 9]], device="cuda")
    rules = fh.logits.Constraints(history=h, lengths=torch.tensor([99, -5, 2], dtype=torch.int32, device="cuda"), frequency=1.0,
                                  prompt_lengths=torch.tensor([-1, 7, 99], dtype=torch.int32, device="cuda"))
    out = fh.logits.constrain(z, rules)
    assert out[0, [4, 9]].tolist() == [-2.0, -1.0] and not out[1].any() and not out[2].any()
    values = torch.tensor([1e8, 1.0, -1e8, 1.0], device="cuda").repeat(512)
    tokens = torch.full((2048,), 77, device="cuda")
    got = fh.logits.constrain(z, fh.logits.Constraints(bias_tokens=tokens, bias_values=values))
    want = np.float32(0)
    for v in values.cpu().numpy():
        want = np.float32(want + v)          # float32, one after the other
    assert got[0, 77] == float(want) and torch.count_nonzero(got) == 3


def test_same_bits_again_and_on_another_stream():
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(9)
    R, V = 12, 33333
    rules = rules_to_gpu(fh, make_rules(rng, R, V, hist=300, sparse=50, mask="words"), "words")
    z = _logits(rng, R, V, torch.bfloat16).cuda()
    g = torch.from_numpy(rng.gumbel(size=(R, V)).astype(np.float32)).cuda()
    first = fh.logits.choose(z, rules, temperature=0.9, gumbel=g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(fh.logits.choose(z, rules, temperature=0.9, gumbel=g))
    torch.cuda.synchronize()
    for token, logprob in got:
        assert torch.equal(token, first[0]) and torch.equal(logprob, first[1])


def test_captured_and_replayed():
    """Two graphs captured from the same calls replay side by side on new inputs, with eager calls between them."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(10)
    R, V = 5, 20011
    c = make_rules(rng, R, V, hist=64, prompt=True, sparse=10, mask="words")
    rules = rules_to_gpu(fh, c, "words")
    z = _logits(rng, R, V, torch.float16).cuda()
    g = torch.from_numpy(rng.gumbel(size=(R, V)).astype(np.float32)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fh.logits.choose(z, rules, temperature=0.5, gumbel=g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (*fh.logits.choose(z, rules, temperature=0.5, gumbel=g), fh.logits.constrain(z, rules))
        graphs.append((graph, out))
    for k in range(3):
        z.copy_(_logits(rng, R, V, torch.float16))
        rules.lengths.copy_(torch.from_numpy(rng.integers(0, 65, R).astype(np.int32)))
        for graph, _ in graphs:
            graph.replay()
        want = (*fh.logits.choose(z, rules, temperature=0.5, gumbel=g), fh.logits.constrain(z, rules))
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), k


def test_far_rows():
    """Offsets beyond 2^31 elements: the last rows of a tall batch."""
    import torch
    import flowrl_hip as fh
    R, V = 1100, 2_000_003
    z = torch.zeros((R, V), dtype=torch.bfloat16, device="cuda")
    z[-1, V - 1] = 3.0
    z[-2, 17] = 3.0
    token, logprob = fh.logits.choose(z)
    assert token[-2:].tolist() == [17, V - 1] and not token[:-2].any()
    want = 3.0 - np.log(V - 1 + np.exp(3.0))
    assert (logprob[-2:].cpu().double() - want).abs().max() <= 2.0 ** -21 * (np.log(V) + 7)
    h = torch.full((R, 1), V - 1, device="cuda")
    out = fh.logits.constrain(z, fh.logits.Constraints(history=h, frequency=1.0), out=z)
    assert out[-1, V - 1] == 2.0 and out[-2, V - 1] == -1.0 and out[-2, 17] == 3.0


def test_critic_choice_with_candidates_ruled_out():
    """critic_select(allowed=...): the critic's own values, chosen among what is allowed; a state without candidates answers -1 and NaN."""
    import torch
    import flowrl_hip as fh
    import flowrl_oracle as orc_net
    B, N, S, A = 33, 50, 11, 3
    rng = np.random.default_rng(3)
    critic = fh.Ensemblize(base=fh.ScalarCritic(backbone=fh.MLP(hidden_dims=[256, 256], activation="mish")), ensemble_size=2)
    p = fh.tree_from_numpy(orc_net.make_critic_params(S, A, (256, 256), 2, 4), "cuda")
    obs = torch.from_numpy(rng.standard_normal((B, S)).astype(np.float32)).cuda()
    actions = torch.from_numpy(rng.standard_normal((B, N, A)).astype(np.float32)).cuda()
    allowed = torch.from_numpy(rng.random((B, N)) < 0.3).cuda()
    allowed[5] = False
    g = torch.from_numpy(rng.gumbel(size=(B, N)).astype(np.float32)).cuda()
    _, _, q = fh.critic_select(critic, p, obs, actions, N)
    for T, noise in ((0.0, None), (0.5, g)):
        best, idx, q2 = fh.critic_select(critic, p, obs, actions, N, temperature=T, gumbel=noise, allowed=allowed)
        assert torch.equal(q, q2)
        key = torch.where(allowed, q if noise is None else q.double() / (1e-6 + T) + noise.double(), -torch.inf)
        assert idx[5] == -1 and torch.isnan(best[5]).all()
        some = torch.arange(B, device="cuda") != 5
        picked = key.gather(1, idx.long().clamp(min=0)[:, None])[:, 0]
        assert ((key.amax(1) - picked)[some] <= 2.0 ** -20 * (1 + key.amax(1)[some].abs())).all()
        assert torch.equal(best[some], actions[torch.arange(B, device="cuda"), idx.long()][some])
    everything = torch.ones((B, N), dtype=torch.bool, device="cuda")
    a, b = fh.critic_select(critic, p, obs, actions, N, allowed=everything), fh.critic_select(critic, p, obs, actions, N)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_in_place_is_noticed_by_graphs():
    """torch's graphs refuse a backward whose saved tensor `out=` has overwritten."""
    import torch
    import flowrl_hip as fh
    z = torch.randn(3, 40, device="cuda")
    s = torch.ones((), device="cuda", requires_grad=True)
    y = (z * s).sum()                              # keeps z for the gradient of s
    fh.logits.constrain(z, fh.logits.Constraints(bias=torch.ones(40, device="cuda")), out=z)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        q = torch.zeros(3, 40, device="cuda")
        fh.logits.constrain(z, out=q)
        assert torch.equal(q, z)
    with pytest.raises(NotImplementedError):
        fh.logits.constrain(z, out=torch.zeros(3, 40, device="cuda", requires_grad=True))
