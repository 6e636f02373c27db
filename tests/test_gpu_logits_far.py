"""GPU: choices from rows whose logits lie far from zero: fills of masked entries, forced tokens, temperatures near nothing.

The log-probability of the largest entry is -log sum exp(y - max y), whose arguments are differences: its error does not grow with the
distance from zero.  Tolerance as in test_gpu_logits.py, 2^-21 (max y - y[token] + ln V + 4), without a term in |max y|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FILLS = [-1e9, -1e10, -1e20, -1e30, -3.4e38, 1e9, 1e10, 1e20, 1e30]


def _logprob(y, v):
    y = np.asarray(y, np.float64)
    m = y[v]
    with np.errstate(over="ignore"):
        return -np.log(np.exp(y - m).sum())


@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("R,V", [(3, 40), (3, 3000), (3, 70000), (600, 4097), (300, 33000)])
def test_choice_far_from_zero(R, V, fill):
    """A row of one value throughout, a row with one entry ahead of the others, a row of two levels; greedy and drawn."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    tol = 2.0 ** -21 * (np.log(V) + 4)
    for dtype in (torch.float32, torch.bfloat16):
        near = torch.tensor(max(fill, torch.finfo(dtype).min)).to(dtype)      # -3.4e38 is no bfloat16 number but -inf
        z = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32)).to(dtype)
        z[0] = near
        z[1] = 2 * near if fill < 0 else 0.0
        z[1, V // 2] = near
        z[2, : V // 4] = near                          # ahead of the ordinary entries, or behind them
        token, logprob = fh.logits.choose(z.cuda())
        token, logprob = token.tolist(), logprob.tolist()
        assert token[:2] == [0, V // 2]
        assert abs(logprob[0] + np.log(V)) <= tol and abs(logprob[1]) <= tol
        want = z.double().numpy()
        for r in (2, R - 1):
            assert want[r, token[r]] == want[r].max() and abs(logprob[r] - _logprob(want[r], token[r])) <= tol
        # 1 / (1e-6 + 0.5) scales every entry of a level alike, and noise of this size is lost in it
        g = torch.from_numpy(rng.gumbel(size=(R, V)).astype(np.float32)).cuda()
        if abs(fill) < 1e38:
            token, logprob = fh.logits.choose(z.cuda(), temperature=0.5, gumbel=g)
            assert token[:2].tolist() == [0, V // 2]
            assert abs(float(logprob[0]) + np.log(V)) <= tol and abs(float(logprob[1])) <= tol


@pytest.mark.parametrize("V", [40, 3000, 70000])
def test_forced_tokens(V):
    """A bias of 1e10 on one token leaves it a probability of 1; -1e10 on all others, too; on every token, what there was up to its rounding."""
    import torch
    import flowrl_hip as fh
    z = torch.randn((2, V), device="cuda")
    at = V // 3
    one = fh.logits.Constraints(bias_tokens=torch.tensor([at], device="cuda"), bias_values=torch.tensor([1e10], device="cuda"))
    others = torch.full((V,), -1e10, device="cuda")
    others[at] = 0.0
    for rules in (one, fh.logits.Constraints(bias=others)):
        token, logprob = fh.logits.choose(z, rules)
        assert token.tolist() == [at, at] and float(logprob.abs().max()) <= 2.0 ** -21 * (np.log(V) + 4)
    token, logprob = fh.logits.choose(z, fh.logits.Constraints(bias=torch.full((V,), 1e10, device="cuda")))
    assert token.tolist() == [0, 0]                    # |z| < 512 is less than half a step of 1e10
    assert float((logprob + float(np.log(V))).abs().max()) <= 2.0 ** -21 * (np.log(V) + 4)


@pytest.mark.parametrize("level", [3.0e4, 4.54e4, -4.54e4, 9.1e4, 1e6])
@pytest.mark.parametrize("R,V", [(2, 500), (2, 9000), (2, 200001), (300, 33000)])
def test_levels_in_between(R, V, level):
    """Maxima of threads, chunks and parts on either side of where the exponent's product is no longer taken in one step."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(V)
    z = torch.from_numpy((level + 40 * rng.standard_normal((R, V))).astype(np.float32))
    token, logprob = fh.logits.choose(z.cuda())
    zn = z.double().numpy()
    for r in range(2):
        v = int(token[r])
        assert v == int(zn[r].argmax()) and abs(float(logprob[r]) - _logprob(zn[r], v)) <= 2.0 ** -21 * (np.log(V) + 4)


@pytest.mark.parametrize("T", [1e-30, 1e-9, 1e-6, 1e-4])
def test_logprob_at_tiny_temperatures(T):
    """y = x / (1e-6 + T) reaches 1e7; three roundings of y[token] and of the maximum count beside the differences."""
    import torch
    import flowrl_hip as fh
    rng = np.random.default_rng(7)
    for R, V in ((3, 300), (3, 5000), (2, 70000)):
        x = (4 * rng.standard_normal((R, V))).astype(np.float32)
        x[0] = np.float32(3.0)
        g = rng.gumbel(size=(R, V)).astype(np.float32)
        token, logprob = fh.logits.choose(torch.from_numpy(x).cuda(), temperature=T, gumbel=torch.from_numpy(g).cuda())
        y = x.astype(np.float64) / (1e-6 + T)
        for r in range(R):
            v = int(token[r])
            m = y[r].max()
            want = y[r, v] - m - np.log(np.exp(y[r] - m).sum())
            tol = 2.0 ** -21 * (m - y[r, v] + np.log(V) + 4) + (0 if r == 0 else 2 * 3 * 2.0 ** -24 * abs(m))
            assert abs(float(logprob[r]) - want) <= tol
