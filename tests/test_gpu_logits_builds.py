"""GPU: every build of the kernel for rows of logits by name (frl_last_kernels), on the lists that it is compiled for: groups of 64, 256 and 1024 threads,
without lists, with a history, with listed biases, with both; one group a row and several."""
import numpy as np
import pytest

from logits_cases import make_rules, rules_to_gpu
from test_gpu_logits import _check_chosen, _check_constrained, _logits

pytestmark = pytest.mark.gpu

# rows, vocabulary, rules, mask, threads of constrain, threads of choose, whether a choice joins several groups a row
CASES = [
    (9, 500, dict(), "bool", 64, 64, False),
    (9, 500, dict(hist=300, prompt=True), None, 64, 64, False),
    (9, 500, dict(sparse=200), None, 64, 64, False),
    (9, 500, dict(hist=300, sparse=200), "words", 64, 64, False),
    (30, 33333, dict(), None, 256, 256, True),
    (30, 33333, dict(hist=100, dense="shared"), "bool", 256, 256, True),
    (30, 33333, dict(sparse=50), "words", 256, 256, True),
    (4300, 4001, dict(hist=50, sparse=5), None, 256, 256, False),
    (512, 20011, dict(), "words", 1024, 1024, False),
    (512, 33333, dict(dense="rows"), None, 1024, 1024, False),
    (512, 33333, dict(sparse=64), "bool", 1024, 1024, False),
    (300, 70001, dict(sparse=2048), None, 1024, 1024, True),
    (40, 70001, dict(hist=4000, prompt=True, wide=True), "bool", 1024, 1024, True),
    (300, 20011, dict(hist=4000, prompt=True), None, 1024, 1024, False),
    (128, 70001, dict(hist=4000, sparse=64), "words", 1024, 1024, True),
    (128, 5003, dict(hist=4000, prompt=True, sparse=64, dense="shared"), "words", 1024, 1024, False),
]


@pytest.mark.parametrize("R,V,kw,mask,by_constrain,by_choose,joined", CASES, ids=[f"{c[0]}x{c[1]}-{'-'.join(c[2])}-{c[3]}" for c in CASES])
def test_builds(R, V, kw, mask, by_constrain, by_choose, joined):
    import torch
    import flowrl_hip as fh
    from flowrl_hip import _lib
    lib = _lib.load()
    rng = np.random.default_rng(R * 100043 + V)
    c = make_rules(rng, R, V, mask=mask, **kw)
    rules = rules_to_gpu(fh, c, mask)
    rows = sorted({0, 1, 2, 3, R - 1, *rng.integers(0, R, 8).tolist()})
    gumbel = rng.gumbel(size=(R, V)).astype(np.float32)
    temperature = (rng.random(R) * 1.5 * (rng.random(R) < 0.8)).astype(np.float32)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z = _logits(rng, R, V, dtype)
        out = fh.logits.constrain(z.cuda(), rules)
        ran = lib.frl_last_kernels().decode()
        assert f"<constrain, {by_constrain} threads>" in ran, ran
        _check_constrained(out, z, c, kw.get("sparse", 0), rows)
        for noise in (None, gumbel):
            token, logprob = fh.logits.choose(z.cuda(), rules, temperature=torch.from_numpy(temperature).cuda(), gumbel=None if noise is None else torch.from_numpy(noise).cuda())
            ran = lib.frl_last_kernels().decode()
            assert f"<choose, {by_choose} threads>" in ran and ("join" in ran) == joined, ran
            _check_chosen(token, logprob, z, c, kw.get("sparse", 0), temperature, noise, rows)
