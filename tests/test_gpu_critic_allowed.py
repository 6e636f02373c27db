"""GPU: choosing among the candidates that a mask leaves (critic_select(allowed=...)): the choice is the one made without a mask, of what is left."""
import numpy as np
import pytest

import flowrl_oracle as orc
from logits_cases import pack_words

pytestmark = pytest.mark.gpu


def _critic(S, A, E=2, seed=4):
    import flowrl_hip as fh
    critic = fh.Ensemblize(base=fh.ScalarCritic(backbone=fh.MLP(hidden_dims=[256, 256], activation="mish")), ensemble_size=E)
    return critic, fh.tree_from_numpy(orc.make_critic_params(S, A, (256, 256), E, seed), "cuda")


@pytest.mark.parametrize("B,N", [(700, 64), (37, 130), (50, 5)])
@pytest.mark.parametrize("T", [0.3, 1.0])
def test_near_ties_are_decided_as_without_a_mask(B, N, T):
    """Noise that brings all keys of a state to within a rounding of one another: the index depends on how a key is rounded."""
    import torch
    import flowrl_hip as fh
    S, A = 11, 3
    rng = np.random.default_rng(B)
    critic, p = _critic(S, A)
    obs = torch.from_numpy(rng.standard_normal((B, S)).astype(np.float32)).cuda()
    actions = torch.from_numpy(rng.standard_normal((B, N, A)).astype(np.float32)).cuda()
    _, _, q = fh.critic_select(critic, p, obs, actions, N)
    g = (7.0 - q.double() / (1e-6 + T)).float()
    plain = fh.critic_select(critic, p, obs, actions, N, temperature=T, gumbel=g)
    every = torch.ones((B, N), dtype=torch.bool, device="cuda")
    for allowed in (every, every[0], torch.from_numpy(pack_words(every.cpu().numpy())).cuda()):
        got = fh.critic_select(critic, p, obs, actions, N, temperature=T, gumbel=g, allowed=allowed)
        assert all(torch.equal(x, y) for x, y in zip(got, plain))
    # what is left, with what is ruled out put out of the running by its noise
    allowed = torch.from_numpy(rng.random((B, N)) < 0.4).cuda()
    allowed[:, 0] |= ~allowed.any(1)
    out = fh.critic_select(critic, p, obs, actions, N, temperature=T, gumbel=torch.where(allowed, g, -1e30))
    for a in (allowed, torch.from_numpy(pack_words(allowed.cpu().numpy())).cuda()):
        got = fh.critic_select(critic, p, obs, actions, N, temperature=T, gumbel=g, allowed=a)
        assert all(torch.equal(x, y) for x, y in zip(got, out))


@pytest.mark.parametrize("N", [3, 64, 200])
def test_what_is_ruled_out_does_not_count(N):
    """NaN and infinite actions behind the mask; a state with nothing left; one mask for every state; a NaN that is allowed is the largest, as for argmax."""
    import torch
    import flowrl_hip as fh
    B, S, A = 41, 5, 2
    rng = np.random.default_rng(N)
    critic, p = _critic(S, A)
    obs = torch.from_numpy(rng.standard_normal((B, S)).astype(np.float32)).cuda()
    clean = torch.from_numpy(rng.standard_normal((B, N, A)).astype(np.float32)).cuda()
    allowed = torch.from_numpy(rng.random((B, N)) < 0.5).cuda()
    allowed[:, 1] = True
    allowed[7] = False
    bad = torch.where(allowed[:, :, None], clean, torch.nan)
    _, _, q = fh.critic_select(critic, p, obs, clean, N)
    best, idx, q2 = fh.critic_select(critic, p, obs, bad, N, allowed=allowed)
    some = torch.arange(B, device="cuda") != 7
    want = torch.where(allowed, q, -torch.inf).argmax(1)
    assert torch.equal(idx.long()[some], want[some]) and idx[7] == -1 and torch.isnan(best[7]).all()
    assert torch.equal(best[some], clean[torch.arange(B, device="cuda"), want][some])
    assert torch.equal(q2[allowed], q[allowed])
    one = allowed[0]
    _, idx, _ = fh.critic_select(critic, p, obs, clean, N, allowed=one, want_q=False)
    assert torch.equal(idx.long(), torch.where(one, q, -torch.inf).argmax(1))
    _, idx, q3 = fh.critic_select(critic, p, obs, torch.where(torch.arange(N, device="cuda")[None, :, None] == 1, torch.nan, clean), N, allowed=allowed)
    assert torch.isnan(q3[:, 1]).all() and (idx[some] == 1).all()


def test_the_chosen_action_is_a_value():
    """As without a mask, no graph leads from the chosen action to the candidates; wrong masks are refused."""
    import torch
    import flowrl_hip as fh
    B, N, S, A = 6, 8, 5, 2
    critic, p = _critic(S, A)
    obs, actions = torch.randn((B, S), device="cuda"), torch.randn((B, N, A), device="cuda", requires_grad=True)
    allowed = torch.ones((B, N), dtype=torch.bool, device="cuda")
    for kw in (dict(), dict(allowed=allowed)):
        best, _, q = fh.critic_select(critic, p, obs, actions, N, **kw)
        assert not best.requires_grad and not q.requires_grad
    for wrong, err in ((allowed[:, :-1], ValueError), (allowed.float(), TypeError), (allowed.cpu(), ValueError), (allowed[:2], ValueError)):
        with pytest.raises(err):
            fh.critic_select(critic, p, obs, actions, N, allowed=wrong)
    with pytest.raises(ValueError, match="gumbel"):
        fh.critic_select(critic, p, obs, actions, N, temperature=0.5, allowed=allowed)


def test_captured_with_a_mask():
    import torch
    import flowrl_hip as fh
    B, N, S, A = 30, 16, 11, 3
    rng = np.random.default_rng(1)
    critic, p = _critic(S, A)
    obs = torch.from_numpy(rng.standard_normal((B, S)).astype(np.float32)).cuda()
    actions = torch.from_numpy(rng.standard_normal((B, N, A)).astype(np.float32)).cuda()
    allowed = torch.from_numpy(rng.random((B, N)) < 0.5).cuda()
    g = torch.from_numpy(rng.gumbel(size=(B, N)).astype(np.float32)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fh.critic_select(critic, p, obs, actions, N, temperature=0.5, gumbel=g, allowed=allowed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = fh.critic_select(critic, p, obs, actions, N, temperature=0.5, gumbel=g, allowed=allowed)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        actions.copy_(torch.from_numpy(rng.standard_normal((B, N, A)).astype(np.float32)))
        allowed.copy_(torch.from_numpy(rng.random((B, N)) < 0.5))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = fh.critic_select(critic, p, obs, actions, N, temperature=0.5, gumbel=g, allowed=allowed)
        assert all(torch.equal(torch.nan_to_num(a, nan=-9.0), torch.nan_to_num(b, nan=-9.0)) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [0.0, 0.7])
def test_sample_and_select_with_a_mask(T):
    """The sampled candidates, chosen from as critic_select chooses: with a mask of everything what it answers without one; builds that have no mask refuse."""
    import torch
    import flowrl_hip as fh
    import helpers as H
    B, N = 40, 8
    c = H.Case("allowed", "ddpm", A=3, S=11, T=5, B=B * N, particles=N, seed=11)
    params, xT, cond, noise = H.make_inputs(c)
    model = H.product_model(c, params)
    critic, p = _critic(11, 3)
    rng = np.random.default_rng(12)
    obs = torch.from_numpy(cond).cuda()
    g = torch.from_numpy(rng.gumbel(size=(B, N)).astype(np.float32)).cuda() if T > 0 else None
    kw = dict(xT=torch.from_numpy(xT.reshape(B, N, 3)).cuda(), noise=torch.from_numpy(noise).cuda(), gumbel=g)
    allowed = torch.from_numpy(rng.random((B, N)) < 0.5).cuda()
    allowed[3] = False
    run = lambda **k: fh.sample_and_select(model, critic, p, None, obs, False, N, "ddpm", T, **kw, **k)[1]  # noqa: E731
    _, x0, _ = model.sample(None, kw["xT"], obs, False, "ddpm", noise=kw["noise"], particles=N)
    best = run(allowed=allowed)
    want, idx, _ = fh.critic_select(critic, p, obs, x0, N, temperature=T, gumbel=g, allowed=allowed)
    assert idx[3] == -1 and torch.isnan(best[3]).all() and allowed[torch.arange(B, device="cuda"), idx.long()][idx >= 0].all()
    assert torch.equal(torch.nan_to_num(best, nan=9.0), torch.nan_to_num(want, nan=9.0))
    assert torch.equal(run(allowed=torch.ones_like(allowed)), run(fused=False))
    with pytest.raises(fh.FlowRLHipUnsupported, match="allowed"):
        run(allowed=allowed, fused=True)
    with pytest.raises(ValueError, match="temperature"):
        fh.sample_and_select(model, critic, p, None, obs, False, N, "ddpm", None, allowed=allowed, **kw)
