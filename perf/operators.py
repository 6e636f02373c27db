"""The operators over a vocabulary of discrete choices, as cases that can be timed and compared.

  constrain   logits with repetition / frequency / presence penalties, biases and an allowed-token mask applied
  choose      the same, then the argmax or the Gumbel-max draw of every row and its log-probability
  distill     KL divergence of a student's softmax from a teacher's top entries: value, value + gradient, autograd

``own`` False: the plain form in elementary torch operations; True: flowrl_hip's kernels on the same inputs.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _logits(op, name, rows, vocab, dtype, hist=0, prompt=False, wide_ids=False, sparse=0, dense=False, mask="none", out="same", draw="greedy"):
    return dict(name=name, op=op, rows=rows, vocab=vocab, dtype=dtype, hist=hist, prompt=prompt, wide_ids=wide_ids, sparse=sparse,
                dense=dense, mask=mask, out=out, draw=draw)


def _distill(name, rows, vocab, dtype, top, kind, how, weights=False, wide_ids=False, ragged=False, temperature=1.0):
    return dict(name=name, op="distill", rows=rows, vocab=vocab, dtype=dtype, top=top, kind=kind, how=how, weights=weights,
                wide_ids=wide_ids, ragged=ragged, temperature=temperature)


def listed():
    return [
        # one sequence being answered: every rule of a serving request at once
        _logits("constrain", "constrain one row", 1, 32000, "bf16", hist=512, prompt=True, sparse=300, mask="words"),
        # a mid-sized batch with an odd vocabulary, half precision in, float32 out for a sampler elsewhere
        _logits("constrain", "constrain odd batch", 64, 50001, "f16", hist=2048, dense=True, mask="bool", out="f32", wide_ids=True),
        # a full serving batch over a large vocabulary and long histories
        _logits("constrain", "constrain full batch", 512, 131072, "f32", hist=4096, prompt=True, sparse=32, mask="words"),
        # best-of-N: 8192 states x 64 candidate actions with some of them ruled out, categorical over the critic's values
        _logits("choose", "choose candidates", 8192, 64, "f32", mask="bool", draw="all"),
        # greedy decoding of one sequence under a grammar
        _logits("choose", "choose greedy row", 1, 128000, "bf16", hist=1024, mask="words"),
        # a serving batch in which some requests are greedy and the others sample
        _logits("choose", "choose full batch", 256, 131072, "bf16", hist=4096, prompt=True, sparse=300, mask="words", draw="mixed"),
        # a policy over 64 candidates learning from a teacher's best 8
        _distill("distill candidates", 8192, 64, "f32", 8, "logits", "grad", temperature=2.0),
        # validation loss of a student over a large vocabulary, the teacher's remaining mass as one class
        _distill("distill value", 2048, 131072, "bf16", 64, "logprobs", "value", wide_ids=True),
        # an ordinary training batch: padded positions carry no weight, the teacher's lists are ragged
        _distill("distill training batch", 4096, 32000, "bf16", 64, "logits", "grad", weights=True, ragged=True, temperature=2.0),
        # a float32 student with an odd vocabulary, through autograd
        _distill("distill odd autograd", 1024, 50001, "f32", 50, "logprobs", "autograd", weights=True),
        # the last positions of a few sequences
        _distill("distill few rows", 3, 200001, "f16", 20, "logits", "grad"),
        # the largest training batch
        _distill("distill large batch", 8192, 131072, "bf16", 128, "logprobs", "grad", weights=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["constrain", "choose", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    vocab = _log_between(rng, 32, 200000)
    if op == "distill":
        rows = _log_between(rng, 1, max(2, min(16384, 600_000_000 // vocab)))
        top = min(_log_between(rng, 1, 256), vocab // 2)
        case = _distill("", rows, vocab, dtype, top, rng.choice(["logits", "logprobs"]), rng.choice(["value", "grad", "autograd"]),
                        weights=rng.random() < 0.5, wide_ids=rng.random() < 0.5, ragged=rng.random() < 0.5,
                        temperature=rng.choice([1.0, 1.0, 2.0, 0.7]))
        del case["name"]
        return case
    rows = _log_between(rng, 1, max(2, min(8192, 60_000_000 // vocab)))
    hist = 0 if rng.random() < 0.25 else min(_log_between(rng, 1, 16384), max(1, 30_000_000 // rows))
    sparse = 0 if rng.random() < 0.4 else min(_log_between(rng, 1, 512), vocab // 2)
    case = _logits(op, "", rows, vocab, dtype, hist=hist, prompt=rng.random() < 0.5, wide_ids=rng.random() < 0.5, sparse=sparse,
                   dense=rng.random() < 0.3, mask=rng.choice(["none", "words", "bool"]), out=rng.choice(["same", "f32"]),
                   draw=rng.choice(["greedy", "mixed", "all"]))
    del case["name"]
    return case


def _distinct(gen, rows, count, vocab):
    """(rows, count) distinct tokens of a row in no order: one out of each of ``count`` equal stretches, in an order of the row's own."""
    u = torch.rand((rows, count), generator=gen, device="cuda", dtype=torch.float64)
    at = torch.arange(count, device="cuda", dtype=torch.float64)
    lo, hi = (at * vocab / count).ceil(), ((at + 1) * vocab / count).ceil()
    # a device's quotient can be a rounding above vocab at the last end (32000 * 300 / 300), one token too many
    ids = torch.minimum((lo + u * (hi - lo)).floor(), hi - 1).clamp_(max=vocab - 1).long()
    order = torch.rand((rows, count), generator=gen, device="cuda").argsort(dim=1)
    return ids.gather(1, order)


def _prepare_logits(case, gen):
    R, V, L, dev = case["rows"], case["vocab"], case["hist"], "cuda"
    rand = lambda *s: torch.rand(s, generator=gen, device=dev)  # noqa: E731
    z = torch.randn((R, V), generator=gen, device=dev).mul_(4.0)
    z[:, V - V // 50:] = -math.inf                       # entries that pad the vocabulary to a round size
    s = {"case": case, "z": z.to(DTYPES[case["dtype"]])}
    ids = torch.int64 if case["wide_ids"] else torch.int32
    if L:
        s["history"] = (V * rand(R, L) ** 3).long().clamp_(max=V - 1).to(ids)      # some tokens come again and again
        s["lengths"] = (rand(R) * (L + 1)).long().clamp_(max=L).to(torch.int32)
        s["lengths"][0] = L
        if case["prompt"]:
            s["prompt_lengths"] = (s["lengths"] * rand(R)).to(torch.int32)
        s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.5 * rand(R), 0.3 * rand(R), rand(R) - 0.3
    if case["dense"]:
        s["bias"] = torch.randn((V,), generator=gen, device=dev)
    if case["sparse"]:
        s["bias_tokens"] = _distinct(gen, R, case["sparse"], V).to(ids)
        s["bias_values"] = torch.randn((R, case["sparse"]), generator=gen, device=dev) * 5.0
    if case["mask"] != "none":
        share = torch.tensor([0.02, 0.9, 0.5, 1.0], device=dev)[(torch.arange(R, device=dev) + 1) % 4]
        allowed = rand(R, V) < share[:, None]
        if R > 4:
            allowed[R // 2] = False                      # a request whose rules leave nothing
        if case["mask"] == "words":
            W = -(-V // 32)
            bits = torch.zeros((R, W * 32), dtype=torch.int64, device=dev)
            bits[:, :V] = allowed
            words = (bits.view(R, W, 32) << torch.arange(32, device=dev)).sum(-1)
            allowed = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        s["allowed"] = allowed
    if case["op"] == "choose":
        temperature = 0.3 + rand(R)
        greedy = {"greedy": 1, "mixed": 8, "all": R + 1}[case["draw"]]
        temperature[greedy - 1::greedy] = 0.0
        s["temperature"] = temperature
        if case["draw"] != "greedy":
            u = torch.rand((R, V), generator=gen, device=dev).clamp_(min=1e-30, max=1.0 - 6e-8)
            s["gumbel"] = u.log_().neg_().log_().neg_()
    return s


def _prepare_distill(case, gen):
    N, V, K, dev = case["rows"], case["vocab"], case["top"], "cuda"
    z = torch.randn((N, V), generator=gen, device=dev, dtype=DTYPES[case["dtype"]]).mul_(2.0)
    ids = _distinct(gen, N, K, V)
    lift = 4.0 + 2.0 * torch.randn((N, K), generator=gen, device=dev)
    z.scatter_add_(1, ids, lift.to(z.dtype))             # a student that already agrees in part
    t = lift + torch.randn((N, K), generator=gen, device=dev) + 6.0
    s = {"case": case, "z": z, "weights": None}
    if case["kind"] == "logprobs":
        mass = 0.5 + 0.499 * torch.rand((N, 1), generator=gen, device=dev)
        t = torch.log_softmax(t.double(), -1).add(mass.double().log()).float()
    if case["ragged"]:
        ids = torch.where(torch.arange(K, device=dev) < 1 + (torch.rand((N, 1), generator=gen, device=dev) * K).long(), ids, -1)
    if case["weights"]:
        s["weights"] = torch.rand((N,), generator=gen, device=dev).add_(0.5)
        s["weights"][1::8] = 0.0
    s["ids"], s["teacher"] = ids.to(torch.int64 if case["wide_ids"] else torch.int32), t
    if case["how"] == "autograd":
        z.requires_grad_(True)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    return _prepare_distill(case, gen) if case["op"] == "distill" else _prepare_logits(case, gen)


# ---- plain forms ---------------------------------------------------------------------------------------------------------

def _plain_constrained(s):
    case, z = s["case"], s["z"].float()
    R, V = z.shape
    if case["hist"]:
        L = case["hist"]
        at, ids = torch.arange(L, device=z.device), s["history"].long()
        live = at < s["lengths"][:, None]
        counts = torch.zeros((R, V), device=z.device)
        if case["prompt"]:
            made = live & (at >= s["prompt_lengths"][:, None])
            seen = torch.zeros((R, V), device=z.device).scatter_add_(1, ids, live.float()) > 0
            counts.scatter_add_(1, ids, made.float())
        else:
            counts.scatter_add_(1, ids, live.float())
            seen = counts > 0
        rep = s["repetition"][:, None]
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
        z = z - (s["frequency"][:, None] * counts + torch.where(counts > 0, s["presence"][:, None], 0.0))
    if case["dense"]:
        z = z + s["bias"]
    if case["sparse"]:
        z = z + torch.zeros_like(z).scatter_add_(1, s["bias_tokens"].long(), s["bias_values"])
    if case["mask"] != "none":
        allowed = s["allowed"]
        if case["mask"] == "words":
            allowed = ((allowed[:, :, None] >> torch.arange(32, device=z.device)) & 1).view(R, -1)[:, :V] != 0
        z = torch.where(allowed, z, -math.inf)
    return z


def _plain_choose(s):
    z = _plain_constrained(s)
    sampled = s["temperature"][:, None] > 0
    y = torch.where(sampled, z * (1.0 / (1e-6 + s["temperature"][:, None])), z)
    key = torch.where(sampled, y + s["gumbel"], z) if "gumbel" in s else z
    token = key.argmax(dim=1)
    m = y.amax(dim=1, keepdim=True)
    logprob = y.gather(1, token[:, None]) - m - (y - m).exp().sum(dim=1, keepdim=True).log()
    empty = m[:, 0] == -math.inf
    return {"token": torch.where(empty, -1, token).to(torch.int32), "logprob": torch.where(empty, -math.inf, logprob[:, 0])}


def _plain_distill(s):
    case, T = s["case"], s["case"]["temperature"]
    y = s["z"].detach().float() / T
    valid = s["ids"] >= 0
    ids = s["ids"].long().clamp(min=0)
    t = torch.where(valid, s["teacher"].double(), -math.inf)
    w = s["weights"] if s["weights"] is not None else torch.ones(y.shape[0], device=y.device)
    m = y.amax(dim=1, keepdim=True)
    e = (y - m).exp()
    total = e.sum(dim=1, keepdim=True)
    logq = y.gather(1, ids) - m - total.log()
    if case["kind"] == "logits":
        t = t / T
        t = t - t.amax(dim=1, keepdim=True)
        logp = t - t.exp().sum(dim=1, keepdim=True).log()
    else:
        logp = t
    p = logp.exp()
    row = torch.where(p > 0, p * (logp - logq), 0.0).sum(dim=1)
    coef = torch.ones_like(total)
    if case["kind"] == "logprobs":
        top = torch.zeros(y.shape, dtype=torch.bool, device=y.device)
        at = torch.nonzero(valid)
        top[at[:, 0], ids[at[:, 0], at[:, 1]]] = True
        rest_q = torch.where(top, 0.0, e).sum(dim=1, keepdim=True) / total
        rest_p = 1.0 - p.sum(dim=1, keepdim=True)
        rest = rest_p > 0
        row = row + torch.where(rest, rest_p * (rest_p.log() - rest_q.log()), 0.0)[:, 0]
        coef = torch.where(rest, 1.0 - rest_p / rest_q, p.sum(dim=1, keepdim=True)).float()
    row = row.float()
    if case["how"] == "value":
        return {"rows": row * w}
    scale = 1.0 / w.sum()
    loss = (row * w).sum() * scale
    q = e / total
    if case["kind"] == "logits":
        g = q.scatter_add(1, ids, -p.float())
    else:
        g = torch.where(top, q, coef * q).scatter_add(1, ids, torch.where(valid, -p, 0.0).float())
    return {"loss": loss, "grad": (g * (w * scale / T)[:, None]).to(s["z"].dtype)}


# ---- the framework's calls -----------------------------------------------------------------------------------------------

def _framework():
    if "flowrl_hip" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "flow-rl_amd"))
    import flowrl_hip
    return flowrl_hip


RULES = ("history", "lengths", "prompt_lengths", "repetition", "frequency", "presence", "bias", "bias_tokens", "bias_values", "allowed")


def _own(s):
    fh, case = _framework(), s["case"]
    if case["op"] == "distill":
        how = dict(kind=case["kind"], temperature=case["temperature"], weights=s["weights"])
        if case["how"] == "value":
            return {"rows": fh.logits.distill_loss(s["z"], s["ids"], s["teacher"], reduction="none", **how)}
        if case["how"] == "grad":
            loss, grad = fh.logits.distill_loss(s["z"], s["ids"], s["teacher"], want_grad=True, **how)
        else:
            loss = fh.autograd.distill_loss(s["z"], s["ids"], s["teacher"], **how)
            grad, = torch.autograd.grad(loss, s["z"])
            loss = loss.detach()
        return {"loss": loss, "grad": grad}
    rules = fh.logits.Constraints(**{k: s[k] for k in RULES if k in s})
    if case["op"] == "constrain":
        return fh.logits.constrain(s["z"], rules, out_dtype=torch.float32 if case["out"] == "f32" else None)
    token, logprob = fh.logits.choose(s["z"], rules, temperature=s["temperature"], gumbel=s.get("gumbel"))
    return {"token": token, "logprob": logprob}


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "distill":
        return _plain_distill(state)
    if case["op"] == "choose":
        return _plain_choose(state)
    z = _plain_constrained(state)
    return z if case["out"] == "f32" else z.to(state["z"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    R, V, size = case["rows"], case["vocab"], SIZE[case["dtype"]]
    idsize = 8 if case["wide_ids"] else 4
    if case["op"] == "distill":
        passes = 1 if case["how"] == "value" else 2
        return {"bytes": R * V * size * passes + R * case["top"] * (idsize + 4) + 8 * R, "flops": R * V * (4 if passes == 1 else 7)}
    small = R * (case["hist"] * idsize // 2 + case["sparse"] * (idsize + 4) + 24)     # a history is half full on the average
    small += (4 * V if case["dense"] else 0) + {"none": 0, "words": R * V // 8, "bool": R * V}[case["mask"]]
    if case["op"] == "constrain":
        return {"bytes": R * V * (size + (4 if case["out"] == "f32" else size)) + small, "flops": 6 * R * V}
    sampled = {"greedy": 0, "mixed": R - R // 8, "all": R}[case["draw"]]
    return {"bytes": R * V * size + 4 * sampled * V + small + 8 * R, "flops": 10 * R * V}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_row(s, r):
    """One row of the constrained logits: one token's rules after the other, by counts of the row's own lists."""
    case, V = s["case"], s["case"]["vocab"]
    x = s["z"][r].double()
    if case["hist"]:
        n = int(s["lengths"][r])
        first = int(s["prompt_lengths"][r]) if case["prompt"] else 0
        told = s["history"][r, :n].long()
        c = torch.bincount(told[first:], minlength=V).double()
        seen = torch.bincount(told, minlength=V) > 0
        rep, freq, pres = (s[k][r].double() for k in ("repetition", "frequency", "presence"))
        pushed = torch.maximum(x, torch.zeros_like(x)) / rep + torch.minimum(x, torch.zeros_like(x)) * rep
        x = torch.where(seen, pushed, x) - freq * c - pres * c.clamp(max=1.0)
    if case["dense"]:
        x = x + s["bias"].double()
    if case["sparse"]:
        x = x.index_add(0, s["bias_tokens"][r].long(), s["bias_values"][r].double())
    if case["mask"] == "bool":
        x = x.masked_fill(~s["allowed"][r], -math.inf)
    elif case["mask"] == "words":
        v = torch.arange(V, device=x.device)
        x = x.masked_fill((s["allowed"][r].long()[v // 32] >> (v % 32)) % 2 == 0, -math.inf)
    return x


def _exact_logits(s):
    case, R = s["case"], s["case"]["rows"]
    if case["op"] == "constrain":
        return torch.stack([_exact_row(s, r) for r in range(R)])
    token, logprob, clear = [], [], True
    for r in range(R):
        x = _exact_row(s, r)
        if bool((x == -math.inf).all()):
            token.append(-1)
            logprob.append(-math.inf)
            continue
        T = float(s["temperature"][r])
        y = x / (1e-6 + T) if T > 0 else x
        key = y + s["gumbel"][r].double() if T > 0 else y
        best = key.topk(2)
        at = int((key == best.values[0]).nonzero()[0])
        gap = float(best.values[0] - best.values[1])
        clear = clear and (gap > 3e-5 or (T <= 0 and gap == 0.0))
        token.append(at)
        logprob.append(float(y[at] - torch.logsumexp(y, 0)))
    # a row whose two best keys differ by less than float32 resolves has no certain choice
    return {"token": torch.tensor(token, dtype=torch.int32) if clear else None, "logprob": torch.tensor(logprob, dtype=torch.float64)}


def _exact_distill(s):
    case, T = s["case"], s["case"]["temperature"]
    N, V, dev = case["rows"], case["vocab"], s["z"].device
    w = s["weights"].double() if s["weights"] is not None else torch.ones(N, dtype=torch.float64, device=dev)
    value, grads = [], []
    step = max(1, 100_000_000 // V)
    for a in range(0, N, step):
        z = s["z"].detach()[a:a + step].double()
        logq = torch.log_softmax(z / T, dim=1)
        n = z.shape[0]
        ids, t = s["ids"][a:a + step].long(), s["teacher"][a:a + step].double()
        if case["kind"] == "logits":
            logp = torch.log_softmax((t / T).masked_fill(ids < 0, -math.inf), dim=1)
        else:
            logp = t.masked_fill(ids < 0, -math.inf)
        # the teacher's distribution laid out over the vocabulary and one column for tokens that are none
        p = torch.zeros((n, V + 1), dtype=torch.float64, device=dev)
        p.scatter_(1, torch.where(ids < 0, V, ids), logp.exp())
        p = p[:, :V]
        named = torch.zeros((n, V + 1), dtype=torch.bool, device=dev).scatter_(1, torch.where(ids < 0, V, ids), True)[:, :V]
        row = (torch.special.xlogy(p, p) - p * logq).sum(1)
        g = p.sum(1, keepdim=True) * logq.exp() - p
        if case["kind"] == "logprobs":
            P = 1.0 - p.sum(1)
            Q = torch.logsumexp(logq.masked_fill(named, -math.inf), dim=1)
            some = P > 0
            row = row + torch.where(some, P * (torch.log(P) - Q), 0.0)
            inside = logq - Q[:, None]
            g = g + torch.where(some[:, None], P[:, None] * (logq.exp() - torch.where(named, 0.0, inside.exp())), 0.0)
        value.append(row)
        if case["how"] != "value":
            grads.append(g * (w[a:a + step, None] / (w.sum() * T)))
    value = torch.cat(value)
    if case["how"] == "value":
        return {"rows": value * w}
    return {"loss": (value * w).sum() / w.sum(), "grad": torch.cat(grads) if len(grads) > 1 else grads[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_distill(s) if case["op"] == "distill" else _exact_logits(s)
