"""Inputs shared by the tests of the operators over rows of logits."""
import numpy as np
import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # the smallest subnormal step


def pack_words(allowed: np.ndarray) -> np.ndarray:
    lead, V = allowed.shape[:-1], allowed.shape[-1]
    bits = np.zeros((*lead, (V + 31) // 32 * 32), np.uint64)
    bits[..., :V] = allowed
    words = (bits.reshape(*lead, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return words.astype(np.uint32).view(np.int32)


def make_rules(rng, R, V, *, hist=0, prompt=False, sparse=0, dense=None, mask=None, wide=False, tensors=True):
    """Rules as numpy arrays (the oracle's keyword arguments).  Tokens repeat, some lie outside the vocabulary, lengths run from 0 to full."""
    ids = np.int64 if wide else np.int32
    c = {}
    if hist:
        h = (rng.random((R, hist)) ** 3 * V).astype(ids)
        h[rng.random((R, hist)) < 0.05] = -1
        h[rng.random((R, hist)) < 0.05] = V
        c["history"] = h
        c["lengths"] = rng.integers(0, hist + 1, R).astype(np.int32)
        c["lengths"][0] = hist
        if R > 2:
            c["lengths"][1], c["lengths"][2] = 0, 1
        if prompt:
            c["prompt_lengths"] = rng.integers(0, hist + 1, R).astype(np.int32)
        c["repetition"] = (0.6 + rng.random(R)).astype(np.float32) if tensors else 1.25
        c["frequency"] = rng.standard_normal(R).astype(np.float32) if tensors else 0.5
        c["presence"] = rng.standard_normal(R).astype(np.float32) if tensors else -0.25
    if dense:
        c["bias"] = rng.standard_normal((V,) if dense == "shared" else (R, V)).astype(np.float32)
    if sparse:
        t = rng.integers(-1, V + 1, (R, sparse)).astype(ids)      # repeats and padding
        c["bias_tokens"], c["bias_values"] = t, (3 * rng.standard_normal((R, sparse))).astype(np.float32)
    if mask:
        a = rng.random((R, V)) < rng.choice([0.02, 0.5, 0.97], (R, 1))
        if R > 3:
            a[3] = False
        c["allowed"] = a
    return c


def rules_to_gpu(fh, c, mask):
    t = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() if isinstance(v, np.ndarray) else v for k, v in c.items() if k != "allowed"}
    if "allowed" in c:
        t["allowed"] = torch.from_numpy(pack_words(c["allowed"]) if mask == "words" else np.ascontiguousarray(c["allowed"])).cuda()
    return fh.logits.Constraints(**t)


def make_distill(rng, N, V, K, kind, dtype, *, ragged=False, repeats=False, wide=False):
    z = torch.from_numpy((2.0 * rng.standard_normal((N, V))).astype(np.float32)).to(dtype)
    ids = np.stack([rng.choice(V, K, replace=False) for _ in range(N)]) if not repeats else rng.integers(0, V, (N, K))
    t = 3.0 * rng.standard_normal((N, K))
    if kind == "logprobs":
        mass = 0.2 + 0.79 * rng.random((N, 1))
        t = t - np.log(np.exp(t).sum(1, keepdims=True)) + np.log(mass)
    if ragged:
        drop = np.arange(K) >= 1 + (rng.random((N, 1)) * K).astype(int)
        ids = np.where(drop, rng.choice([-1, V, V + 5], (N, K)), ids)
    return z, ids.astype(np.int64 if wide else np.int32), t.astype(np.float32)
