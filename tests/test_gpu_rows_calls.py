"""GPU: calls on rows of logits that lie in memory, or are made, in ways of their own."""
import ctypes as C

import numpy as np
import pytest

from logits_cases import make_distill, make_rules, rules_to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("R,V", [(7, 1000), (5, 40), (3, 9001), (300, 4099)])
def test_results_between_the_logits_rows(R, V, gap):
    """Column blocks of one buffer: no entry is shared, and the logits and what lies beside the blocks stay as they are."""
    import torch
    import flowrl_hip as fh
    from flowrl_hip import _lib
    rng = np.random.default_rng(V)
    for dtype in (torch.float32, torch.bfloat16):
        rules = rules_to_gpu(fh, make_rules(rng, R, V, hist=20, sparse=5, mask="words"), "words")
        z = torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32)).to(dtype).cuda()
        want = fh.logits.constrain(z, rules)
        ids, t = make_distill(rng, R, V, 6, "logits", dtype)[1:]
        ids, t = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
        loss, grad = fh.logits.distill_loss(z, ids, t, want_grad=True, reduction="sum")
        for first in (True, False):
            buf = torch.full((R, 2 * (V + gap)), 5.0, dtype=dtype, device="cuda")
            a, b = buf[:, :V], buf[:, V + gap:2 * V + gap]
            src, dst = (a, b) if first else (b, a)
            src.copy_(z)
            assert fh.logits.constrain(src, rules, out=dst) is dst
            assert torch.equal(dst, want) and torch.equal(src, z)
            rest = torch.ones(2 * (V + gap), dtype=torch.bool, device="cuda")
            rest[:V] = rest[V + gap:2 * V + gap] = False
            assert (buf[:, rest] == 5.0).all()
            # the gradient, through the C entry point (the Python one allocates it)
            out = torch.empty((), device="cuda")
            dst.fill_(7.0)
            d, bufs, keep = fh.logits._distill_marshal(src, ids, t, "logits", 1.0, None, "sum", out.data_ptr(), 0, 0, dst.data_ptr())
            d.grad_stride = dst.stride(0)
            lib = _lib.load()
            ws = torch.empty(lib.frl_distill_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
            _lib.check(lib.frl_distill_fwd(C.byref(d), C.byref(bufs), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
            # where a row starts decides the order of its sum: 2^-16 is far above its rounding and far below a misplaced entry
            assert torch.equal(src, z) and (buf[:, rest] == 5.0).all()
            assert abs(float(out - loss)) <= 2.0 ** -16 * R * 10
            assert float((dst.float() - grad.float()).abs().max()) <= (2.0 ** -16 if dtype == torch.float32 else 2.0 ** -8)


def _built():
    from flowrl_hip import _lib
    return _lib.load().frl_last_kernels().decode()


@pytest.mark.parametrize("N,V,value,grad", [(70000, 100, 16, 64), (70000, 300, 64, 64), (600, 5001, 512, 1024), (2048, 3001, 256, 256), (300, 70001, 1024, 1024), (3, 50001, 256, 256)])
def test_the_builds_that_are_named_are_those_that_ran(N, V, value, grad):
    """frl_last_kernels after the forward and after the backward."""
    import torch
    import flowrl_hip as fh
    z = torch.zeros((N, V), dtype=torch.bfloat16, device="cuda")
    ids, t = torch.zeros((N, 1), dtype=torch.int32, device="cuda"), torch.zeros((N, 1), device="cuda")
    loss, _, stats = fh.logits.distill_forward(z, ids, t, "logits", 1.0, None, "sum", want_stats=True)
    forward = _built()
    fh.logits.distill_backward(z, ids, t, "logits", 1.0, None, "sum", stats, torch.ones((), device="cuda"))
    backward = _built()
    assert f"<value, {value} threads" in forward or (N < 256 and "frl_distill_part_kernel" in forward), forward
    assert f"frl_distill_grad_kernel<{grad} threads>" in backward, backward


def test_listed_tokens_at_equal_distances():
    """Tokens a multiple of 8192 apart, as rows of a product vocabulary have them, cost what other tokens do.  Measured 1.1 times as much; where they all began
    at one place of the table of tokens, 75 times: 3 is between."""
    import torch
    import flowrl_hip as fh
    K, step = 1000, 8192
    V = K * step
    z = torch.randn((1, V), device="cuda").to(torch.bfloat16)
    values = torch.randn(K, device="cuda")
    took = {}
    for name, tokens in (("apart", torch.randperm(V, device="cuda")[:K]), ("equal", torch.randperm(K, device="cuda") * step)):
        rules = fh.logits.Constraints(bias_tokens=tokens, bias_values=values)
        want = z.float()
        want[0, tokens] += values
        assert torch.equal(fh.logits.constrain(z, rules, out_dtype=torch.float32), want)
        for _ in range(5):
            fh.logits.choose(z, rules)
        times = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                fh.logits.choose(z, rules)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        took[name] = sorted(times)[3]
    print(took)
    assert took["equal"] < 3 * took["apart"], took
