"""CPU: the operators over rows of logits at their boundary — struct layouts, refusals before any launch, argument checks of the Python
side — and the float64 restatement they are tested against, itself checked by hand-made rows and by differences."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import flowrl_hip as fh
import logits_oracle as orc
from flowrl_hip import _lib
from logits_cases import make_distill, make_rules, pack_words

ROOT = Path(__file__).resolve().parent.parent


def _desc(**kw):
    d = _lib.FrlLogitsDesc()
    d.abi_version, d.dtype, d.out_dtype, d.vocab, d.rows = _lib.FRL_ABI_VERSION, _lib.FRL_ELT_BF16, _lib.FRL_ELT_F32, 32000, 4
    d.logits_stride = d.out_stride = d.gumbel_stride = 32000
    d.repetition = 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _bufs(**kw):
    b = _lib.FrlLogitsBufs()
    b.logits, b.out, b.token = 1 << 20, 1 << 30, 1 << 12      # never dereferenced: every call below is refused
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def _ddesc(**kw):
    d = _lib.FrlDistillDesc()
    d.abi_version, d.vocab, d.top, d.rows, d.temperature, d.reduction = _lib.FRL_ABI_VERSION, 32000, 64, 4, 1.0, _lib.FRL_REDUCE_MEAN
    d.logits_stride = d.grad_stride = 32000
    d.ids_stride = d.teacher_stride = 64
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _dbufs(**kw):
    b = _lib.FrlDistillBufs()
    b.logits, b.ids, b.teacher, b.loss, b.grad, b.row_stats, b.g_loss = 1 << 20, 1 << 12, 1 << 13, 1 << 14, 1 << 30, 1 << 16, 1 << 15
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc is not available")
    structs = ("FrlLogitsDesc", "FrlLogitsBufs", "FrlDistillDesc", "FrlDistillBufs")
    lines = []
    for s in structs:
        lines.append(f'printf("%zu\\n", sizeof({s}));')
        lines += [f'printf("%zu\\n", offsetof({s}, {f}));' for f, _ in getattr(_lib, s)._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "flowrl_hip.h"\nint main(void) {' + "".join(lines) + "return 0; }\n")
    subprocess.run([gcc, f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for s in structs:
        t = getattr(_lib, s)
        want += [C.sizeof(t), *[getattr(t, f).offset for f, _ in t._fields_]]
    assert got == want


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=5), _lib.FRL_EINVAL), (dict(dtype=3), _lib.FRL_EINVAL), (dict(dtype=-1), _lib.FRL_EINVAL),
    (dict(out_dtype=_lib.FRL_ELT_F16), _lib.FRL_EINVAL), (dict(vocab=0), _lib.FRL_EINVAL), (dict(rows=-1), _lib.FRL_EINVAL),
    (dict(history_len=-1), _lib.FRL_EINVAL), (dict(n_sparse=-1), _lib.FRL_EINVAL), (dict(n_sparse=2049), _lib.FRL_EUNSUPPORTED),
    (dict(mask=3), _lib.FRL_EINVAL), (dict(vocab=(1 << 30) + 1, logits_stride=1 << 31, out_stride=1 << 31), _lib.FRL_EUNSUPPORTED),
    (dict(rows=1 << 40), _lib.FRL_EUNSUPPORTED), (dict(n_sparse=4, history_len=1 << 19), _lib.FRL_EUNSUPPORTED), (dict(logits_stride=31999), _lib.FRL_EINVAL), (dict(out_stride=31999), _lib.FRL_EINVAL),
    (dict(history_len=4), _lib.FRL_EINVAL), (dict(n_sparse=4), _lib.FRL_EINVAL), (dict(mask=1), _lib.FRL_EINVAL),
])
def test_constrain_refuses(lib, kw, code):
    d, b = _desc(**kw), _bufs()
    assert lib.frl_logits_constrain(C.byref(d), C.byref(b), None) == code
    assert lib.frl_last_error() != b""


@pytest.mark.parametrize("kw", [dict(logits=None), dict(out=None), dict(allowed=1 << 13), dict(out=(1 << 20) + 64), dict(out=1 << 20), dict(out=(1 << 20) - 64)])
def test_constrain_refuses_buffers(lib, kw):
    d, b = _desc(), _bufs(**kw)
    assert lib.frl_logits_constrain(C.byref(d), C.byref(b), None) == _lib.FRL_EINVAL
    d = _desc(history_len=3, repetition=0.0)
    assert lib.frl_logits_constrain(C.byref(d), C.byref(_bufs(history=1 << 13)), None) == _lib.FRL_EINVAL
    assert b"repetition" in lib.frl_last_error()
    assert lib.frl_logits_constrain(None, C.byref(b), None) == _lib.FRL_EINVAL
    assert lib.frl_logits_constrain(C.byref(_desc()), None, None) == _lib.FRL_EINVAL


def test_choose_refuses(lib):
    d = _desc()
    need = lib.frl_logits_workspace_bytes(C.byref(d))
    assert need > 0 and need % 256 == 0
    for b, ws, n, code in ((_bufs(token=None), 4096, need, _lib.FRL_EINVAL), (_bufs(), None, need, _lib.FRL_EWORKSPACE), (_bufs(), 4100, need, _lib.FRL_EWORKSPACE),
                           (_bufs(), 4096, need - 1, _lib.FRL_EWORKSPACE)):
        assert lib.frl_logits_choose(C.byref(d), C.byref(b), ws, n, None) == code
    d = _desc(temperature=0.5)                      # draws without noise
    assert lib.frl_logits_choose(C.byref(d), C.byref(_bufs()), 4096, need, None) == _lib.FRL_EINVAL
    assert b"gumbel" in lib.frl_last_error()
    d = _desc(gumbel_stride=3)
    assert lib.frl_logits_choose(C.byref(d), C.byref(_bufs(gumbel=1 << 25)), 4096, need, None) == _lib.FRL_EINVAL
    assert lib.frl_logits_workspace_bytes(C.byref(_desc(vocab=-2))) == 0
    d = _desc(rows=0)
    assert lib.frl_logits_choose(C.byref(d), C.byref(_bufs()), None, 0, None) == _lib.FRL_OK


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=5), _lib.FRL_EINVAL), (dict(dtype=3), _lib.FRL_EINVAL), (dict(teacher_dtype=-1), _lib.FRL_EINVAL), (dict(kind=2), _lib.FRL_EINVAL),
    (dict(reduction=3), _lib.FRL_EINVAL), (dict(rows=-1), _lib.FRL_EINVAL), (dict(vocab=0), _lib.FRL_EINVAL), (dict(top=0), _lib.FRL_EINVAL),
    (dict(top=1025), _lib.FRL_EUNSUPPORTED), (dict(temperature=0.0), _lib.FRL_EINVAL), (dict(temperature=float("nan")), _lib.FRL_EINVAL), (dict(temperature=float("inf")), _lib.FRL_EINVAL), (dict(temperature=1e-38), _lib.FRL_EINVAL),
    (dict(vocab=(1 << 30) + 1), _lib.FRL_EUNSUPPORTED), (dict(rows=(1 << 30) + 1), _lib.FRL_EUNSUPPORTED), (dict(logits_stride=31999), _lib.FRL_EINVAL),
    (dict(grad_stride=31999), _lib.FRL_EINVAL),
])
def test_distill_refuses(lib, kw, code):
    d, b = _ddesc(**kw), _dbufs()
    assert lib.frl_distill_fwd(C.byref(d), C.byref(b), 4096, 1 << 30, None) == code
    assert lib.frl_last_error() != b""
    assert lib.frl_distill_bwd(C.byref(d), C.byref(b), None) == code


def test_distill_refuses_buffers(lib):
    d = _ddesc()
    need = lib.frl_distill_workspace_bytes(C.byref(d))
    assert need > 0
    for kw in (dict(logits=None), dict(ids=None), dict(teacher=None), dict(loss=None), dict(grad=(1 << 20) + 128), dict(row_stats=(1 << 16) + 4)):
        assert lib.frl_distill_fwd(C.byref(d), C.byref(_dbufs(**kw)), 4096, need, None) == _lib.FRL_EINVAL, kw
    for kw in (dict(logits=None), dict(ids=None), dict(teacher=None), dict(row_stats=None), dict(g_loss=None), dict(grad=None), dict(grad=1 << 20), dict(row_stats=(1 << 16) + 4)):
        assert lib.frl_distill_bwd(C.byref(d), C.byref(_dbufs(**kw)), None) == _lib.FRL_EINVAL, kw
    for ws, n in ((None, need), (4100, need), (4096, need - 1)):
        assert lib.frl_distill_fwd(C.byref(d), C.byref(_dbufs()), ws, n, None) == _lib.FRL_EWORKSPACE
    assert lib.frl_distill_bwd(C.byref(_ddesc(rows=0)), C.byref(_dbufs()), None) == _lib.FRL_OK


def test_host_tensors_and_wrong_arguments_are_refused():
    z = torch.zeros((2, 8))
    for call in (lambda: fh.logits.constrain(z), lambda: fh.logits.choose(z), lambda: fh.logits.distill_loss(z, torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1))),
                 lambda: fh.autograd.distill_loss(z.requires_grad_(True), torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
        z = torch.zeros((2, 8))
    with pytest.raises(ValueError, match="kind"):
        fh.logits.distill_loss(z, torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)), kind="soft")
    with pytest.raises(ValueError, match="reduction"):
        fh.logits.distill_loss(z, torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)), reduction="batchmean")
    with pytest.raises(NotImplementedError, match="detach"):
        fh.logits.choose(torch.zeros((2, 8), requires_grad=True))
    with pytest.raises(NotImplementedError, match="detach"):
        fh.logits.choose(torch.zeros((2, 8)), temperature=torch.ones(2, requires_grad=True))
    with pytest.raises(NotImplementedError, match="detach"):
        fh.logits.constrain(torch.zeros((2, 8)), fh.logits.Constraints(repetition=torch.ones(2, requires_grad=True)))


def test_marshalling_refuses_shapes_and_types():
    """The checks that run before a pointer is taken, on host tensors."""
    z, Cn = torch.zeros((3, 40)), fh.logits.Constraints
    m = lambda **kw: fh.logits._marshal(z, 3, 40, Cn(**kw))  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for kw, err in [
        (dict(history=torch.zeros((3, 5))), TypeError), (dict(history=i32(2, 5)), ValueError), (dict(history=i32(15)), ValueError),
        (dict(lengths=i32(3)), ValueError), (dict(history=i32(3, 5), lengths=torch.zeros(3, dtype=torch.int64)), TypeError),
        (dict(history=i32(3, 5), lengths=i32(2)), TypeError), (dict(history=i32(3, 5), repetition=torch.ones(2)), TypeError),
        (dict(history=i32(3, 5), presence=torch.ones(3, dtype=torch.float64)), TypeError),
        (dict(bias=torch.zeros(39)), ValueError), (dict(bias=torch.zeros((2, 40))), ValueError), (dict(bias=torch.zeros(40, dtype=torch.float16)), TypeError),
        (dict(bias_tokens=i32(3, 4)), ValueError), (dict(bias_values=torch.zeros((3, 4))), ValueError),
        (dict(bias_tokens=i32(3, 4), bias_values=torch.zeros((3, 5))), TypeError), (dict(bias_tokens=torch.zeros((3, 4)), bias_values=torch.zeros((3, 4))), TypeError),
        (dict(allowed=torch.ones((3, 40))), TypeError), (dict(allowed=torch.ones((3, 39), dtype=torch.bool)), ValueError), (dict(allowed=i32(3, 40)), ValueError),
    ]:
        with pytest.raises(err):
            m(**kw)
    d, b, keep = m(history=i32(3, 5), bias_tokens=torch.zeros((4,), dtype=torch.int64), bias_values=torch.zeros(4), allowed=i32(2))
    assert d.ids64 == 1 and d.history_len == 5 and d.n_sparse == 4 and d.sparse_stride == 0 and d.mask_stride == 0 and d.mask == _lib.FRL_MASK_WORDS
    d, b, keep = m(bias_tokens=i32(1, 4).expand(3, 4), bias_values=torch.zeros((3, 4)), allowed=torch.ones((3, 40), dtype=torch.bool), bias=torch.zeros((1, 40)).expand(3, 40))
    assert d.sparse_stride == 4 and d.mask_stride == 40 and d.bias_stride == 0


def test_words_hold_the_bits():
    a = np.zeros((2, 70), bool)
    a[0, [0, 31, 32, 69]] = True
    w = pack_words(a)
    assert w.shape == (2, 3) and w[0].tolist() == [1 - (1 << 31), 1, 1 << 5] and not w[1].any()


def test_oracle_by_hand():
    z = np.array([[2.0, -2.0, 0.5, 1.0, 3.0]])
    x, _ = orc.constrain_row(z, 0, history=np.array([[0, 1, 1, 7, 2]]), lengths=[4], prompt_lengths=[1], repetition=2.0, frequency=0.5, presence=0.25,
                             bias_tokens=np.array([3, 3, 9]), bias_values=np.array([1.0, 2.0, 5.0]), allowed=np.array([True, True, True, True, False]))
    np.testing.assert_array_equal(x, [1.0, -4.0 - 1.0 - 0.25, 0.5, 4.0, -np.inf])
    v, lp = orc.choose_row(*orc.keys_of(np.array([0.0, np.log(3.0), -np.inf]), 0.0, None))
    assert v == 1 and abs(lp - np.log(0.75)) < 1e-15
    assert orc.choose_row(np.full(3, -np.inf), np.full(3, -np.inf)) == (-1, -np.inf)
    # a student equal to the teacher's own distribution has divergence 0 and no gradient
    lp = np.log(np.array([0.5, 0.3, 0.15, 0.05]))
    for ids, kind in (([0, 1, 2, 3], "logits"), ([1, 3], "logprobs")):
        L, g, _, _ = orc.distill_row(lp, np.array(ids), lp[ids], kind, 1.0)
        assert abs(L) < 1e-15 and np.abs(g).max() < 1e-15
    L, g, _, _ = orc.distill_row(np.zeros(4), np.array([2]), np.array([0.0]), "logits", 1.0)
    assert abs(L - np.log(4.0)) < 1e-15 and np.allclose(g, [0.25, 0.25, -0.75, 0.25], atol=1e-15)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("ragged,repeats", [(False, False), (True, False), (True, True)])
def test_oracle_gradient_by_differences(kind, ragged, repeats):
    rng = np.random.default_rng(4)
    z, ids, t = make_distill(rng, 3, 12, 5, kind, torch.float32, ragged=ragged, repeats=repeats)
    zn, h, T = z.double().numpy(), 1e-5, 1.7
    for r in range(3):
        _, g, _, _ = orc.distill_row(zn[r], ids[r], t[r], kind, T)
        for v in range(12):
            d = np.zeros(12)
            d[v] = h
            up, down = (orc.distill_row(zn[r] + s * d, ids[r], t[r], kind, T)[0] for s in (1, -1))
            # truncation h^2 / 6 * 1.54 / T^3 < 2e-11, rounding 1e-15 / h
            assert abs((up - down) / (2 * h) - g[v]) < 1e-9


def test_rules_cover_what_they_are_for():
    rng = np.random.default_rng(0)
    c = make_rules(rng, 6, 50, hist=30, prompt=True, sparse=40, mask="bool")
    assert (c["history"] < 0).any() and (c["history"] >= 50).any() and c["lengths"][1] == 0 and not c["allowed"][3].any()
    assert any(len(set(row)) < len(row) for row in c["bias_tokens"].tolist())
