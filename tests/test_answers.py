"""CPU tests of the answer operators: the ABI's argument checks, the Python
refusals, the argument structs, and the reference gradients against
differences."""
import ctypes as ct
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from tests.answers_ref import ref_loss
from ytm_b200 import _lib, answers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,mirror", [("ytm_answer_args", _lib.AnswerArgs), ("ytm_loss_args", _lib.LossArgs)])
def test_argument_structs_match_the_header(tmp_path, name, mirror):
    src = open(os.path.join(ROOT, "include", "ytm.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [re.sub(r"\s*\*?\s*", "", f.split()[-1] if i == 0 else f) for line in body.split(";") if line.strip()
              for i, f in enumerate(line.split(","))]
    assert fields == [f for f, _ in mirror._fields_]
    c = tmp_path / "s.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ytm.h"\nint main(void) {\n' +
                 "".join('printf("%%zu ", offsetof(%s, %s));\n' % (name, f) for f in fields) +
                 'printf("%%zu", sizeof(%s)); return 0; }\n' % name)
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(mirror, f).offset for f in fields] + [ct.sizeof(mirror)]


def test_entry_points_reject_bad_arguments_without_a_gpu():
    lib = _lib.load()
    one = ct.c_void_p(16)  # never read: every check comes before any launch
    pack = lambda **kw: lib.ytm_q4_pack(*[{**dict(w=one, wt=0, ws=4, C=8, K=4, g=64, p=one, s=one, st=1), **kw}[i]  # noqa: E731
                                          for i in ("w", "wt", "ws", "C", "K", "g", "p", "s", "st")], None)
    for kw in (dict(C=0), dict(K=0), dict(g=48), dict(st=0), dict(wt=2), dict(ws=3), dict(w=None), dict(p=None),
               dict(s=None)):
        assert pack(**kw) == 1, kw
    votes = lambda **kw: lib.ytm_q4_votes(*[{**dict(x=one, xt=1, xs=8, N=1, C=8, p=one, s=one, st=1, g=64, K=4,  # noqa: E731
                                                    b=None, y=one, yt=1, ws=one), **kw}[i]
                                            for i in ("x", "xt", "xs", "N", "C", "p", "s", "st", "g", "K", "b", "y", "yt", "ws")],
                                          None)
    for kw in (dict(xt=0), dict(xt=5), dict(xs=-1), dict(N=-1), dict(C=0), dict(p=None), dict(p=ct.c_void_p(8)), dict(st=4),
               dict(g=16), dict(K=0), dict(y=None), dict(yt=0), dict(x=None), dict(s=None), dict(ws=None), dict(ws=ct.c_void_p(8))):
        assert votes(**kw) == 1, kw
    assert votes(N=0) == 0
    assert votes(K=(1 << 30) + 1) == 3 and votes(C=(1 << 30) + 1) == 3
    good = dict(cs=16, cs_stride=4, n=1, k=4, cs_type=0)
    for kw in (dict(k=0), dict(n=-1), dict(cs_type=4), dict(cs=None), dict(cs_stride=-1), dict(bias_stride=-1),
               dict(allowed_stride=-1), dict(history_len=-1), dict(lengths=16)):
        assert lib.ytm_answer(ct.byref(_lib.AnswerArgs(**{**good, **kw})), None) == 1, kw
    assert lib.ytm_answer(None, None) == 1
    assert lib.ytm_answer(ct.byref(_lib.AnswerArgs(**{**good, "n": 0})), None) == 0
    good = dict(cs=16, cs_stride=4, n=1, k=4, cs_type=0, target=16, loss=16)
    for kw in (dict(k=0), dict(n=-1), dict(cs_type=4), dict(cs=None), dict(dcs=16), dict(target=None), dict(loss=None),
               dict(cs_stride=-1), dict(allowed_stride=-1)):
        assert lib.ytm_class_loss(ct.byref(_lib.LossArgs(**{**good, **kw})), one, None) == 1, kw
    assert lib.ytm_class_loss(ct.byref(_lib.LossArgs(**{**good, "n": 100000})), None, None) == 1
    assert lib.ytm_class_loss_workspace_bytes(100000, 4, 1, 4) > 0
    assert lib.ytm_class_loss(ct.byref(_lib.LossArgs(**{**good, "n": 1 << 31})), one, None) == 3
    assert lib.ytm_class_loss(ct.byref(_lib.LossArgs(**{**good, "k": (1 << 30) + 1})), one, None) == 3
    assert lib.ytm_class_loss(None, one, None) == 1
    assert lib.ytm_class_loss(ct.byref(_lib.LossArgs(**{**good, "n": 0})), None, None) == 0
    assert lib.ytm_class_loss_workspace_bytes(-1, 4, 1, 4) == 0
    cfg = _lib.make_config(clauses_per_class=8, T=5, s=3.0, dim=(16, 1, 1), n_classes=2)
    assert lib.ytm_infer_fired(ct.byref(cfg), None, None, 4, None, None, None) == 1
    assert lib.ytm_infer_fired(ct.byref(cfg), None, None, 0, None, None, None) == 0


def test_cpu_tensors_and_wrong_types_are_refused():
    f, i = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        answers.answer(f)
    with pytest.raises(ValueError, match="CUDA"):
        answers.class_loss(f, i)
    with pytest.raises(ValueError, match="CUDA"):
        answers.q4_pack(f)
    with pytest.raises(TypeError, match="cs must be"):
        answers.answer(f.double())
    with pytest.raises(TypeError, match="torch tensor"):
        answers.answer(np.zeros((2, 4)))
    with pytest.raises(ValueError, match="dimension"):
        answers.answer(f[0])


def test_pack_allowed():
    rng = np.random.default_rng(0)
    a = rng.random((3, 45)) < 0.5
    w = answers.pack_allowed(a)
    assert w.shape == (3, 2) and w.dtype == torch.int32
    for k in range(64):
        bit = (w.numpy().view(np.uint32)[:, k // 32] >> (k % 32)) & 1
        np.testing.assert_array_equal(bit, a[:, k] if k < 45 else 0)
    assert torch.equal(answers.pack_allowed(torch.from_numpy(a)), w)
    assert answers.pack_allowed(a[0]).shape == (1, 2)
    with pytest.raises(ValueError):
        answers.pack_allowed(a, 44)


def test_reference_gradients_against_differences():
    """ref_loss's formulas, which the kernels are held to, against central
    differences of its loss in 64 bits: h = 1e-5, error O(h^2) + 1e-16 / h."""
    rng = np.random.default_rng(1)
    n, k = 4, 7
    cs, b, w = rng.normal(size=(n, k)) * 3, rng.normal(size=k), rng.random(n)
    allowed = rng.random((n, k)) < 0.7
    y = np.array([1, 3, -1, 6])
    allowed[[0, 1, 3], [1, 3, 6]] = True
    t, h = 1.7, 1e-5
    _, dcs, db, dt = ref_loss(cs, y, b, allowed, t, w)
    f = lambda cs=cs, b=b, t=t: ref_loss(cs, y, b, allowed, t, w)[0].sum()  # noqa: E731
    for i in range(n):
        for j in range(k):
            e = np.zeros((n, k))
            e[i, j] = h
            assert abs((f(cs=cs + e) - f(cs=cs - e)) / (2 * h) - dcs[i, j]) < 1e-8
    for j in range(k):
        e = np.zeros(k)
        e[j] = h
        assert abs((f(b=b + e) - f(b=b - e)) / (2 * h) - db[j]) < 1e-8
    assert abs((f(t=t + h) - f(t=t - h)) / (2 * h) - dt) < 1e-8
