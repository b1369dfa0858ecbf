"""GPU tests of the answer operators at their edges: C callers' arguments,
sums that cancel, infinities and large whole numbers, large batches.

Tolerances count roundings: u = 2^-24 is half a step of fp32."""
import ctypes as ct

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.answers_ref import nibbles
from tests.test_gpu_answers import check_loss, check_votes, votes_inputs
from ytm_b200 import _lib, answers
from ytm_b200.cutm import MultiClassTM

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
CODE = {"i32": _lib.YTM_I32, "f32": _lib.YTM_F32, "f16": _lib.YTM_F16, "bf16": _lib.YTM_BF16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def stream():
    return ct.c_void_p(torch.cuda.current_stream().cuda_stream)


# ------------------------------------------------------- the C ABI's arguments

@pytest.mark.parametrize("dt", ["i32", "bf16"])
@pytest.mark.parametrize("k", [10, 100, 400, 1000, 5003])
def test_strides_beside_null_pointers_count_for_nothing(k, dt):
    n, lib = 5, _lib.load()
    rng = np.random.default_rng(k)
    cs = dev(rng.integers(-20, 21, (n, k)).astype(np.int32)).to(DT[dt])
    y = dev(rng.integers(0, k, n))
    choice, logprob, z = answers.answer(cs)
    c2, l2, z2 = torch.empty_like(choice), torch.empty_like(logprob), torch.empty_like(z)
    a = _lib.AnswerArgs(cs=cs.data_ptr(), cs_stride=k, n=n, k=k, cs_type=CODE[dt], bias_stride=k, allowed_stride=(k + 31) // 32,
                        history_stride=9, temperature_all=1.0, repetition_all=1.0, choice=c2.data_ptr(), logprob=l2.data_ptr(),
                        adjusted=z2.data_ptr())
    _lib.check(lib.ytm_answer(ct.byref(a), stream()))
    assert torch.equal(c2, choice) and torch.equal(l2, logprob) and torch.equal(z2, z)
    loss, dcs, _, dtem = answers.class_loss(cs, y)
    loss2, dtem2 = torch.empty_like(loss), torch.empty_like(dtem)
    dcs2 = None if dcs is None else torch.empty_like(dcs)
    ws = torch.empty(max(16, lib.ytm_class_loss_workspace_bytes(n, k, CODE[dt], k)), dtype=torch.uint8, device="cuda")
    a = _lib.LossArgs(cs=cs.data_ptr(), cs_stride=k, n=n, k=k, cs_type=CODE[dt], allowed_stride=(k + 31) // 32, target=y.data_ptr(),
                      target_64=1, temperature_all=1.0, loss=loss2.data_ptr(), dcs=None if dcs is None else dcs2.data_ptr(),
                      dtemperature=dtem2.data_ptr())
    _lib.check(lib.ytm_class_loss(ct.byref(a), ws.data_ptr(), stream()))
    assert torch.equal(loss2, loss) and torch.equal(dtem2, dtem) and (dcs is None or torch.equal(dcs2, dcs))


# ------------------------------------------------------------ sums that cancel

@pytest.mark.parametrize("dt", ["i32", "f32", "bf16"])
@pytest.mark.parametrize("n,k", [(4_000_000, 10), (1_000_000, 100), (300_000, 300), (100_000, 1000)])
def test_bias_gradient_of_many_certain_rows(n, k, dt):
    """Rows that are all right with probability 1 - (k - 1) e^-9: a label's
    gradient is the small rest of its weight.  All terms of a class have one
    sign, so every rounding counts relative to the sum.  A term: the exponent 13
    off by 2 u of itself (18 u of the exponential), ex2 by 2 steps, the row's sum
    by its chain, the quotients by 6 u, a long row's difference from its weight
    by u of 1; the sum: at most 256 rows one after another, 64 teams of a block."""
    cs = torch.zeros((1, k), dtype=DT[dt], device="cuda")
    cs[0, 3] = 9
    y = torch.full((n,), 3, device="cuda")
    loss, _, dbias, _ = answers.class_loss(cs.expand(n, k), y, bias=torch.zeros(k, device="cuda"))
    e = np.exp(-9.0)
    p = np.full(k, e / (1 + (k - 1) * e))
    p[3] = -(k - 1) * p[0]
    chain = k / 32 + 64
    tol = (22 + chain + 6 + 256 + 64 + 4) * U * np.abs(n * p)
    if k > 512:
        tol[3] += n * 2 * U
    err = np.abs(f64(dbias) - n * p)
    assert (err <= tol).all(), (err / tol).max()
    want = np.log1p((k - 1) * e)
    assert (loss - want).abs().max().item() <= (2 * chain + 64) * U


# --------------------------------------------------- infinities and large sums

@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("k", [40, 500, 1025, 5003, 40001])
def test_class_loss_of_unusual_values_wherever_they_lie(k, shift, dt):
    """A NaN or +inf among the allowed makes a row's loss and gradients NaN, -inf
    is a probability of 0, and a masked value counts for nothing, at a row's
    first, middle and last class and at any alignment of its memory."""
    rng = np.random.default_rng(k + shift)
    cases = [(v, at, masked) for v in (np.nan, np.inf, -np.inf) for at in (0, 5, k // 2, k - 1) for masked in (False, True)]
    n = len(cases)
    wide = torch.zeros((n, k + 5), dtype=DT[dt], device="cuda")
    cs = wide[:, shift:shift + k]
    cs.copy_(dev(rng.normal(size=(n, k)).astype(np.float32)))
    open_ = np.ones((n, k), bool)
    y = dev(np.full(n, 1))
    clean = open_.copy()
    for i, (v, at, masked) in enumerate(cases):
        open_[i, at] = not masked
        clean[i, at] = False
    want = answers.class_loss(cs, y, allowed=answers.pack_allowed(clean).cuda())
    check_loss(want, cs, y.cpu().numpy(), {"allowed": clean, "temperature": np.float32(1.0)})
    for i, (v, at, masked) in enumerate(cases):
        cs[i, at] = v
    loss, dcs, _, _ = answers.class_loss(cs, y, allowed=answers.pack_allowed(open_).cuda())
    for i, (v, at, masked) in enumerate(cases):
        if masked or v == -np.inf:
            assert torch.equal(loss[i], want[0][i]) and torch.equal(dcs[i], want[1][i]), cases[i]
        else:
            assert torch.isnan(loss[i]) and torch.isnan(dcs[i]).all(), cases[i]


def check_whole_loss(cs, y, mask, bias, t, far=None):
    """The loss of int32 sums (64 bits in `cs`) against 64 bits.  A row's
    gradients and, its gradients' sum being 0, the temperature's do not change
    when a number is taken from all of the row; less their largest, the sums
    are as near as they lie, which is what the bounds of check_loss count."""
    kw = {"temperature": np.float32(t)}
    kt = {"temperature": float(t)}
    if mask is not None:
        kw["allowed"], kt["allowed"] = mask, answers.pack_allowed(mask).cuda()
    if bias is not None:
        kw["bias"], kt["bias"] = bias, dev(bias)
    got = answers.class_loss(dev(cs.astype(np.int32)), dev(y), **kt)
    open_ = np.ones(cs.shape, bool) if mask is None else np.broadcast_to(mask, cs.shape)
    if far is not None:  # classes whose probability is 0 in fp32
        open_ = open_ & ~far
        kw["allowed"] = open_
    top = np.where(open_, cs, np.iinfo(np.int64).min).max(1, keepdims=True)
    # A sum v below 2^24 is not moved: with a bias, fp32 rounds v + b by up to u of
    # |v + b|, which check_loss counts where v itself is given to it.
    if bias is not None:
        top[((np.abs(cs) < 2 ** 24) & open_).any(1)] = 0
    check_loss(got, torch.from_numpy(np.where(open_, cs - top, 0)), y, kw)


BASES = [0, 12345, 2 ** 24, -2 ** 24 - 30, 2 ** 24 - 7, -2 ** 24 - 1, 2 ** 30 + 7, 2 ** 31 - 61, -2 ** 31]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mask", [None, "all", "row"])
@pytest.mark.parametrize("k", [3, 10, 100, 300, 1000, 5003])
def test_class_loss_of_large_whole_sums(k, mask, bias):
    """Whole numbers above 2^24 keep their differences."""
    rng = np.random.default_rng(k)
    n = 4 * len(BASES)
    base = np.array(BASES)[np.arange(n) % len(BASES)][:, None]
    y = rng.integers(0, k, n)
    a = None
    if mask:
        a = rng.random((n if mask == "row" else 1, k)) < 0.7
        a[np.arange(n) if mask == "row" else 0, y] = True
    b = rng.normal(size=k).astype(np.float32) if bias else None
    cs = base + rng.integers(0, 61, (n, k))
    check_whole_loss(cs, y, a, b, 1.0)
    check_whole_loss(cs, y, a, b, 15.5)
    check_whole_loss(rng.integers(-2 ** 26, 2 ** 26, (n, k)), y, a, b, 2.0 ** 20)
    check_whole_loss(rng.integers(-2 ** 31, 2 ** 31, (n, k)), y, a, b, 2.0 ** 29)
    # some classes far below, beyond an int32 difference for the highest rows
    far = rng.random((n, k)) < 0.4
    far[np.arange(n), y] = False
    rows = (base[:, 0] > 0)
    cs = np.where(far, rng.integers(-2 ** 31, -2 ** 30, (n, k)), cs)
    check_whole_loss(cs[rows], y[rows], a[rows] if mask == "row" else a, b, 3.0, far[rows])


@pytest.mark.parametrize("n,k", [(250, 10), (120, 100), (20000, 40), (3000, 257), (603, 9001), (1300, 600)])
def test_class_loss_of_large_whole_sums_in_many_rows(n, k):
    """Large sums and others in turn, in one thread's rows and in one row's rounds."""
    rng = np.random.default_rng(n)
    base = rng.choice(np.array(BASES), (n, 1))
    y = rng.integers(0, k, n)
    b = rng.normal(size=k).astype(np.float32)
    check_whole_loss(base + rng.integers(0, 61, (n, k)), y, None, None, 7.5)
    check_whole_loss(base + rng.integers(0, 61, (n, k)), y, None, b, 7.5)
    # a row's classes in runs of different magnitude, the largest anywhere
    runs = np.repeat(rng.integers(0, 32, (n, -(-k // 37))), 37, 1)[:, :k]
    cs = np.where(rng.random((n, 1)) < 0.5, 1, -1) * (2 ** runs.astype(np.int64) - 1) + rng.integers(0, 2, (n, k))
    cs = np.clip(cs, -2 ** 31, 2 ** 31 - 1)
    check_whole_loss(cs, y, None, b, 2.0 ** 26)


def test_class_loss_tells_neighbouring_whole_sums_apart():
    for k in (5, 700):
        cs = np.zeros((2, k), np.int32)
        cs[:, 0], cs[:, 1], cs[:, 2:] = 16777217, 16777216, -2 ** 31
        loss, _, db, _ = answers.class_loss(dev(cs), dev(np.array([0, 1])), bias=torch.zeros(k, device="cuda"))
        q = 1 / (1 + np.exp(-1.0))
        np.testing.assert_allclose(f64(loss), [-np.log(q), -np.log(1 - q)], rtol=16 * U)
        np.testing.assert_allclose(f64(db)[:2], [2 * q - 1, 1 - 2 * q], rtol=32 * U)


# ---------------------------------------------------------------- large batches

@pytest.mark.parametrize("x,n,c,k", [("bits", 20001, 65536, 100), ("bits", 9001, 65536, 600), ("bf16", 9000, 65536, 520),
                                     ("f32", 4100, 65536, 40)])
def test_votes_of_more_activations_than_are_laid_out_at_once(x, n, c, k):
    """Several launches of one call, against 64 bits for some of the samples and
    against calls of 64 samples for all: two sums of the same terms, each within
    the bound of check_votes."""
    torch.manual_seed(n)
    _, _, packed, q, scales, bias = votes_inputs(1, c, k, x, 64, "f32")
    if x == "bits":
        xt = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, c // 32), dtype=torch.int32, device="cuda")
        some = lambda r: ((xt[r].cpu().numpy().view(np.uint32)[:, np.arange(c) // 32] >> (np.arange(c) % 32)) & 1).astype(np.float64)  # noqa: E731
        most = torch.ones((1, c), device="cuda")
    else:
        xt = torch.randn((n, c), device="cuda").to(DT[x])
        some = lambda r: f64(xt[r])  # noqa: E731
        most = xt.abs().amax(0, keepdim=True).float()
    y = answers.q4_votes(xt, packed, scales, 64, bias=dev(bias), clauses=c)
    rows, cols = np.r_[0:3, n // 2 - 40:n // 2 + 40, n - 3:n], np.r_[0:4, k - 4:k]
    check_votes(y[rows][:, cols], some(rows), q[cols], scales[cols], 64, bias[cols], "f32", c)
    parts = torch.cat([answers.q4_votes(xt[i:i + 64], packed, scales, 64, bias=dev(bias), clauses=c) for i in range(0, n, 64)])
    w = dev(np.abs(q).astype(np.float32)) * scales.repeat_interleave(64, 1)[:, :c]
    mag = ((most.double() @ w.double().t()) + dev(bias).abs()) * 1.001
    depth = 64 + c // 64 + 64 + 1  # and the result's own rounding
    assert ((y.double() - parts.double()).abs() <= 2 * depth * 2 * U * mag).all()


@pytest.mark.parametrize("n", [1, 3, 64])
def test_nan_votes_of_nan_activations_are_no_wait_given_up(n):
    xt, _, packed, _, scales, _ = votes_inputs(n, 1000, 3001, "bf16", 64, "f32")
    xt[:, 7] = float("nan")
    assert torch.isnan(answers.q4_votes(xt, packed, scales, 64)).all()
    assert answers.q4_votes_gave_up() == 0 and answers.q4_votes_gave_up(xt.device) == 0


# ------------------------------------------------------------- unusual tensors

def test_forward_mode_tangents_are_refused():
    z, i = torch.randn((3, 40), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    p, s = answers.q4_pack(torch.ones((40, 8), device="cuda"), 32)
    b = torch.zeros(40, device="cuda")
    want = answers.answer(z)
    with fwad.dual_level():
        d, db = fwad.make_dual(z, torch.ones_like(z)), fwad.make_dual(b, torch.ones_like(b))
        for f in (lambda: answers.answer(d), lambda: answers.answer(z, bias=db), lambda: answers.class_loss(d, i),
                  lambda: answers.class_loss(z, i, bias=db), lambda: answers.q4_pack(d), lambda: answers.q4_votes(d, p, s, 32)):
            with pytest.raises(ValueError, match="tangent"):
                f()
        with torch.no_grad(), fwad._set_fwd_grad_enabled(False):
            got = answers.answer(d)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        assert torch.equal(answers.answer(fwad.unpack_dual(d).primal.detach())[1], want[1])


def test_negated_views_are_read_with_their_sign():
    z, i = torch.randn((3, 40), device="cuda"), torch.tensor([1, 2, 3], device="cuda")
    b = torch.randn(40, device="cuda")
    n, nb = torch._neg_view(z), torch._neg_view(b)
    assert n.is_neg() and nb.is_neg()
    p, s = answers.q4_pack(-z.t(), 32)
    p2, s2 = answers.q4_pack(n.t(), 32)
    assert torch.equal(p, p2) and torch.equal(s, s2)
    p, s = answers.q4_pack(torch.randn((40, 5), device="cuda"), 32)
    for got, want in ((answers.answer(n, bias=nb), answers.answer(-z, bias=-b)),
                      (answers.class_loss(n, i, bias=nb), answers.class_loss(-z, i, bias=-b)),
                      ((answers.q4_votes(n, p, s, 32),), (answers.q4_votes(-z, p, s, 32),))):
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_arguments_without_memory_of_their_own_are_refused():
    """Such a bias or mask would have been no bias and no mask."""
    z, i = torch.randn((3, 40), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with FakeTensorMode():
        b, a = torch.empty(40, device="cuda"), torch.empty((3, 2), dtype=torch.int32, device="cuda")
    for f in (lambda: answers.answer(z, bias=b), lambda: answers.answer(z, allowed=a), lambda: answers.class_loss(z, i, bias=b),
              lambda: answers.class_loss(z, i, allowed=a), lambda: answers.answer(z, temperature=b[:3])):
        with pytest.raises(ValueError, match="memory"):
            f()
    with pytest.raises(TypeError, match="strided"):
        answers.answer(z.to_sparse())


def test_knobs_without_dimensions():
    """A tensor [] counts for all rows, on the device or, as a number, on the CPU."""
    torch.manual_seed(0)
    z, h = torch.randn((5, 40), device="cuda") * 4, torch.randint(0, 40, (5, 9), device="cuda")
    kw = {"repetition": 1.25, "frequency": 0.5, "presence": 0.75, "temperature": 1.5}
    want = answers.answer(z, history=h, **kw)
    y = torch.tensor([0, 1, 2, 3, 39], device="cuda")
    want_loss = answers.class_loss(z, y, temperature=1.5)
    for make in (lambda v: torch.tensor(v, device="cuda"), torch.tensor, lambda v: torch.tensor(v, dtype=torch.float64), np.float32, np.array):
        got = answers.answer(z, history=h, **{k: make(v) for k, v in kw.items()})
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = answers.class_loss(z, y, temperature=make(1.5))
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, want_loss))
    with pytest.raises(TypeError, match="temperature"):
        answers.answer(z, temperature=torch.tensor(1.5, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="positive"):
        answers.answer(z, temperature=torch.tensor(-1.0))
    tm = MultiClassTM(number_of_clauses_per_class=20, T=15, s=4.0, dim=(8, 8, 1), n_classes=3, seed=2)
    X = (np.random.default_rng(0).random((6, 64)) < 0.4).astype(np.uint32)
    tm.fit(X, np.arange(6) % 3)
    want = tm.answer(X, temperature=2.5)
    for t in (torch.tensor(2.5), torch.tensor(2.5, device="cuda"), torch.tensor(2.5, device="cuda", dtype=torch.float64), np.float64(2.5),
              np.full(6, 2.5), torch.full((6,), 2.5)):
        assert all(np.array_equal(a, b) for a, b in zip(tm.answer(X, temperature=t), want))


# ------------------------------------------------------- offsets past 32 bits

def test_loss_and_answer_of_more_than_2_to_the_32_bytes_and_2_to_the_31_classes():
    """The last rows of 2.2e9 class sums against the same rows alone: two sums of
    the same k exponentials, each within (108 + 4 (k / 32 + 64)) u."""
    n, k = 68000, 32001
    cs = torch.empty((n, k), dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 4000):
        cs[i:i + 4000] = torch.randn((min(4000, n - i), k), device="cuda") * 4
    y = torch.arange(n, device="cuda") % k
    rel = 2 * (108 + 4 * (k / 32 + 64)) * U
    loss, dcs, _, _ = answers.class_loss(cs, y)
    some = [0, n // 2, n - 2, n - 1]
    want = answers.class_loss(cs[some], y[some])
    assert ((loss[some] - want[0]).abs() <= rel * (1 + want[0].abs())).all()
    err = (dcs[some].double() - want[1].double()).abs()
    assert (err <= 2.0 ** -7 * want[1].double().abs() + rel).all()  # a rounding each to bf16
    del dcs
    choice, logprob, z = answers.answer(cs, temperature=0.5)
    c, lp, zz = answers.answer(cs[some], temperature=0.5)
    assert torch.equal(choice[some], c) and torch.equal(z[some], zz)
    assert ((logprob[some] - lp).abs() <= rel * (1 + lp.abs())).all()


def test_votes_of_activations_and_weights_past_32_bits():
    n, c, k = 66000, 33000, 5
    _, _, packed, _, scales, bias = votes_inputs(1, c, k, "f32", 64, "f32")
    x = torch.empty((n, c), dtype=torch.float16, device="cuda")
    for i in range(0, n, 4000):
        x[i:i + 4000] = torch.randn((min(4000, n - i), c), device="cuda")
    y = answers.q4_votes(x, packed, scales, 64)
    some = [0, n // 2, n - 2, n - 1]
    q = nibbles(packed.cpu().numpy(), c).astype(np.int64) - 8
    check_votes(y[some], f64(x[some]), q, scales, 64, np.zeros(k), "f32", c)
    del x, y
    torch.cuda.empty_cache()
    c, k = 32768, 140001
    packed = torch.randint(0, 256, (k, c // 2), dtype=torch.uint8, device="cuda")
    scales = torch.rand((k, c // 64), device="cuda") + 0.1
    for xs in (torch.randn((1, c), device="cuda"), torch.randn((64, c), device="cuda").half()):
        y = answers.q4_votes(xs, packed, scales, 64)
        some = [0, 70000, k - 2, k - 1]
        q = nibbles(packed[some].cpu().numpy(), c).astype(np.int64) - 8
        check_votes(y[:, some], f64(xs), q, scales[some], 64, np.zeros(4), "f32", c)
