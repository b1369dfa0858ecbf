"""GPU tests of the answer operators (ytm_b200.answers, CudaEngine.infer_fired
and the model methods over them) against plain 64-bit implementations.

Tolerances count roundings: u = 2^-24 is half a step of fp32, eps / 2 of the
output type the rounding of a result."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from tests.answers_ref import nibbles, ref_answer, ref_loss, ref_pack, ref_votes
from ytm_b200 import _lib, answers
from ytm_b200.cutm import MultiClassTM, MultiOutputTM
from ytm_b200.engine import CudaEngine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def half_step(dt, value):
    """Half a step of the type at |value|, and half its smallest step at 0."""
    info = torch.finfo(dt)
    return info.eps / 2 * np.abs(value) + info.smallest_normal * info.eps / 2


def bit_words(bits):
    pad = np.zeros((bits.shape[0], -(-bits.shape[1] // 32) * 32), bool)
    pad[:, :bits.shape[1]] = bits
    return np.packbits(pad, axis=1, bitorder="little").view(np.int32)


# ------------------------------------------------------------------ packing

@pytest.mark.parametrize("c,k,group,kind,scale", [(1, 1, 32, "i32", "f32"), (33, 5, 32, "i32", "bf16"),
                                                  (200, 17, 64, "f32", "f16"), (1000, 7, 128, "i32", "f32"),
                                                  (129, 40, 128, "f32", "bf16")])
def test_q4_pack(c, k, group, kind, scale):
    rng = np.random.default_rng(c)
    w = rng.integers(-30, 31, (c, k)).astype(np.int32) if kind == "i32" else rng.normal(size=(c, k)).astype(np.float32)
    w[:, 0] = 0  # a class whose groups are all zero
    wide = torch.zeros((c, k + 3), dtype=DT[kind], device="cuda")
    wide[:, :k] = dev(w)
    packed, scales = answers.q4_pack(wide[:, :k], group, DT[scale])
    q, s = ref_pack(w, group)
    assert packed.shape == (k, -(-c // 32) * 16)
    got = nibbles(packed.cpu().numpy(), packed.shape[1] * 2).astype(int) - 8
    np.testing.assert_array_equal(got[:, :c], q)
    assert (got[:, c:] == 0).all()
    # a / 7 to fp32, then to the scale's type
    assert (np.abs(f64(scales) - s) <= half_step(DT[scale], s) * (1 + 2.0 ** -8) + U * s).all()
    assert torch.equal(answers.q4_pack(wide[:, :k].t().contiguous().t(), group, DT[scale])[0], packed)


# -------------------------------------------------------------------- votes

def votes_inputs(n, c, k, x, group, scale, seed=0):
    rng = np.random.default_rng(seed)
    words = -(-c // 32)
    packed = rng.integers(0, 256, (k, words * 16)).astype(np.uint8)  # the halves behind c are anything
    scales = dev(rng.random((k, -(-c // group))).astype(np.float32) + 0.1).to(DT[scale])
    if x == "bits":
        xw = rng.integers(-2 ** 31, 2 ** 31, (n, words)).astype(np.int32)  # bits behind c too
        xv = ((xw.view(np.uint32)[:, np.arange(c) // 32] >> (np.arange(c) % 32)) & 1).astype(np.float64)
        xt = dev(xw)
    else:
        xt = dev(rng.normal(size=(n, c)).astype(np.float32)).to(DT[x])
        xv = f64(xt)
    bias = rng.normal(size=k).astype(np.float32)
    return xt, xv, dev(packed), nibbles(packed, c).astype(np.int64) - 8, scales, bias


def check_votes(y, xv, q, scales, group, bias, out, c):
    """Any order of the sum has at most `depth` additions one after another if
    groups are summed apart (group terms, then the groups, then 64 for the
    joins), each off by at most a step (2 u: matrix units cut off) of the sum
    of magnitudes; then the rounding to the output's type."""
    want, mag = ref_votes(xv, q, f64(scales), group, bias)
    depth = min(group, c) + -(-c // group) + 64
    tol = depth * 2 * U * mag + half_step(DT[out], want) * (1 + 2.0 ** -7)
    err = np.abs(f64(y) - want)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c,k,group,scale,out", [
    (1, 1, 1, 32, "f32", "f32"), (1, 33, 3, 32, "f16", "f32"), (2, 127, 17, 64, "bf16", "f16"),
    (3, 128, 16, 128, "f32", "bf16"), (5, 1000, 100, 32, "f32", "f32"), (1, 4097, 33, 64, "bf16", "f32"),
    (8, 2048, 65, 128, "f16", "f32"), (9, 1023, 130, 64, "f32", "f32"), (17, 640, 16, 32, "bf16", "bf16"),
    (40, 3000, 257, 64, "f16", "f32"), (70, 129, 31, 128, "f32", "f16"), (130, 512, 48, 64, "f32", "f32"),
    (1, 65536, 100, 64, "f32", "f32"), (300, 96, 2, 32, "f32", "f32")])
def test_votes(n, c, k, group, scale, out, x):
    xt, xv, packed, q, scales, bias = votes_inputs(n, c, k, x, group, scale, seed=n + c)
    y = answers.q4_votes(xt, packed, scales, group, bias=dev(bias), clauses=c, out_dtype=DT[out])
    check_votes(y, xv, q, scales, group, bias, out, c)
    again = answers.q4_votes(xt, packed, scales, group, bias=dev(bias), clauses=c, out_dtype=DT[out])
    assert torch.equal(y, again)  # a fixed order of summation
    check_votes(answers.q4_votes(xt, packed, scales, group, clauses=c), xv, q, scales, group, np.zeros(k), "f32", c)


@pytest.mark.parametrize("x", ["bits", "f16", "bf16"])
@pytest.mark.parametrize("n,c,k,group,scale,out", [
    (3, 64, 512, 64, "f32", "f32"), (3, 1, 513, 32, "f32", "f32"), (16, 256, 700, 32, "f16", "f32"), (17, 257, 1025, 128, "f32", "f16"),
    (33, 4000, 600, 64, "bf16", "f32"), (48, 2500, 2000, 32, "f16", "bf16"), (49, 1023, 999, 128, "f32", "f32"),
    (64, 2048, 512, 64, "f32", "f32"), (65, 700, 777, 32, "f32", "f32"), (150, 3001, 1500, 128, "bf16", "f32"),
    (5, 20000, 4100, 64, "f16", "f32"), (64, 5000, 9000, 32, "f32", "f32"), (33, 1, 70001, 64, "f32", "f32"),
    (40, 300, 40000, 128, "f16", "bf16"), (64, 1300, 3001, 128, "bf16", "f32"), (20, 1500, 20011, 64, "f32", "f16"),
    (130, 9000, 1500, 128, "f16", "f32"), (100, 20000, 700, 64, "f32", "f32"), (70, 1000, 30000, 32, "bf16", "f32"),
    (64, 4097, 5000, 32, "f16", "f32"), (1000, 3000, 600, 64, "f32", "bf16")])
def test_votes_of_many_classes_and_several_samples(n, c, k, group, scale, out, x):
    test_votes(n, c, k, group, scale, out, x)


@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
def test_votes_strides_and_alignment(x):
    """Rows of a wider array that start off any 16-byte boundary, one row
    repeated, transposed memory, a slice of the classes."""
    n, c, k, group = 6, 301, 37, 32
    xt, xv, packed, q, scales, bias = votes_inputs(n, c, k, x, group, "f32")
    wide = torch.full((n, xt.shape[1] + 5), 7, dtype=xt.dtype, device="cuda")
    wide[:, 3:-2] = xt
    for view, v in ((wide[:, 3:-2], xv), (xt[2:3].expand(n, -1), np.repeat(xv[2:3], n, 0)),
                    (xt.t().contiguous().t(), xv), (xt[::2], xv[::2])):
        y = answers.q4_votes(view, packed, scales, group, clauses=c)
        check_votes(y, v, q, scales, group, np.zeros(k), "f32", c)
    y = answers.q4_votes(xt, packed[5:20], scales[5:20], group, bias=dev(bias)[5:20], clauses=c)
    check_votes(y, xv, q[5:20], scales[5:20], group, bias[5:20], "f32", c)


@pytest.mark.parametrize("x", ["bits", "f16", "bf16"])
def test_votes_of_many_classes_strides_and_infinities(x):
    """As above for 64 samples of many classes: rows off any boundary, memory
    full of NaN behind a block's last sample, infinities that stay in their row."""
    n, c, k, group = 64, 1301, 3001, 128
    xt, xv, packed, q, scales, bias = votes_inputs(n, c, k, x, group, "f32")
    wide = torch.full((n, xt.shape[1] + 5), 7, dtype=xt.dtype, device="cuda")
    wide[:, 3:-2] = xt
    for view, v in ((wide[:, 3:-2], xv), (xt[2:3].expand(n, -1), np.repeat(xv[2:3], n, 0)), (xt[:50], xv[:50])):
        trash = torch.full((1 << 22,), float("nan"), device="cuda")
        del trash
        check_votes(answers.q4_votes(view, packed, scales, group, clauses=c), v, q, scales, group, np.zeros(k), "f32", c)
    part = answers.q4_votes(xt, packed[8:2905], scales[8:2905], group, bias=dev(bias)[8:2905], clauses=c)
    check_votes(part, xv, q[8:2905], scales[8:2905], group, bias[8:2905], "f32", c)
    if x == "bits":
        return
    y = answers.q4_votes(xt, packed, scales, group)
    xt[5, 77], xt[9, 1300] = float("inf"), float("nan")
    z = answers.q4_votes(xt, packed, scales, group)
    w = dev(q[:, 77])
    assert (z[5][w > 0] == float("inf")).all() and (z[5][w < 0] == -float("inf")).all() and torch.isnan(z[5][w == 0]).all()
    assert torch.isnan(z[9]).all()
    others = [i for i in range(n) if i not in (5, 9)]
    assert torch.equal(z[others], y[others])


def test_votes_of_many_classes_captured_and_on_two_streams():
    sets = []
    for seed, x, n in ((0, "f16", 64), (1, "bits", 40), (2, "bf16", 130)):
        xt, _, packed, _, scales, _ = votes_inputs(n, 1500, 5000, x, 64, "f32", seed=seed)
        sets.append((xt, packed, scales, 64, None, 1500))
    want = [answers.q4_votes(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 3, answers.q4_votes(*sets[i % 3])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [answers.q4_votes(*s) for s in sets]
    for _ in range(3):
        for y in outs:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(outs, want))
    sets[0][0].mul_(-1)  # a replay reads what is there then
    graph.replay()
    assert torch.equal(outs[0], -want[0])


def test_votes_of_more_samples_than_one_launch_takes():
    n, c, k = 530001, 33, 2  # blocks of eight fp32 samples, 65,535 of them a launch
    xt, xv, packed, q, scales, bias = votes_inputs(n, c, k, "f32", 32, "f32")
    check_votes(answers.q4_votes(xt, packed, scales, 32, bias=dev(bias)), xv, q, scales, 32, bias, "f32", c)


def test_votes_of_no_samples_and_infinite_activations():
    xt, xv, packed, q, scales, bias = votes_inputs(4, 100, 20, "f32", 64, "f32")
    assert answers.q4_votes(xt[:0], packed, scales, 64).shape == (0, 20)
    packed = packed.fill_(0x99)  # every weight is 1
    xt[1, 50], xt[2, 99], xt[3, 1] = np.inf, np.nan, -np.inf
    y = f64(answers.q4_votes(xt, packed, scales, 64))
    assert np.isfinite(y[0]).all() and (y[1] == np.inf).all() and np.isnan(y[2]).all() and (y[3] == -np.inf).all()
    big = torch.full((1, 64), 3.0e38, device="cuda")  # finite, above what bf16 rounds to infinity
    big[0, 1:] = 1e-30
    one = torch.full((20, 32), 0x99, dtype=torch.uint8, device="cuda")
    y = f64(answers.q4_votes(big, one, torch.full((20, 1), 0.5, device="cuda"), 64))
    assert (np.abs(y / (0.5 * f64(big)[0, 0]) - 1) <= 4 * U).all()


@pytest.mark.parametrize("n,c,k,x,group,scale", [(1, 16384, 32768, "bf16", 32, "f32"), (1, 16384, 20011, "f32", 128, "f16"),
                                                 (2, 8192, 30000, "f16", 64, "bf16"), (7, 8192, 20000, "bf16", 32, "f32"),
                                                 (1, 16384, 30000, "bits", 64, "f32"), (64, 16384, 8192, "bf16", 32, "f32"),
                                                 (64, 16384, 9000, "bits", 64, "f16"),
                                                 (40, 16384, 20011, "f16", 64, "f16"), (48, 10000, 16000, "bf16", 128, "f32")])
def test_votes_again_and_again(n, c, k, x, group, scale):
    """Streams of many stages over all SMs, call after call on two inputs: a
    stage that is copied over before it is read shows as another result, once
    in some hundred calls."""
    sets = []
    for seed in (1, 2):
        torch.manual_seed(seed)
        words = -(-c // 32)
        packed = torch.randint(0, 256, (k, words * 16), dtype=torch.uint8, device="cuda")
        scales = (torch.rand(k, -(-c // group), device="cuda") + 0.1).to(DT[scale])
        xt = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, words), device="cuda").to(torch.int32) if x == "bits" \
            else torch.randn(n, c, device="cuda").to(DT[x])
        sets.append((xt, packed, scales))
    want = [answers.q4_votes(*s, group, clauses=c) for s in sets]
    other = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        for s, w in zip(sets, want):
            other += (answers.q4_votes(*s, group, clauses=c) != w).sum()
    assert other.item() == 0
    for (xt, packed, scales), w in zip(sets, want):
        rows = torch.randint(0, k, (64,), device="cuda")
        q = nibbles(packed[rows].cpu().numpy(), c).astype(np.int64) - 8
        if x == "bits":
            xv = ((xt.cpu().numpy().view(np.uint32)[:, np.arange(c) // 32] >> (np.arange(c) % 32)) & 1).astype(np.float64)
        else:
            xv = f64(xt)
        check_votes(w[:, rows], xv, q, scales[rows], group, np.zeros(64), "f32", c)


# ------------------------------------------------------------------- answer

def answer_inputs(n, k, dt, hist, mask, bias, seed=0, knobs=True):
    rng = np.random.default_rng(seed)
    cs = rng.integers(-40, 41, (n, k)).astype(np.int32) if dt == "i32" else rng.normal(size=(n, k)).astype(np.float32) * 4
    cst = dev(cs).to(DT[dt])
    kw, kt = {}, {}
    if mask:
        a = rng.random((n if mask == "row" else 1, k)) < 0.6
        if mask == "row" and n > 2:
            a[n // 2] = False
        kw["allowed"] = a
        kt["allowed"] = answers.pack_allowed(a).cuda()
    if bias:
        kw["bias"] = rng.normal(size=(n, k) if bias == "row" else k).astype(np.float32)
        kt["bias"] = dev(kw["bias"])
    if hist:
        h = rng.integers(-2, max(2, min(k + 2, 3 * hist)), (n, hist))
        kw["history"], kt["history"] = h, dev(h).to(torch.int32 if seed % 2 else torch.int64)
        kw["lengths"] = rng.integers(0, hist + 1, n).astype(np.int32)
        kw["lengths"][0] = hist
        kt["lengths"] = dev(kw["lengths"])
    if knobs:
        vals = {"repetition": 1 + rng.random(n), "frequency": rng.random(n), "presence": rng.random(n) * 2,
                "temperature": 0.3 + rng.random(n)}
        for name, v in vals.items():
            v = v.astype(np.float32)
            kw[name], kt[name] = (v, dev(v)) if seed % 3 else (float(v[0]), float(v[0]))
    return cst, kw, kt


def check_answer(got, cst, kw):
    """z: 64-bit arithmetic (a relative 2^-46 of the terms at most) and one
    rounding.  The choice from the rounded z, equal.  The sum S behind the
    log-probability: each term's exponent is off by u of its size (at most 104
    before it vanishes) and exp by 2 steps, and at most k / 32 + 64 merges
    follow one another, 4 roundings each; log1p and the result 3 more."""
    choice, logprob, z = got
    n, k = cst.shape
    want_c, want_lp, want_z = ref_answer(f64(cst), **kw)
    np.testing.assert_array_equal(choice.cpu().numpy(), want_c)
    S = np.expm1(-np.where(np.isfinite(want_lp), want_lp, 0.0))
    rel = (104 + 4 + 4 * (k / 32 + 64)) * U
    tol = rel * S / (1 + S) + 3 * U * np.abs(np.where(np.isfinite(want_lp), want_lp, 0)) + 2.0 ** -126
    lp = f64(logprob)
    fin = np.isfinite(want_lp)
    np.testing.assert_array_equal(np.where(fin, 0, lp), np.where(fin, 0, want_lp))
    assert (np.abs(lp - want_lp)[fin] <= tol[fin]).all()
    if z is not None:
        z = f64(z)
        fin = np.isfinite(want_z) & (np.abs(want_z) < 3.4e38)
        np.testing.assert_array_equal(z[~fin], want_z[~fin].astype(np.float32))
        scale = np.abs(f64(cst)) + 1 + (np.abs(kw["bias"]) if "bias" in kw else 0)
        tol = half_step(torch.float32, want_z) * (1 + 2.0 ** -20) + 2.0 ** -46 * scale * 8
        assert (np.abs(z - np.where(fin, want_z, 0))[fin] <= tol[fin]).all()


@pytest.mark.parametrize("dt", ["i32", "f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,hist,mask,bias", [
    (1, 1, 0, None, None), (1, 2, 1, None, "class"), (3, 10, 5, "row", "class"), (7, 31, 0, "all", "row"),
    (64, 100, 33, "row", None), (5, 257, 40, None, "row"), (33, 1000, 100, "all", "class"), (2, 1025, 0, "row", "row"),
    (3, 4099, 700, "row", "class"), (1, 8193, 9000, "all", None), (2, 40001, 300, "row", "class"),
    (1, 131072, 2000, "row", "class"), (200, 3, 2, None, "class"),
    # clusters without a history, blocks of many tiles, more than fit one count
    (1, 131072, 0, None, "class"), (2, 70001, 0, "row", None), (160, 9000, 0, None, None), (150, 20000, 30, "row", "class"),
    (1, 300001, 50, None, None)])
def test_answer(n, k, hist, mask, bias, dt):
    seed = n + k + (0 if dt == "i32" else len(dt))
    cst, kw, kt = answer_inputs(n, k, dt, hist, mask, bias, seed=seed)
    got = answers.answer(cst, **kt)
    check_answer(got, cst, kw)
    short = answers.answer(cst, adjusted=False, **kt)
    assert short[2] is None and torch.equal(short[0], got[0]) and torch.equal(short[1], got[1])


def test_answer_ties_infinities_nan_and_masked_values():
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    cs = np.array([[3, 3, 1, 3, 0], [-inf, -inf, -inf, -inf, -inf], [low, low, low, low, low], [nan, 1, inf, nan, 2],
                   [1, nan, nan, 5, inf], [1, inf, 2, 3, inf], [inf, 0, 1, -inf, 2], [0, 0, 0, 0, 0],
                   [nan, inf, 7, -inf, low], [1, 2, nan, 3, 4]], np.float32)
    allowed = np.ones((10, 5), bool)
    allowed[4, 1:3] = False  # NaN under the mask
    allowed[4, 4] = False
    allowed[7] = False
    allowed[8, [0, 1, 3, 4]] = False  # one class is left
    allowed[1, [0, 2]] = False
    check_answer(answers.answer(dev(cs), allowed=answers.pack_allowed(allowed).cuda()), dev(cs), {"allowed": allowed})
    for k in (5, 300, 5000):  # equal values far apart: the lowest class
        row = np.zeros((1, k), np.int32)
        row[0, k // 2:] = 9
        assert answers.answer(dev(row))[0].item() == k // 2
    bits = answers.pack_allowed(allowed)
    bits |= ~0x1F  # bits behind the last class are not read
    check_answer(answers.answer(dev(cs), allowed=bits.cuda()), dev(cs), {"allowed": allowed})


def test_answer_int32_extremes_and_large_counts():
    big = 2 ** 31 - 1
    cs = np.array([[big, big - 1, -big - 1, 0, 16777217], [16777217, 16777216, 16777215, 5, 4]], np.int32)
    b = np.array([0.25, 1.5, 0, -3, 0], np.float32)
    for kw in ({}, {"bias": b}, {"bias": b, "temperature": 3.7}):
        kt = {key: dev(v) if isinstance(v, np.ndarray) else v for key, v in kw.items()}
        got = answers.answer(dev(cs), **kt)
        want = ref_answer(cs.astype(np.float64), **kw)
        np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
        np.testing.assert_array_equal(got[2].cpu().numpy(), want[2].astype(np.float32))
    h = np.full((2, 70001), 4)
    h[1, :10] = 0
    kw = {"history": h, "frequency": 0.001, "presence": 0.5, "repetition": 2.0}
    check_answer(answers.answer(dev(cs), **{**kw, "history": dev(h)}), dev(cs), kw)


def test_answer_lengths_outside_the_history_and_no_rows():
    cst, kw, kt = answer_inputs(4, 20, "f32", 6, None, None, seed=1)
    kw["lengths"] = np.array([-3, 0, 6, 100], np.int32)
    got = answers.answer(cst, **{**kt, "lengths": dev(kw["lengths"])})
    check_answer(got, cst, {**kw, "lengths": np.clip(kw["lengths"], 0, 6)})
    empty = answers.answer(cst[:0])
    assert [tuple(t.shape) for t in empty] == [(0,), (0,), (0, 20)]
    none = answers.answer(cst, history=torch.zeros((4, 0), dtype=torch.int64, device="cuda"))
    check_answer(none, cst, {})


@pytest.mark.parametrize("k", [37, 1500, 9001])
def test_answer_strides(k):
    n = 5
    cst, kw, kt = answer_inputs(n, k, "bf16", 50, "row", "row", seed=2)
    wide = torch.zeros((n, k + 3), dtype=torch.bfloat16, device="cuda")
    wide[:, 1:-2] = cst
    wb = torch.zeros((n, k + 5), device="cuda")
    wb[:, 3:-2] = kt["bias"]
    wa = torch.zeros((n, kt["allowed"].shape[1] + 1), dtype=torch.int32, device="cuda")
    wa[:, 1:] = kt["allowed"]
    wh = torch.zeros((n, 57), dtype=kt["history"].dtype, device="cuda")
    wh[:, 7:] = kt["history"]
    check_answer(answers.answer(wide[:, 1:-2], **{**kt, "bias": wb[:, 3:-2], "allowed": wa[:, 1:], "history": wh[:, 7:]}),
                 cst, kw)
    check_answer(answers.answer(cst.t().contiguous().t(), **kt), cst, kw)
    one = cst[:1].expand(n, k)
    check_answer(answers.answer(one, **{**kt, "bias": kt["bias"][:1].expand(n, k)}), one,
                 {**kw, "bias": np.repeat(kw["bias"][:1], n, 0)})


# --------------------------------------------------------------------- loss

def loss_inputs(n, k, dt, mask, weights, bias=True, seed=0, big=1.0):
    rng = np.random.default_rng(seed)
    cs = rng.integers(-60, 61, (n, k)).astype(np.int32) if dt == "i32" else (rng.normal(size=(n, k)) * 4 * big).astype(np.float32)
    cst = dev(cs).to(DT[dt])
    y = rng.integers(0, k, n)
    kw, kt = {}, {}
    if mask:
        a = rng.random((n if mask == "row" else 1, k)) < 0.7
        a[np.arange(n) if mask == "row" else 0, y] = True
        if mask == "row" and n > 3:
            a[n // 2] = False       # nothing allowed
            a[0, y[0]] = k == 1     # the label forbidden
        kw["allowed"], kt["allowed"] = a, answers.pack_allowed(a).cuda()
    if n > 3:
        y[1], y[2] = -100, k  # no label
    if bias:
        kw["bias"] = rng.normal(size=k).astype(np.float32)
        kt["bias"] = dev(kw["bias"])
    if weights:
        w = rng.normal(size=n).astype(np.float32)
        w[-1] = 0 if n > 1 else w[-1]
        kw["weight"], kt["weight"] = w, dev(w)
    t = np.float32(15.5 if dt == "i32" else 0.8)
    kw["temperature"] = t
    kt["temperature"] = dev(np.array([t])) if seed % 2 else float(t)
    return cst, y, kw, kt


def check_loss(got, cst, y, kw):
    """z is off by 4 roundings of (|cs| + |b|) / t at most, so z - m by E, exp
    by 2 steps more, the sum of exp by its longest chain (k / 32 + 64 additions
    or rescalings of 4 roundings), p by P relatively; the gradients by P of p,
    2 roundings of d, and sums over n by their own rounding."""
    loss, dcs, dbias, dt = got
    n, k = cst.shape
    cs = f64(cst)
    want = ref_loss(cs, y, **kw)
    b = kw.get("bias")
    t = float(kw["temperature"])
    w = np.abs(kw["weight"]) if "weight" in kw else np.ones(n)
    mag = np.abs(cs) + (0 if b is None else np.abs(b))
    E = 10 * U * mag.max(1) / t
    P = (E + (4 + 4 * (k / 32 + 64)) * U)[:, None]
    fin = np.isfinite(want[0])
    lo = f64(loss)
    np.testing.assert_array_equal(lo[~fin], want[0][~fin])
    zmax = (mag / t).max(1)
    tol = w * (2 * E + P[:, 0] + 6 * U * (zmax + np.log(k) + 1)) + 2.0 ** -140
    assert (np.abs(lo - want[0])[fin] <= tol[fin]).all()
    d = want[1]
    onehot = np.zeros((n, k))
    use = (np.asarray(y) >= 0) & (np.asarray(y) < k)
    onehot[use, np.asarray(y)[use]] = 1
    p = np.where((w > 0)[:, None], d * t / np.where(w > 0, w, 1)[:, None] * np.sign(kw.get("weight", np.ones(n)))[:, None], 0) + onehot
    dtol = w[:, None] / t * (np.abs(p) * P + 4 * U * (np.abs(p) + onehot)) + 2.0 ** -140
    if dcs is not None:
        tol = dtol + half_step(cst.dtype, np.abs(d) + dtol)
        assert (np.abs(f64(dcs) - d) <= tol).all(), (np.abs(f64(dcs) - d) / tol).max()
        assert (f64(dcs)[(d == 0).all(1)] == 0).all()
    if dbias is not None:
        tol = dtol.sum(0) + (n + 8) * U * np.abs(d).sum(0) + 2.0 ** -140
        assert (np.abs(f64(dbias) - want[2]) <= tol).all(), (np.abs(f64(dbias) - want[2]) / tol).max()
    zz = 2 * mag / t  # |z| and |z - m| are at most this, m as well
    tol = ((dtol * (zz.max(1)[:, None] * 2)).sum() + (np.abs(d) * E[:, None] * 2).sum()
           + (k / 32 + 64) * 2 * U * (np.abs(d) * zz.max(1)[:, None]).sum()) + 2.0 ** -140
    assert abs(float(dt) - want[3]) <= tol + U * abs(want[3])


@pytest.mark.parametrize("dt", ["i32", "f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,mask,weights,bias", [
    (1, 1, None, False, True), (1, 2, None, True, False), (4, 3, "row", True, True), (256, 10, None, False, True),
    (37, 31, "all", True, True), (65, 100, "row", True, False), (1000, 33, "all", False, True), (9, 257, None, True, True),
    (20, 1000, "row", True, True), (7, 1025, "all", False, True), (5, 4099, "row", True, True), (300, 2049, None, False, True),
    (3, 40001, "row", False, True), (4, 131072, None, True, True)])
def test_class_loss(n, k, mask, weights, bias, dt):
    cst, y, kw, kt = loss_inputs(n, k, dt, mask, weights, bias, seed=n + k + len(dt))
    yt = dev(y).to(torch.int64 if n % 2 else torch.int32)
    got = answers.class_loss(cst, yt, **kt)
    assert (got[1] is None) == (dt == "i32") and (got[2] is None) == (not bias)
    check_loss(got, cst, y, kw)
    again = answers.class_loss(cst, yt, **kt)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))  # a fixed order


def test_class_loss_strides_and_no_rows():
    n, k = 6, 1100
    cst, y, kw, kt = loss_inputs(n, k, "f32", "row", True, seed=3)
    wide = torch.zeros((n, k + 3), device="cuda")
    wide[:, 1:-2] = cst
    wa = torch.zeros((n, kt["allowed"].shape[1] + 1), dtype=torch.int32, device="cuda")
    wa[:, 1:] = kt["allowed"]
    yt = dev(np.stack([y, y], 1))[:, 0]
    check_loss(answers.class_loss(wide[:, 1:-2], yt, **{**kt, "allowed": wa[:, 1:]}), cst, y, kw)
    one = cst[:1].expand(n, k)
    check_loss(answers.class_loss(one, yt, **kt), one, y, kw)
    loss, dcs, db, dt = answers.class_loss(cst[:0], yt[:0], bias=kt["bias"])
    assert loss.shape == (0,) and dcs.shape == (0, k) and (db == 0).all() and (dt == 0).all()


def test_class_loss_values_under_the_mask_and_unusual_rows():
    """NaN, infinities and the lowest value count for nothing where masked; a
    row's NaN stays in that row; a certain row has no gradient left."""
    k = 40
    rng = np.random.default_rng(0)
    cs = rng.normal(size=(6, k)).astype(np.float32)
    a = np.ones((6, k), bool)
    a[:4, 5] = False
    y = np.array([0, 1, 2, 3, 7, 8])
    clean = cs.copy()
    cs[:4, 5] = [np.nan, np.inf, -np.inf, np.finfo(np.float32).min]
    clean[:4, 5] = 0
    kw = {"allowed": a, "temperature": np.float32(1.0)}
    got = answers.class_loss(dev(cs), dev(y), allowed=answers.pack_allowed(a).cuda())
    check_loss(got, dev(clean), y, kw)
    cs[4, 30] = np.nan
    loss, dcs, _, _ = answers.class_loss(dev(cs), dev(y), allowed=answers.pack_allowed(a).cuda())
    assert np.isnan(loss[4].item()) and torch.isfinite(loss[[0, 1, 2, 3, 5]]).all()
    assert torch.isnan(dcs[4]).all() and torch.equal(dcs[[0, 1, 2, 3, 5]], got[1][[0, 1, 2, 3, 5]])
    sure = np.full((1, k), -1e4, np.float32)
    sure[0, 3] = 1e4
    loss, dcs, _, dt = answers.class_loss(dev(sure), dev(np.array([3])))
    assert loss.item() == 0 and (dcs == 0).all() and dt.item() == 0
    low = np.full((1, k), -np.inf, np.float32)  # -inf without a mask: probability 0
    low[0, :3] = [1, 2, 3]
    loss, dcs, _, dt = answers.class_loss(dev(low), dev(np.array([1])))
    want = ref_loss(low[:, :3].astype(np.float64), [1])
    assert abs(loss.item() - want[0][0]) <= 8 * U * 4 and (dcs[0, 3:] == 0).all() and np.isfinite(dt.item())


@pytest.mark.parametrize("k", [12, 300, 1000, 5003])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_class_loss_of_the_types_lowest_values(k, dt):
    """A row of nothing but the lowest value is uniform; a label there has a
    finite loss while others are ordinary; the largest value does no harm."""
    tt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dt]
    low, high = torch.finfo(tt).min, torch.finfo(tt).max
    cs = torch.zeros(5, k, dtype=tt, device="cuda")
    cs[0] = low
    cs[1, 3:] = low
    cs[2, 5] = low
    cs[3, 7] = high
    cs[4] = high
    y = np.array([1, 0, 5, 7, k - 1])
    loss, dcs, _, _ = answers.class_loss(cs, dev(y))
    # less the row's largest, which changes no loss: beside 3e38 even 64 bits lose log k
    want = ref_loss(f64(cs) - f64(cs).max(1, keepdims=True), y, temperature=1.0)
    # log k by the sum's chain, the lowest value by four roundings
    tol = 16 * U * np.abs(want[0]) + (k / 32 + 64) * 4 * U
    assert np.isfinite(f64(loss)).all() and (np.abs(f64(loss) - want[0]) <= tol).all()
    # p by ex2 and the sum's chain, its rounding to the type
    tol = (np.abs(want[1]) + 1 / k) * (k / 32 + 72) * 4 * U
    assert (np.abs(f64(dcs) - want[1]) <= tol + half_step(tt, np.abs(want[1]) + tol)).all()


@pytest.mark.parametrize("k", [40, 1030])
def test_class_loss_of_an_infinite_temperature_is_uniform(k):
    rng = np.random.default_rng(1)
    a = rng.random((7, k)) < 0.5
    a[:, 0] = True
    cs = dev(rng.normal(size=(7, k)).astype(np.float32) * 1e4)
    loss, dcs, _, dt = answers.class_loss(cs, dev(np.zeros(7, np.int64)), allowed=answers.pack_allowed(a).cuda(), temperature=float("inf"))
    assert (np.abs(f64(loss) - np.log(a.sum(1))) <= 64 * U).all() and (dcs == 0).all() and dt.item() == 0


def test_class_loss_of_more_chunks_than_one_grid_dimension():
    """Nine million rows of one memory; every row's loss is its label's."""
    n, k = 9_000_001, 513
    cs = dev(np.arange(k, dtype=np.int32)[None] % 7).expand(n, k)
    y = torch.arange(n, device="cuda") % k
    loss, dcs, db, dt = answers.class_loss(cs, y, bias=torch.zeros(k, device="cuda"))
    z = np.arange(k) % 7
    lse = np.log(np.exp(z.astype(np.float64)).sum())
    # ex2 and the sum's chain of 513 terms over 256 threads
    assert (loss - dev((lse - z).astype(np.float32))[y]).abs().max().item() <= 64 * U
    want = n * np.exp(z - lse) - np.bincount(np.arange(n) % k, minlength=k)
    # chunks of 128 rows in fp32, joined in 64 bits: (128 + 64) roundings of the sums' parts
    assert (np.abs(f64(db) - want) <= 192 * U * (n * np.exp(z - lse) + n / k + 1)).all()


def test_class_loss_gradients_against_differences():
    """Central differences of the 64-bit loss (h = 1e-5: error about 1e-9), and
    the kernel's fp32 error as in check_loss, here below 1e-5 of the weights."""
    n, k = 3, 12
    cst, y, kw, kt = loss_inputs(n, k, "f32", "all", True, seed=5)
    got = answers.class_loss(cst, dev(y), **kt)
    cs, h = f64(cst), 1e-5
    f = lambda cs=cs, **over: ref_loss(cs, y, **{**kw, **over})[0].sum()  # noqa: E731
    for i in range(n):
        for j in range(k):
            e = np.zeros((n, k))
            e[i, j] = h
            assert abs((f(cs + e) - f(cs - e)) / (2 * h) - got[1][i, j].item()) < 1e-5
    b, t = kw["bias"].astype(np.float64), float(kw["temperature"])
    for j in range(k):
        e = np.zeros(k)
        e[j] = h
        assert abs((f(bias=b + e) - f(bias=b - e)) / (2 * h) - got[2][j].item()) < 1e-5
    assert abs((f(temperature=t + h) - f(temperature=t - h)) / (2 * h) - got[3].item()) < 1e-4


# ----------------------------------------------------- refusals, streams, graphs

def test_refusals():
    z = torch.zeros((3, 8), device="cuda")
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    bad = [
        lambda: answers.answer(z, bias=torch.zeros(7, device="cuda")),
        lambda: answers.answer(z, bias=torch.zeros((2, 8), device="cuda")),
        lambda: answers.answer(z, bias=torch.zeros(8)),
        lambda: answers.answer(z, bias=[0.0] * 8),
        lambda: answers.answer(z, allowed=torch.zeros((2, 1), dtype=torch.int32, device="cuda")),
        lambda: answers.answer(z, allowed=torch.ones((3, 8), dtype=torch.bool, device="cuda")),
        lambda: answers.answer(z, lengths=i.int()),
        lambda: answers.answer(z, history=torch.zeros((2, 4), dtype=torch.int64, device="cuda")),
        lambda: answers.answer(z, history=torch.zeros((3, 4), device="cuda")),
        lambda: answers.answer(z, history=torch.zeros((3, 4), dtype=torch.int64, device="cuda"), lengths=i),
        lambda: answers.answer(z, temperature=0.0), lambda: answers.answer(z, temperature=1e-50),
        lambda: answers.answer(z, temperature=float("nan")),
        lambda: answers.answer(z, repetition=-1.0),
        lambda: answers.answer(z, presence=torch.zeros(2, device="cuda")),
        lambda: answers.answer(torch.zeros((3, 0), device="cuda")),
        lambda: answers.answer(z.clone().requires_grad_()),
        lambda: answers.class_loss(z, i[:2]),
        lambda: answers.class_loss(z, i.float()),
        lambda: answers.class_loss(z, i, temperature=-1),
        lambda: answers.class_loss(z, i, weight=torch.zeros(3, dtype=torch.float64, device="cuda")),
        lambda: answers.class_loss(z.clone().requires_grad_(), i),
        lambda: answers.q4_pack(z, group=16),
        lambda: answers.q4_pack(z, scale_dtype=torch.float64),
        lambda: answers.q4_pack(z[:0]),
    ]
    p, s = answers.q4_pack(torch.ones((40, 8), device="cuda"), 32)
    x = torch.zeros((2, 40), device="cuda")
    assert answers.q4_votes(x, p, s, 32).shape == (2, 8)
    bad += [
        lambda: answers.q4_votes(x[:, :39], p, s, 32, clauses=40),
        lambda: answers.q4_votes(x, p, s, 64),
        lambda: answers.q4_votes(x, p, s, 48),
        lambda: answers.q4_votes(x, p[:, :16], s, 32),
        lambda: answers.q4_votes(x, p[::2], s[:4], 32),
        lambda: answers.q4_votes(x, p, s[:, :1], 32),
        lambda: answers.q4_votes(torch.zeros((2, 2), dtype=torch.int32, device="cuda"), p, s, 32),
        lambda: answers.q4_votes(x, p, s, 32, out_dtype=torch.int32),
        lambda: answers.q4_votes(x, p, s, 32, bias=torch.zeros(9, device="cuda")),
        lambda: answers.q4_votes(x.double(), p, s, 32),
    ]
    for f in bad:
        with pytest.raises((TypeError, ValueError)):
            f()
    off = torch.zeros(8 * 32 + 1, dtype=torch.uint8, device="cuda")[1:].view(8, 32)
    with pytest.raises(_lib.YTMError, match="16-byte"):
        answers.q4_votes(x, off, s, 32)
    with torch.no_grad():  # leaves are fine where nothing is recorded
        answers.answer(z.clone().requires_grad_())


def _chain(x, packed, scales, bias, allowed, history, y):
    cs = answers.q4_votes(x, packed, scales, 64, bias=bias)
    out = answers.answer(cs, bias=bias, allowed=allowed, history=history, frequency=0.5, temperature=2.0)
    return [cs, *out, *answers.class_loss(cs, y, bias=bias, allowed=allowed, temperature=3.0)]


def _chain_inputs(n, c, k, seed):
    xt, _, packed, _, scales, bias = votes_inputs(n, c, k, "f32", 64, "f32", seed)
    rng = np.random.default_rng(seed)
    a = answers.pack_allowed(rng.random((n, k)) < 0.8).cuda()
    h = dev(rng.integers(0, k, (n, 9)))
    return [xt, packed, scales, dev(bias), a, h, dev(rng.integers(0, k, n))]


@pytest.mark.parametrize("n,c,k", [(1, 300, 50), (6, 2000, 3001)])
def test_captured_calls_follow_their_inputs(n, c, k):
    """The three operators one after another in a graph, two graphs of them
    replayed in turn on new inputs, against the same calls made eagerly."""
    sets = [_chain_inputs(n, c, k, s) for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _chain(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _chain(*s)
        graphs.append((g, s, outs))
    for seed in (11, 12, 13):
        new = [_chain_inputs(n, c, k, seed + 10 * j) for j in range(2)]
        for (g, s, _), v in zip(graphs, new):
            for t, u in zip(s, v):
                t.copy_(u)
            g.replay()
        for (g, s, outs), v in zip(graphs, new):
            for a, b in zip(outs, _chain(*v)):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    sets = [_chain_inputs(4, 3000, 2000, s) for s in range(6)]
    want = [_chain(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_chain(*s))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ------------------------------------------------------------ the model's path

@pytest.mark.parametrize("patch,count_empty,clauses", [((5, 5), False, 40), (None, False, 301), ((5, 5), True, 40)])
def test_infer_fired_gives_the_counted_clauses(patch, count_empty, clauses):
    cfg = _lib.make_config(clauses_per_class=clauses, T=20, s=4.0, dim=(8, 8, 1), n_classes=3, patch_dim=patch, seed=3,
                           count_empty=count_empty)
    eng = CudaEngine(cfg, "cuda:0")
    rng = np.random.default_rng(0)
    half = cfg.number_of_ta_states // 2
    ta = rng.integers(0, half + 1, size=(eng.C, eng.L), dtype=np.uint32)
    for c in range(eng.C):
        if c % 5:
            ta[c, rng.choice(eng.L, size=rng.integers(1, 4), replace=False)] = half + 3
    eng.set_ta_state(ta)
    lits = eng.encode(dev((rng.random((50, 64)) < 0.4).astype(np.int32)))
    fired = eng.infer_fired(lits).cpu().numpy().view(np.uint32)
    bits = (fired[:, np.arange(eng.C) // 32] >> (np.arange(eng.C) % 32)) & 1
    want = eng.transform(lits).cpu().numpy().astype(np.uint32)
    if not count_empty:
        want[:, (ta > half).sum(1) == 0] = 0
    np.testing.assert_array_equal(bits, want)
    if eng.C % 32:
        assert (fired[:, -1] >> (eng.C % 32) == 0).all()
    assert eng.infer_fired(lits[:0]).shape == (0, (eng.C + 31) // 32)


def test_model_path_from_packed_votes_to_answers():
    """fit, pack, calibrate and answer as a user would, against the oracle's
    clause outputs, the reference packing and the reference adjustment."""
    rng = np.random.default_rng(4)
    n, k = 80, 5
    y = rng.integers(0, k, n)
    proto = rng.random((k, 64)) < 0.3
    X = (proto[y] ^ (rng.random((n, 64)) < 0.05)).astype(np.uint32)
    kw = dict(number_of_clauses_per_class=70, T=30, s=4.0, dim=(8, 8, 1), n_classes=k, patch_dim=(6, 6), seed=9)
    tm = MultiClassTM(**kw)
    tm.fit(X, y, batch_size=8)
    votes = tm.pack_votes(group=32)
    o = O.Oracle(**kw)
    ta, w = tm.get_ta_state().reshape(o.C, -1), tm.get_weights().reshape(o.C, k)
    fired = o.transform(ta, o.encode(X)).astype(np.float64)
    fired[:, (ta > 128).sum(1) == 0] = 0
    q, _ = ref_pack(w, 32)
    s = f64(votes.scales)
    want, mag = ref_votes(fired, q, s, 32)
    cs = tm.score(X, False, votes=votes)
    assert cs.dtype == np.float32 and (np.abs(cs - want) <= (32 + 3 + 64) * 2 * U * mag + 1e-30).all()
    preds, cs2 = tm.predict(X, votes=votes)
    np.testing.assert_array_equal(cs2, cs)
    np.testing.assert_array_equal(preds, np.argmax(cs, 1))
    # rounding a weight moves it by at most half a scale
    full = tm.score(X, False)
    assert (np.abs(cs - full) <= np.repeat(s, 32, 1)[:, :o.C].sum(1) / 2 + 1e-3).all()
    bias, t = tm.calibrate(X, y, steps=20)
    assert bias.shape == (k,) and bias.dtype == np.float32 and t > 0 and np.isfinite(bias).all()
    allowed = rng.random((n, k)) < 0.7
    allowed[3] = False
    hist = rng.integers(-1, k, (n, 4))
    lens = rng.integers(0, 5, n)
    rep = (1 + rng.random(n)).astype(np.float32)
    choice, logprob, z = tm.answer(X, bias=bias, allowed=allowed, history=hist, lengths=lens, repetition=rep, presence=0.5,
                                   temperature=t)
    wc, wl, wz = ref_answer(full.astype(np.float64), bias, allowed, hist, lens, rep, 0.0, 0.5, t)
    np.testing.assert_array_equal(choice, wc)
    np.testing.assert_array_equal(z, wz.astype(np.float32))
    assert choice[3] == -1 and (logprob[3] == -np.inf) and (choice[allowed.any(1)] >= 0).all()
    plain = tm.answer(X)
    np.testing.assert_array_equal(plain[0], tm.predict(X)[0])
    np.testing.assert_array_equal(plain[2], full)
    tm.fit(X, y, batch_size=8)  # the packed copy stays as it was
    votes2 = tm.pack_votes(group=32)
    assert votes2.packed.data_ptr() != votes.packed.data_ptr()


def test_multi_output_scores_from_packed_votes():
    rng = np.random.default_rng(6)
    X = (rng.random((40, 64)) < 0.4).astype(np.uint32)
    Y = (rng.random((40, 3)) < 0.5).astype(np.uint32)
    tm = MultiOutputTM(number_of_clauses_per_class=20, T=15, s=4.0, dim=(8, 8, 1), n_classes=3, seed=2)
    tm.fit(X, Y)
    votes = tm.pack_votes(group=64)
    full, cs = tm.score(X, False), tm.score(X, False, votes=votes)
    # rounding a weight moves it by at most half a scale
    assert (np.abs(cs - full) <= 64 * f64(votes.scales).sum(1) / 2 + 1e-3).all()
    preds, cs2 = tm.predict(X, votes=votes)
    np.testing.assert_array_equal(cs2, cs)
    np.testing.assert_array_equal(preds, (cs >= 0).astype(np.uint32))
