"""Workloads of the operators between clause outputs and answers (ytm_b200.answers).

Three operators: the vote of 4-bit clause weights with group scales
(`q4_votes`), the adjustment of class sums by biases, allowed classes and
penalties with the choice of an answer (`answer`), and the cross entropy of
adjusted class sums with its gradients (`class_loss`).  `run` computes them in
their plain form from elementary torch operations, or, with `own` set, by the
framework's calls.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one sample's vote in the 10,000-clause, 10-class coalesced machine: latency only
        _votes("votes digits, one", 1, 10000, 10, "bits", 64, "f32"),
        # one sample's vote in the 65,536-clause, 100-class machine
        _votes("votes 64k clauses, one", 1, 65536, 100, "bits", 64, "bf16"),
        # one step of a machine that answers with one of many tokens: 268 MB of weights
        _votes("votes tokens, one", 1, 16384, 32768, "bf16", 128, "f16"),
        # a few samples with real-valued clause activations, sizes that fit no tile
        _votes("votes odd, five", 5, 10007, 5003, "f32", 32, "f32"),
        # a served batch over many tokens
        _votes("votes tokens, batch", 48, 8192, 16384, "f16", 64, "f16", out="bf16"),
        # one sample's ten class sums with a bias
        _answer("answer digits, one", 1, 10, "i32", hist=0, mask="none", bias="class", z=True),
        # one decoding step over a large vocabulary: everything on, only the answer wanted
        _answer("answer tokens, one", 1, 131072, "f32", hist=2000, mask="row", bias="class", z=False),
        # a decoding step of a batch with ragged histories, a grammar mask for each row
        _answer("answer tokens, batch", 64, 32001, "bf16", hist=700, mask="row", bias="row", z=True),
        # the class sums of many samples of the 100-class machine, a common set of allowed classes
        _answer("answer 100 classes, many", 65536, 100, "i32", hist=0, mask="all", bias="class", z=True),
        # calibration on a mini-batch of 256 with ten classes
        _loss("loss digits, batch", 256, 10, "i32", mask="none", weights=False),
        # calibration of the 100-class machine on many samples
        _loss("loss 100 classes, many", 262144, 100, "i32", mask="all", weights=True),
        # a training step's loss over many tokens, sizes that fit no tile
        _loss("loss tokens, step", 2047, 32001, "bf16", mask="row", weights=True),
    ]


def _votes(name, n, c, k, x, group, scale, out="f32"):
    return {"name": name, "op": "votes", "n": n, "c": c, "k": k, "x": x, "group": group, "scale": scale, "out": out}


def _answer(name, n, k, dt, hist, mask, bias, z):
    return {"name": name, "op": "answer", "n": n, "k": k, "dt": dt, "hist": hist, "mask": mask, "bias": bias, "z": z}


def _loss(name, n, k, dt, mask, weights):
    return {"name": name, "op": "loss", "n": n, "k": k, "dt": dt, "mask": mask, "weights": weights}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["votes", "answer", "loss"])
    if op == "votes":
        n = _log(rng, 1, 64)
        c = _log(rng, 500, 65536)
        k = _log(rng, 2, max(2, min(32768, (1 << 29) // c, (1 << 32) // (c * n))))
        case = _votes("", n, c, k, rng.choice(["bits", "f32", "bf16", "f16"]), rng.choice([32, 64, 128]),
                      rng.choice(["f32", "bf16", "f16"]), rng.choice(["f32", "f32", "bf16", "f16"]))
    elif op == "answer":
        k = _log(rng, 2, 131072)
        n = _log(rng, 1, max(1, min(65536, 6000000 // k)))
        hist = rng.choice([0, 1, _log(rng, 2, 4000)]) if n * k > 64 else rng.choice([0, 1, 40])
        case = _answer("", n, k, rng.choice(["i32", "f32", "bf16", "f16"]), min(hist, max(1, 2000000 // n)),
                       rng.choice(["none", "all", "row"]), rng.choice(["none", "class", "row"]), rng.choice([True, True, False]))
    else:
        k = _log(rng, 3, 131072)
        n = _log(rng, 4, max(4, min(262144, 26000000 // k)))
        case = _loss("", n, k, rng.choice(["i32", "f32", "bf16", "f16"]), rng.choice(["none", "all", "row"]),
                     rng.choice([True, False]))
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs

def _words(bits):
    """Booleans [R, 32 * w] as int32 words [R, w], bit j of a word the j-th of its 32."""
    at = torch.arange(32, device=bits.device, dtype=torch.int64)
    w = (bits.view(bits.shape[0], -1, 32).to(torch.int64) << at).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _sums(gen, n, k, dt):
    """Class sums as a machine with a threshold in the hundreds gives them, or logits of the same spread as real numbers."""
    v = torch.randn(n, k, generator=gen, device=DEV)
    return (v * 60).round().to(torch.int32) if dt == "i32" else (v * 4).to(DTYPES[dt])


def _mask(gen, n, k, mask):
    if mask == "none":
        return None
    rows = n if mask == "row" else 1
    bits = torch.rand(rows, -(-k // 32) * 32, generator=gen, device=DEV) < 0.7
    bits[:, 0] |= mask == "all"
    if mask == "row" and n > 4:
        bits[n // 2] = False  # a row whose grammar leaves nothing
    return _words(bits)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    s = {"case": case}
    n, k = case["n"], case["k"]
    if case["op"] == "votes":
        c, group = case["c"], case["group"]
        cp = -(-c // 32) * 32
        rows = max(1, (1 << 26) // cp)
        packed = torch.empty(k, cp // 2, dtype=torch.uint8, device=DEV)
        for i in range(0, k, rows):
            q = (torch.randn(min(rows, k - i), cp, generator=gen, device=DEV) * 2.5 + 8).round_().clamp_(1, 15).to(torch.uint8)
            q[:, c:] = 8
            packed[i:i + rows] = q[:, 0::2] | (q[:, 1::2] << 4)
        s["packed"] = packed
        s["scales"] = (torch.rand(k, -(-c // group), generator=gen, device=DEV) * 4 + 0.5).to(DTYPES[case["scale"]])
        s["bias"] = torch.randn(k, generator=gen, device=DEV) * 10
        if case["x"] == "bits":
            bits = torch.rand(n, cp, generator=gen, device=DEV) < 0.1
            bits[:, c:] = False
            s["x"] = _words(bits)
        else:
            s["x"] = torch.randn(n, c, generator=gen, device=DEV).to(DTYPES[case["x"]])
        return s
    s["cs"] = _sums(gen, n, k, case["dt"])
    s["allowed"] = _mask(gen, n, k, case["mask"])
    if case["op"] == "answer":
        s["bias"] = None
        if case["bias"] != "none":
            s["bias"] = torch.randn(n if case["bias"] == "row" else 1, k, generator=gen, device=DEV)
            s["bias"] = s["bias"] if case["bias"] == "row" else s["bias"][0]
        s["history"] = s["lengths"] = None
        if case["hist"]:
            h = case["hist"]
            u = torch.rand(n, h, generator=gen, device=DEV)
            s["history"] = (u * u * k).to(torch.int64).clamp_(max=k - 1)  # some classes far more often than others
            s["lengths"] = torch.randint(0, h + 1, (n,), generator=gen, device=DEV, dtype=torch.int32)
            s["lengths"][0] = h
        rows = torch.rand(4, n, generator=gen, device=DEV)
        if n > 1:
            s["knobs"] = {"repetition": 1 + rows[0] / 2, "frequency": rows[1] / 2, "presence": rows[2], "temperature": 0.5 + rows[3]}
        else:
            s["knobs"] = {"repetition": 1.25, "frequency": 0.125, "presence": 0.5, "temperature": 0.75}
        if case["dt"] == "i32":  # whole-number class sums lie twenty times as far apart
            s["knobs"]["temperature"] = s["knobs"]["temperature"] * 20
        if not case["hist"]:
            s["knobs"] = {"temperature": s["knobs"]["temperature"]}
        return s
    s["bias"] = torch.randn(k, generator=gen, device=DEV)
    s["target"] = torch.randint(0, k, (n,), generator=gen, device=DEV)
    s["target"][1::17] = -1  # rows without a label
    if s["allowed"] is not None:  # a label is an allowed class: the row's mask gets its bit
        t = s["target"].clamp(min=0)
        bit = (torch.ones_like(t) << (t % 32))
        bit = torch.where(bit >= 2 ** 31, bit - 2 ** 32, bit).to(torch.int32)
        if case["mask"] == "row":
            at = torch.arange(n, device=DEV)
            s["allowed"][at, t // 32] |= bit
            if n > 4:
                s["allowed"][n // 2] = 0
                s["target"][n // 2] = -1
        else:
            s["allowed"].fill_(-1)
            s["allowed"][:, 0] &= ~2  # one class left out for all
            s["target"][s["target"] == 1] = 0
    s["temperature"] = torch.rand(1, generator=gen, device=DEV) + (20 if case["dt"] == "i32" else 0.75)
    s["weight"] = torch.rand(n, generator=gen, device=DEV) / n if case["weights"] else None
    return s


# ------------------------------------------------------------- plain forms

def _unpack(packed, c):
    return torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1)[:, :c]


def _bits(words, count):
    at = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> at) & 1).view(words.shape[0], -1)[:, :count]


def _plain_votes(s, case):
    c, group = case["c"], case["group"]
    q = _unpack(s["packed"], c).float() - 8
    w = q * s["scales"].float().repeat_interleave(group, 1)[:, :c]
    x = _bits(s["x"], c).float() if case["x"] == "bits" else s["x"].float()
    return (x @ w.t() + s["bias"]).to(DTYPES[case["out"]])


def _column(v):
    return v.double().unsqueeze(1) if isinstance(v, torch.Tensor) else v


def _plain_answer(s, case):
    n, k = case["n"], case["k"]
    # 64 bits up to the rounding of the adjusted values: equal and nearly equal values decide the choice
    v = s["cs"].double()
    knobs = s["knobs"]
    if case["hist"]:
        h = case["hist"]
        live = torch.arange(h, device=v.device) < s["lengths"].unsqueeze(1)
        count = torch.zeros(n, k, device=v.device).scatter_add_(1, s["history"], live.float()).double()
        r = _column(knobs["repetition"])
        hit = torch.where(v > 0, v / r, v * r) - _column(knobs["frequency"]) * count - _column(knobs["presence"])
        v = torch.where(count > 0, hit, v)
    if s["bias"] is not None:
        v = v + s["bias"]
    z = (v / _column(knobs["temperature"])).float()
    if s["allowed"] is not None:
        z = torch.where(_bits(s["allowed"], k) > 0, z, -math.inf)
    top = z.amax(1, keepdim=True)
    at = torch.arange(k, device=z.device)
    choice = torch.where(z == top, at, k).amin(1)
    none = top[:, 0] == -math.inf
    others = torch.where(at == choice.unsqueeze(1), 0.0, torch.exp(z - top)).sum(1)
    logprob = torch.where(none, -math.inf, -torch.log1p(others))
    choice = torch.where(none, -1, choice)
    return [choice, logprob, z] if case["z"] else [choice, logprob]


def _plain_loss(s, case):
    n, k = case["n"], case["k"]
    t = s["temperature"]
    z = (s["cs"].float() + s["bias"]) / t
    if s["allowed"] is not None:
        z = torch.where(_bits(s["allowed"], k) > 0, z, -math.inf)
    y = s["target"].clamp(min=0)
    w = torch.where(s["target"] >= 0, 1.0 if s["weight"] is None else s["weight"], 0.0).unsqueeze(1)
    z = torch.where(w > 0, z, 0.0)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    zy = z.gather(1, y.unsqueeze(1))
    loss = (w * (top + torch.log(total) - zy))[:, 0]
    d = e / total
    d = d - (torch.arange(k, device=d.device) == y.unsqueeze(1)).float()
    d = d * w
    dt = -(torch.where(d == 0, 0.0, d * z).sum(1, dtype=torch.float64).sum() / t.double()).float()
    d = d / t
    db = d.sum(0, dtype=torch.float64).float()
    return [loss, db, dt] if case["dt"] == "i32" else [loss, d.to(DTYPES[case["dt"]]), db, dt]


def run(state):
    s, case = state, state["case"]
    if own:
        from ytm_b200 import answers
        if case["op"] == "votes":
            return answers.q4_votes(s["x"], s["packed"], s["scales"], case["group"], bias=s["bias"], clauses=case["c"],
                                    out_dtype=DTYPES[case["out"]])
        if case["op"] == "answer":
            choice, logprob, z = answers.answer(s["cs"], bias=s["bias"], allowed=s["allowed"], history=s["history"],
                                                lengths=s["lengths"], adjusted=case["z"], **s["knobs"])
            return [choice, logprob, z] if case["z"] else [choice, logprob]
        loss, d, db, dt = answers.class_loss(s["cs"], s["target"], bias=s["bias"], allowed=s["allowed"],
                                             temperature=s["temperature"], weight=s["weight"])
        return [loss, db, dt] if case["dt"] == "i32" else [loss, d, db, dt]
    return {"votes": _plain_votes, "answer": _plain_answer, "loss": _plain_loss}[case["op"]](s, case)


def work(case):
    n, k = case["n"], case["k"]
    mask = {"none": 0, "all": 1, "row": n}[case.get("mask", "none")] * -(-k // 32) * 4
    if case["op"] == "votes":
        c = case["c"]
        x = n * (-(-c // 32) * 4 if case["x"] == "bits" else c * BYTES[case["x"]])
        weights = k * (-(-c // 32) * 16 + -(-c // case["group"]) * BYTES[case["scale"]] + 4)
        return {"bytes": weights + x + n * k * BYTES[case["out"]], "flops": 2 * n * k * c}
    if case["op"] == "answer":
        bias = {"none": 0, "class": 1, "row": n}[case["bias"]] * k * 4
        return {"bytes": n * k * (BYTES[case["dt"]] + (4 if case["z"] else 0)) + bias + mask + n * case["hist"] * 8 + n * 32,
                "flops": 10 * n * k}
    return {"bytes": n * k * (4 if case["dt"] == "i32" else 2 * BYTES[case["dt"]]) + 8 * k + mask + n * 16, "flops": 15 * n * k}


# ------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    n, k = case["n"], case["k"]
    bias = None if s["bias"] is None else s["bias"].double()
    if case["op"] == "votes":
        # group by group: whole-number products first, then the scale
        c, group = case["c"], case["group"]
        full = -(-c // group) * group
        x = torch.zeros(n, full, dtype=torch.float64, device=DEV)
        if case["x"] == "bits":
            j = torch.arange(c, device=DEV)
            x[:, :c] = ((s["x"].long()[:, j // 32] >> (j % 32)) % 2).double()
        else:
            x[:, :c] = s["x"].double()
        xg = x.view(n, -1, group).permute(1, 2, 0)  # group, member, sample
        y = torch.empty(n, k, dtype=torch.float64, device=DEV)
        rows = max(1, (1 << 26) // full)
        for i in range(0, k, rows):
            p = s["packed"][i:i + rows].long()
            q = torch.zeros(p.shape[0], full, dtype=torch.float64, device=DEV)
            q[:, 0:c:2] = (p % 16)[:, :(c + 1) // 2].double() - 8
            q[:, 1:c:2] = (p // 16)[:, :c // 2].double() - 8
            part = torch.bmm(q.view(p.shape[0], -1, group).permute(1, 0, 2), xg)
            y[:, i:i + rows] = (part * s["scales"][i:i + rows].double().t().unsqueeze(2)).sum(0).t()
        return y + bias
    if s["allowed"] is not None:
        j = torch.arange(k, device=DEV)
        open_ = ((s["allowed"].long()[:, j // 32] >> (j % 32)) % 2 == 1).expand(n, k)
    else:
        open_ = torch.ones(1, 1, dtype=torch.bool, device=DEV).expand(n, k)
    if case["op"] == "answer":
        col = {a: torch.as_tensor(b, dtype=torch.float64, device=DEV).reshape(-1, 1) for a, b in s["knobs"].items()}
        v = s["cs"].to(torch.float64).clone()
        if case["hist"]:
            live = torch.arange(case["hist"], device=DEV)[None, :] < s["lengths"][:, None]
            places = (torch.arange(n, device=DEV)[:, None] * k + s["history"])[live]
            where, times = places.unique(return_counts=True)
            row = where // k
            old = v.view(-1)[where]
            take = lambda a: col[a].expand(n, 1)[row, 0]  # noqa: E731
            new = torch.where(old > 0, old / take("repetition"), old * take("repetition"))
            v.view(-1)[where] = new - take("frequency") * times - take("presence")
        if bias is not None:
            v += bias
        z = (v / col["temperature"]).masked_fill(~open_, -math.inf)
        some = open_.any(1)
        # equal after the rounding of the adjusted values is equal: the lowest index of them
        shown = z.to(torch.float32)
        choice = torch.where(some, (shown == shown.max(1, keepdim=True).values).to(torch.uint8).argmax(1), -1)
        best = choice.clamp(min=0)[:, None]
        others = (z - z.gather(1, best)).exp().scatter(1, best, 0.0)
        logprob = torch.where(some, -torch.log1p(others.sum(1)), -math.inf)
        return [choice, logprob, z] if case["z"] else [choice, logprob]
    temp = s["temperature"].double()
    loss = torch.zeros(n, dtype=torch.float64, device=DEV)
    weight = torch.ones(n, dtype=torch.float64, device=DEV) if s["weight"] is None else s["weight"].double()
    db, dt = torch.zeros(k, dtype=torch.float64, device=DEV), torch.zeros(1, dtype=torch.float64, device=DEV)
    floats = case["dt"] != "i32"
    dcs = torch.zeros(n, k, dtype=torch.float64, device=DEV) if floats else None
    rows = max(1, (1 << 26) // k)
    for i in range(0, n, rows):
        use = (s["target"][i:i + rows] >= 0).nonzero()[:, 0] + i
        z = ((s["cs"][use].double() + bias) / temp).masked_fill(~open_[use], -math.inf)
        logp = torch.log_softmax(z, 1)
        y, w = s["target"][use][:, None], weight[use][:, None]
        loss[use] = -(w * logp.gather(1, y))[:, 0]
        g = w * logp.exp()
        g.scatter_add_(1, y, -w)
        dt -= (g * z.masked_fill(~open_[use], 0.0)).sum() / temp
        g /= temp
        db += g.sum(0)
        if floats:
            dcs[use] = g
    return [loss, dcs, db, dt] if floats else [loss, db, dt]
