"""What the operators on the features of the rows have to do: sizes, inputs, plain forms.

``attention`` (softmax over the rows of an example, optionally with capped
scores and a bias by distance), ``norm_rotate`` (norm of queries and keys per
head, rotated by the rows' positions) and ``lookup`` (rows by index, and the
gradient of the table) are what a layer of a point-cloud network does with its
rows next to searching their neighbours.  A case is a dict of plain values;
``"op"`` says which operator it goes through.  A pass is one call, with its
gradients where ``"train"`` is set.

Where ``own`` is false the operators are computed in their plain form, from
elementary torch operations in 32 bits (angles in 64), rounded once at the end;
where it is true by this package's entry points.  ``exact`` computes them in 64
bits, example by example.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def listed():
    return [
        # ---- attention ----------------------------------------------------
        # one object of 1,024 points in an interactive program, full precision:
        # all latency
        _attention("one_cloud", examples=1, rows=1024, heads=4, d=32,
                   dtype="f32", axes=3),
        # one query per example against all of its rows (a readout token per
        # scan, per document): 32 examples of very different lengths, shared
        # key heads
        _attention("readout", examples=32, rows=8192, ragged=True,
                   queries=1, heads=8, kv_heads=2, d=128, dtype="bf16"),
        # training of a layer over a batch of objects, biased by distance
        _attention("clouds_train", examples=16, rows=1024, heads=8, d=64,
                   dtype="bf16", axes=3, train=True),
        # the same in full precision with uneven objects and heads of odd
        # width, capped scores
        _attention("ragged_f32_train", examples=12, rows=1300, ragged=True,
                   heads=4, d=48, dtype="f32", cap=20.0, train=True),
        # a mini-batch of many molecule-sized graphs
        _attention("tiny_graphs_train", examples=1000, rows=65, ragged=True,
                   heads=4, d=32, dtype="f16", axes=3, train=True),
        # the largest: long examples, everything on; positions on one axis
        # (time stamps of a sequence)
        _attention("long_train", examples=4, rows=4096, heads=8, d=128,
                   dtype="bf16", axes=1, cap=30.0, train=True),
        # sampled rows (every eighth) look at all rows of their scan
        _attention("samples", examples=4, rows=8192, ragged=True, queries=8,
                   heads=8, d=64, dtype="f16", axes=3),
        # ---- norm_rotate ---------------------------------------------------
        # queries and keys of one small object
        {"name": "rotate_small", "op": "norm_rotate", "rows": 1024,
         "heads": 4, "kv_heads": 4, "d": 32, "axes": 3, "rotated": 15,
         "dtype": "f32", "train": False},
        # a training step's queries and keys over a batch of scans, with the
        # gradients of both gains
        {"name": "rotate_train", "op": "norm_rotate", "rows": 131072,
         "heads": 8, "kv_heads": 2, "d": 128, "axes": 3, "rotated": 63,
         "dtype": "bf16", "train": True},
        # ---- lookup --------------------------------------------------------
        # features of the neighbours of a small graph, inference
        {"name": "edges_small", "op": "lookup", "table": 1024, "width": 64,
         "entries": 16 * 1024, "skew": 1.0, "none": 0.0, "dtype": "f32",
         "train": False},
        # the same over the graph of a batch of clouds, training; a table of
        # fixed degree in which some places are empty
        {"name": "edges_train", "op": "lookup", "table": 65536, "width": 64,
         "entries": 20 * 65536, "skew": 1.0, "none": 0.05, "dtype": "f32",
         "train": True},
        # code-book entries of a million rows, few codes very frequent
        {"name": "codes_train", "op": "lookup", "table": 4096, "width": 64,
         "entries": 1 << 20, "skew": 4.0, "none": 0.0, "dtype": "bf16",
         "train": True},
    ]


def _attention(name, examples, rows, heads, d, dtype, kv_heads=0,
               ragged=False, queries=0, axes=0, cap=0.0, train=False):
    """queries: 0 = every row is a query, 1 = one per example, s > 1 = every
    s-th row."""
    return {"name": name, "op": "attention", "examples": examples,
            "rows": rows, "ragged": ragged, "queries": queries,
            "heads": heads, "kv_heads": kv_heads or heads, "d": d,
            "axes": axes, "cap": cap, "dtype": dtype, "train": train}


def _between(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm_rotate", "lookup"])
    dtype = rng.choice(sorted(DTYPES))
    train = rng.random() < 0.5
    if op == "attention":
        while True:
            kv_heads = rng.choice([1, 2, 3, 4, 8])
            c = _attention(
                None, examples=_between(rng, 1, 1000),
                rows=_between(rng, 1, 8192), ragged=rng.random() < 0.7,
                queries=rng.choice([0, 0, 1, _between(rng, 2, 16)]),
                heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads,
                d=rng.choice([16, 32, 48, 64, 80, 96, 128,
                              rng.randint(5, 128)]),
                dtype=dtype, axes=rng.choice([0, 1, 2, 3]),
                cap=rng.choice([0.0, 10.0, 50.0]), train=train)
            del c["name"]
            # (scores of the plain form, which pads to the longest example)
            nq, nk = _longest(c)
            padded = c["examples"] * nq * nk * c["heads"]
            if (c["heads"] <= 16 and padded <= 4 * 8 * 4096 * 4096
                    and padded >= 1000 and c["examples"] * nk <= 300000):
                return c
    if op == "norm_rotate":
        kv_heads = rng.choice([1, 2, 4, 8])
        d = rng.choice([16, 32, 48, 64, 80, 96, 128, rng.randint(5, 128)])
        return {"op": op, "rows": _between(rng, 1, 100000),
                "heads": kv_heads * rng.choice([1, 1, 2]),
                "kv_heads": kv_heads, "d": d, "axes": rng.randint(1, 3),
                "rotated": rng.choice([d // 2, rng.randint(1, d // 2)]),
                "dtype": dtype, "train": train}
    return {"op": op, "table": _between(rng, 1, 200000),
            "width": rng.choice([16, 32, 64, 128, rng.randint(1, 256)]),
            "entries": _between(rng, 1, 500000),
            "skew": rng.choice([1.0, 2.0, 5.0]),
            "none": rng.choice([0.0, 0.1]), "dtype": dtype, "train": train}


def _sizes(c):
    """Rows of each example, and queries of each.  They belong to the case, not
    to the seed: a hash of the example's number."""
    n = []
    for b in range(c["examples"]):
        part = ((b * 2654435761 + 12345) % 65536) / 65536.0
        n.append(max(1, int(c["rows"] * (0.1 + 0.9 * part)))
                 if c["ragged"] else c["rows"])
    s = c["queries"]
    return [r if s == 0 else 1 if s == 1 else -(-r // s) for r in n], n


def _longest(c):
    nq, nk = _sizes(c)
    return max(nq), max(nk)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    c["type"] = DTYPES[case["dtype"]]
    return {"attention": _prepare_attention,
            "norm_rotate": _prepare_norm_rotate,
            "lookup": _prepare_lookup}[case["op"]](c, g)


def _normal(g, c, *shape, scale=1.0):
    x = torch.randn(*shape, generator=g, device=DEV) * scale
    return x.to(c["type"])


def _prepare_attention(c, g):
    nq, nk = _sizes(c)
    sizes_q = torch.tensor(nq, device=DEV)
    sizes_k = torch.tensor(nk, device=DEV)
    ids = torch.arange(c["examples"], device=DEV)
    c["batch_q"] = ids.repeat_interleave(sizes_q)
    c["batch_k"] = ids.repeat_interleave(sizes_k)
    c["longest"] = (max(nq), max(nk))
    rows_q, rows_k = sum(nq), sum(nk)
    c["q"] = _normal(g, c, rows_q, c["heads"], c["d"])
    c["k"] = _normal(g, c, rows_k, c["kv_heads"], c["d"])
    c["v"] = _normal(g, c, rows_k, c["kv_heads"], c["d"])
    c["scale"] = c["d"] ** -0.5
    c["pos_q"] = c["pos_k"] = c["slope"] = None
    if c["axes"] == 1:
        # running numbers of the rows of an example, a little jittered
        start = torch.cumsum(sizes_k, 0) - sizes_k
        steps = torch.arange(rows_k, device=DEV) - start[c["batch_k"]]
        pos = steps.float() + 0.25 * torch.rand(rows_k, generator=g,
                                                device=DEV)
        c["pos_k"] = pos.view(-1, 1)
    elif c["axes"] > 1:
        # points of a scene, some metres from the origin
        c["pos_k"] = 5.0 * torch.randn(rows_k, c["axes"], generator=g,
                                       device=DEV) + 20.0
    if c["axes"]:
        s = c["queries"]
        if s == 1:
            first = torch.cumsum(sizes_k, 0) - sizes_k
            c["pos_q"] = c["pos_k"][first].contiguous()
        elif s > 1:
            start = torch.cumsum(sizes_k, 0) - sizes_k
            steps = torch.arange(rows_k, device=DEV) - start[c["batch_k"]]
            c["pos_q"] = c["pos_k"][steps % s == 0].contiguous()
        else:
            c["pos_q"] = c["pos_k"]
        # a falling series over the heads: some look far, some near
        h = torch.arange(1, c["heads"] + 1, device=DEV)
        c["slope"] = 2.0 ** (-8.0 * h / c["heads"])
    if c["train"]:
        c["dout"] = _normal(g, c, rows_q, c["heads"], c["d"])
        for name in ("q", "k", "v"):
            c[name].requires_grad_()
    return c


def _prepare_norm_rotate(c, g):
    n, d = c["rows"], c["d"]
    c["q"] = _normal(g, c, n, c["heads"], d, scale=2.0)
    c["k"] = _normal(g, c, n, c["kv_heads"], d, scale=0.5)
    c["weight_q"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)) \
        .to(c["type"])
    c["weight_k"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)) \
        .to(c["type"])
    # points up to 100 m from the scanner; wave lengths from some metres to
    # centimetres, a third of the pairs to each axis
    c["pos"] = 100.0 * torch.rand(n, c["axes"], generator=g, device=DEV) - 50.0
    r = c["rotated"]
    pair = torch.arange(r, device=DEV)
    waves = 100.0 ** (pair.float() / max(1, r))
    axis = pair % c["axes"]
    c["freq"] = torch.where(axis == torch.arange(c["axes"], device=DEV)[:, None],
                            waves, torch.zeros_like(waves)).contiguous()
    c["eps"] = 1e-6
    if c["train"]:
        c["dq"] = _normal(g, c, n, c["heads"], d)
        c["dk"] = _normal(g, c, n, c["kv_heads"], d)
        for name in ("q", "k", "weight_q", "weight_k"):
            c[name].requires_grad_()
    return c


def _prepare_lookup(c, g):
    c["weight"] = _normal(g, c, c["table"], c["width"])
    # row numbers: evenly spread (skew 1), or the low ones far more often
    u = torch.rand(c["entries"], generator=g, device=DEV, dtype=torch.float64)
    index = (u ** c["skew"] * c["table"]).long().clamp_(max=c["table"] - 1)
    # (scattered, so that neighbours in the table are not close in memory)
    order = torch.randperm(c["table"], generator=g, device=DEV)
    index = order[index]
    if c["none"] > 0:
        gone = torch.rand(c["entries"], generator=g, device=DEV) < c["none"]
        index = torch.where(gone, torch.full_like(index, -1), index)
    c["index"] = index
    c["scale"] = c["width"] ** 0.5
    if c["train"]:
        c["dout"] = _normal(g, c, c["entries"], c["width"])
        c["weight"].requires_grad_()
    return c


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():  # (the gradients are written out)
        return {"attention": _plain_attention,
                "norm_rotate": _plain_norm_rotate,
                "lookup": _plain_lookup}[state["op"]](state)


def _run_own(c):
    import pytorch_cluster_amd as pca
    if c["op"] == "attention":
        out = pca.attention(c["q"], c["k"], c["v"], c["batch_q"],
                            c["batch_k"], pos_q=c["pos_q"], pos_k=c["pos_k"],
                            slope=c["slope"], scale=c["scale"], cap=c["cap"])
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (c["q"], c["k"], c["v"]),
                                         c["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "norm_rotate":
        q, k = pca.norm_rotate(c["q"], c["k"], c["pos"], c["freq"],
                               weight_q=c["weight_q"],
                               weight_k=c["weight_k"], eps=c["eps"])
        if not c["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad(
            (q, k), (c["q"], c["k"], c["weight_q"], c["weight_k"]),
            (c["dq"], c["dk"]))
        return {"q": q, "k": k, "dq": grads[0], "dk": grads[1],
                "dweight_q": grads[2], "dweight_k": grads[3]}
    out = pca.lookup(c["weight"], c["index"], scale=c["scale"])
    if not c["train"]:
        return {"out": out}
    dweight, = torch.autograd.grad(out, c["weight"], c["dout"])
    return {"out": out, "dweight": dweight}


# ---- plain forms ------------------------------------------------------------

def _places(batch, examples, longest):
    """Row number of place p of example b ([examples, longest], the last row
    where there is none) and whether there is one."""
    ids = torch.arange(examples + 1, device=batch.device)
    ptr = torch.bucketize(ids, batch)
    place = torch.arange(longest, device=batch.device)
    there = place < (ptr[1:] - ptr[:-1])[:, None]
    rows = (ptr[:-1, None] + place).clamp_(max=batch.numel() - 1)
    return rows, there


def _padded(x, rows):
    """[N, H, D] -> [examples, H, longest, D] in 32 bits."""
    return x.float()[rows].transpose(1, 2).contiguous()


def _packed(x, there, dtype):
    return x.transpose(1, 2)[there].to(dtype)


def _plain_attention(c):
    lq, lk = c["longest"]
    b, hq, hk, d = c["examples"], c["heads"], c["kv_heads"], c["d"]
    group = hq // hk
    rows_q, there_q = _places(c["batch_q"], b, lq)
    rows_k, there_k = _places(c["batch_k"], b, lk)
    q = _padded(c["q"], rows_q).view(b * hk, group * lq, d)
    k = _padded(c["k"], rows_k).view(b * hk, lk, d)
    v = _padded(c["v"], rows_k).view(b * hk, lk, d)
    t = torch.bmm(q, k.transpose(1, 2).contiguous()) * c["scale"]
    t = t.view(b, hk, group, lq, lk)
    if c["cap"] > 0:
        tanh = torch.tanh(t / c["cap"])
        t = tanh * c["cap"]
    if c["slope"] is not None:
        step = (c["pos_q"][rows_q][:, :, None, :]
                - c["pos_k"][rows_k][:, None, :, :])
        dist = step.square().sum(-1).sqrt()
        t = t - (c["slope"].view(1, hk, group, 1, 1)
                 * dist.view(b, 1, 1, lq, lk))
    t = t.masked_fill(~there_k.view(b, 1, 1, 1, lk), -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(b * hk, group * lq, lk)
    del t
    out = torch.bmm(p, v)
    result = {"out": _packed(out.view(b, hq, lq, d), there_q, c["type"])}
    if not c["train"]:
        return result
    # (rows that are padding get a gradient of zero)
    dout = _padded(c["dout"], rows_q) * there_q.view(b, 1, lq, 1)
    dout = dout.view(b * hk, group * lq, d)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), dout)
    dp = torch.bmm(dout, v.transpose(1, 2).contiguous())
    dt = p * (dp - (dout * out).sum(-1, keepdim=True))
    if c["cap"] > 0:
        dt = dt * (1 - tanh.view(b * hk, group * lq, lk).square())
    dt = dt * c["scale"]
    dq = torch.bmm(dt, k)
    dk = torch.bmm(dt.transpose(1, 2).contiguous(), q)
    result["dq"] = _packed(dq.view(b, hq, lq, d), there_q, c["type"])
    result["dk"] = _packed(dk.view(b, hk, lk, d), there_k, c["type"])
    result["dv"] = _packed(dv.view(b, hk, lk, d), there_k, c["type"])
    return result


def _turn(x, cos, sin, r):
    a, b, rest = x[..., :r], x[..., r:2 * r], x[..., 2 * r:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_norm_rotate(c):
    r = c["rotated"]
    angle = (c["pos"].double()[:, :, None] * c["freq"].double()).sum(1)
    cos = torch.cos(angle).float()[:, None]
    sin = torch.sin(angle).float()[:, None]
    result = {}
    for name in ("q", "k"):
        x, weight = c[name].float(), c["weight_" + name].float()
        inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + c["eps"])
        unit = x * inv
        result[name] = _turn(unit * weight, cos, sin, r).to(c["type"])
        if c["train"]:
            back = _turn(c["d" + name].float(), cos, -sin, r)
            result["dweight_" + name] = (back * unit).sum((0, 1)) \
                .to(c["type"])
            back = back * weight
            back = inv * (back - unit * (back * unit).mean(-1, keepdim=True))
            result["d" + name] = back.to(c["type"])
    return result


def _plain_lookup(c):
    index, weight = c["index"], c["weight"]
    there = index >= 0
    rows = index.clamp(min=0)
    out = weight.float()[rows] * c["scale"] * there[:, None]
    result = {"out": out.to(c["type"])}
    if c["train"]:
        dweight = torch.zeros(weight.shape, device=weight.device)
        dweight.index_add_(0, rows, c["dout"].float() * there[:, None])
        result["dweight"] = (dweight * c["scale"]).to(c["type"])
    return result


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    train = case["train"]
    if case["op"] == "attention":
        nq, nk = _sizes(case)
        pairs = sum(a * b for a, b in zip(nq, nk))
        q = sum(nq) * case["heads"] * case["d"] * size
        kv = 2 * sum(nk) * case["kv_heads"] * case["d"] * size
        ids = 8 * (sum(nq) + sum(nk))
        pos = 4 * case["axes"] * (sum(nq) + sum(nk))
        bytes_ = 2 * q + kv + ids + pos
        if train:  # dout in, dq, dk, dv out
            bytes_ += 2 * q + kv
        return {"bytes": bytes_, "flops": (14 if train else 4) * pairs
                * case["heads"] * case["d"]}
    if case["op"] == "norm_rotate":
        rows = case["rows"] * (case["heads"] + case["kv_heads"])
        values = rows * case["d"]
        bytes_ = 2 * values * size + 4 * case["axes"] * case["rows"]
        if train:  # dout in, dx out
            bytes_ += 2 * values * size
        return {"bytes": bytes_, "flops": (22 if train else 8) * values}
    e, n, w = case["entries"], case["table"], case["width"]
    bytes_ = 8 * e + (e + min(e, n)) * w * size
    if train:  # dout in, the table's gradient out
        bytes_ += (e + n) * w * size
    return {"bytes": bytes_, "flops": (2 if train else 1) * e * w}


# ---- the definitions, in 64 bits -----------------------------------------------

def exact(case, seed):
    c = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention,
                "norm_rotate": _exact_norm_rotate,
                "lookup": _exact_lookup}[c["op"]](c)


def _exact_attention(c):
    q, k, v = (c[n].detach().double() for n in ("q", "k", "v"))
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    nq, nk = _sizes(c)
    at_q = at_k = 0
    for a, b in zip(nq, nk):
        iq, ik = slice(at_q, at_q + a), slice(at_k, at_k + b)
        at_q, at_k = at_q + a, at_k + b
        if c["slope"] is not None:
            dist = torch.zeros(a, b, dtype=torch.float64, device=DEV)
            for axis in range(c["axes"]):
                dist += (c["pos_q"][iq, axis].double()[:, None]
                         - c["pos_k"][ik, axis].double()[None]) ** 2
            dist = dist.sqrt()
        # all heads of a few, one by one where they would be large
        step = max(1, min(c["kv_heads"], (1 << 28) // (a * b * group)))
        for h in range(0, c["kv_heads"], step):
            hk = slice(h, min(h + step, c["kv_heads"]))
            hq = slice(hk.start * group, hk.stop * group)
            qs = q[iq, hq].permute(1, 0, 2)
            ks = k[ik, hk].permute(1, 0, 2).repeat_interleave(group, 0)
            vs = v[ik, hk].permute(1, 0, 2).repeat_interleave(group, 0)
            s = qs @ ks.mT * c["scale"]
            slopes = 1.0
            if c["cap"] > 0:
                flat = torch.tanh(s / c["cap"])
                s, slopes = c["cap"] * flat, 1 - flat ** 2
            if c["slope"] is not None:
                s = s - c["slope"][hq].double()[:, None, None] * dist
            p = torch.softmax(s, -1)
            o = p @ vs
            out[iq, hq] = o.permute(1, 0, 2)
            if c["train"]:
                do = c["dout"][iq, hq].double().permute(1, 0, 2)
                gain = do @ vs.mT
                ds = p * (gain - (p * gain).sum(-1, keepdim=True)) * slopes
                dq[iq, hq] = c["scale"] * (ds @ ks).permute(1, 0, 2)
                per_head = (-1, group, b, c["d"])
                dk[ik, hk] = (c["scale"] * (ds.mT @ qs)).view(per_head) \
                    .sum(1).permute(1, 0, 2)
                dv[ik, hk] = (p.mT @ do).view(per_head).sum(1) \
                    .permute(1, 0, 2)
    if not c["train"]:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_norm_rotate(c):
    r = c["rotated"]
    angle = c["pos"].double() @ c["freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    result = {}
    for name in ("q", "k"):
        x = c[name].detach().double()
        weight = c["weight_" + name].detach().double()
        size = (x.pow(2).sum(-1, keepdim=True) / c["d"] + c["eps"]).sqrt()
        y = x / size * weight
        z = torch.complex(y[..., :r], y[..., r:2 * r]) * turn
        result[name] = torch.cat([z.real, z.imag, y[..., 2 * r:]], -1)
        if c["train"]:
            g = c["d" + name].double()
            z = torch.complex(g[..., :r], g[..., r:2 * r]) * turn.conj()
            g = torch.cat([z.real, z.imag, g[..., 2 * r:]], -1)
            result["dweight_" + name] = (g * x / size).flatten(0, 1).sum(0)
            g = g * weight
            along = (g * x).sum(-1, keepdim=True) / (c["d"] * size ** 2)
            result["d" + name] = (g - x * along) / size
    return result


def _exact_lookup(c):
    index = c["index"]
    there = index >= 0
    weight = c["weight"].detach().double()
    out = torch.zeros(index.numel(), c["width"], dtype=torch.float64,
                      device=DEV)
    out[there] = c["scale"] * weight[index[there]]
    if not c["train"]:
        return {"out": out}
    dweight = torch.zeros_like(weight)
    dweight.index_add_(0, index[there], c["dout"][there].double())
    return {"out": out, "dweight": c["scale"] * dweight}
