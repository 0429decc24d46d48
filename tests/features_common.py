"""Definitions of attention, norm_rotate and lookup in 64 bits, with the bounds
that their tests hold the kernels to (imported only by those tests).

A rounding to a type is off by at most half a step, ``finfo.eps / 2`` of the
value (below the smallest normal number: of that).  U is that of the element
type, E = 2^-24 that of fp32.  Every bound is the sum of what the roundings of
the method can do to first order, doubled where second orders could show.
"""
import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(x, dtype):
    """What rounding the result to `dtype` may add."""
    info = torch.finfo(dtype)
    return half_step(dtype) * (x.abs() + info.smallest_normal)


def spans(batch_q, batch_k, nq, nk):
    if batch_q is None:
        return [(slice(0, nq), slice(0, nk))]
    ids = torch.unique(torch.cat([batch_q, batch_k])).tolist()
    out = []
    for b in ids:
        q = (batch_q == b).nonzero().view(-1)
        k = (batch_k == b).nonzero().view(-1)
        out.append((slice(int(q[0]), int(q[-1]) + 1) if len(q) else slice(0, 0),
                    slice(int(k[0]), int(k[-1]) + 1) if len(k) else slice(0, 0)))
    return out


def attention64(q, k, v, batch_q=None, batch_k=None, pos_q=None, pos_k=None,
                slope=None, scale=None, cap=0.0, dout=None):
    """(values, bounds): dicts of out (and dq, dk, dv)."""
    dtype = q.dtype
    u, e = half_step(dtype), E
    group = q.size(1) // k.size(1)
    d = q.size(2)
    scale = d ** -0.5 if scale is None else scale
    q64, k64, v64 = q.double(), k.double(), v.double()
    names = ["out"] + ([] if dout is None else ["dq", "dk", "dv"])
    like = {"out": q64, "dq": q64, "dk": k64, "dv": v64}
    val = {n: torch.zeros_like(like[n]) for n in names}
    err = {n: torch.zeros_like(like[n]) for n in names}
    for sq, sk in spans(batch_q, batch_k, q.size(0), k.size(0)):
        a, b = sq.stop - sq.start, sk.stop - sk.start
        if a == 0 or b == 0:
            continue
        qs = q64[sq].transpose(0, 1)
        ks = k64[sk].transpose(0, 1).repeat_interleave(group, 0).contiguous()
        vs = v64[sk].transpose(0, 1).repeat_interleave(group, 0).contiguous()
        kt, vt = ks.mT.contiguous(), vs.mT.contiguous()
        t = qs @ kt * scale
        # products: d rounded additions, scale and unit of the exponent
        wrong = (d + 6) * e * abs(scale) * (qs.abs() @ kt.abs())
        flat = torch.ones_like(t)
        s = t
        if cap > 0:
            tanh = torch.tanh(t / cap)
            s = cap * tanh
            flat = 1 - tanh ** 2
            # (1 - 2 / (exp2 + 1): six roundings of numbers up to 2)
            wrong = wrong + 12 * e * cap
        if slope is not None:
            dist = (pos_q[sq].double()[:, None] - pos_k[sk].double()[None]) \
                .square().sum(-1).sqrt()
            bias = slope.double()[:, None, None] * dist
            s = s - bias
            # differences, three squares, root (2), product
            wrong = wrong + 10 * e * bias.abs()
        # the score itself, minus the maximum, exp2 (2 steps)
        wrong = wrong + 4 * e * s.abs() + 4 * e
        p = torch.softmax(s, -1)
        # a weight's relative error: its own, its sum's (b additions), rounding
        # for the product; fp16 has no weights below 2^-25 of the largest
        low = 2.0 ** -25 if dtype == torch.float16 else 0.0
        off = wrong + (wrong * p).sum(-1, keepdim=True) + (b + 20) * e
        pu = p * (2 * off + (u if dtype != torch.float32 else 0))
        o = p @ vs
        oe = pu @ vs.abs() + low * vs.abs().sum(1, keepdim=True) \
            + (b + 8) * e * (p @ vs.abs())
        val["out"][sq] = o.transpose(0, 1)
        err["out"][sq] = (oe + rounded(o, dtype)).transpose(0, 1)
        if dout is None:
            continue
        do = dout[sq].double().transpose(0, 1)
        gain = do @ vt
        delta = (p * gain).sum(-1, keepdim=True)
        ds = p * (gain - delta) * flat
        # delta comes from the rounded output
        ge = (d + 4) * e * (do.abs() @ vt.abs())
        de = (do.abs() * (oe + rounded(o, dtype))).sum(-1, keepdim=True) \
            + (d + 4) * e * (do.abs() * o.abs()).sum(-1, keepdim=True)
        xe = ds.abs() * (2 * off + (u if dtype != torch.float32 else 0)) \
            + p * (ge + de + 4 * e * (gain.abs() + delta.abs()))
        if cap > 0:
            xe = xe + 2 * p * (gain - delta).abs() * (
                12 * e + 2 * (d + 6) * e * abs(scale) / cap
                * (qs.abs() @ kt.abs()))
        if dtype == torch.float16:  # (values far below the largest of a step)
            xe = xe + 2.0 ** -36 * ds.abs().amax((1, 2), keepdim=True)
        many = (max(a * group, b) + 8) * e
        dq = scale * (ds @ ks)
        dqe = abs(scale) * (xe @ ks.abs() + many * (ds.abs() @ ks.abs()))
        val["dq"][sq] = dq.transpose(0, 1)
        err["dq"][sq] = (dqe + rounded(dq, dtype)).transpose(0, 1)

        def fold(x):
            return x.view(-1, group, b, d).sum(1).transpose(0, 1)
        dst, pt = ds.mT.contiguous(), p.mT.contiguous()
        xet, put = xe.mT.contiguous(), pu.mT.contiguous()
        dk = fold(scale * (dst @ qs))
        dke = fold(abs(scale) * (xet @ qs.abs()
                                 + many * (dst.abs() @ qs.abs())))
        dv = fold(pt @ do)
        dve = fold(put @ do.abs() + many * (pt @ do.abs())
                   + low * 2.0 ** -14 * do.abs().sum(1, keepdim=True))
        val["dk"][sk], val["dv"][sk] = dk, dv
        err["dk"][sk] = dke + rounded(dk, dtype)
        err["dv"][sk] = dve + rounded(dv, dtype)
    return val, err


def turn64(x, angle, back=False):
    r = angle.size(1)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    if back:
        sin = -sin
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * r:]], -1)


def norm_rotate64(x, pos, freq, weight=None, eps=1e-6, dout=None):
    """(values, bounds): dicts of out (and dx, dweight)."""
    dtype, e, d = x.dtype, E, x.size(2)
    x64 = x.double()
    w = torch.ones(d, dtype=torch.float64, device=x.device) \
        if weight is None else weight.double()
    r = freq.size(1)
    angle = pos.double() @ freq.double()
    size = (x64.square().mean(-1, keepdim=True) + eps).sqrt()
    unit = x64 / size
    y = unit * w
    out = turn64(y, angle)
    # a norm of d squares: d + 6 roundings; weight, cos and sin (2 each), the
    # products and their sum
    many = (d + 16) * e

    def pairs(z):
        z = z.abs()
        other = torch.cat([z[..., r:2 * r], z[..., :r],
                           torch.zeros_like(z[..., 2 * r:])], -1)
        return z + other
    val = {"out": out}
    err = {"out": 2 * many * pairs(y) + rounded(out, dtype)}
    if dout is None:
        return val, err
    g = turn64(dout.double(), angle, back=True)
    ge = 8 * e * pairs(dout.double())
    val["dweight"] = (g * unit).sum((0, 1))
    rows = x.size(0) * x.size(1)
    # (rows of a workgroup one after the other, at least: 1,024 of them)
    chain = rows / 1024 + 1024 + 64
    err["dweight"] = ((ge + 2 * many * g.abs()) * unit.abs()
                      + chain * e * (g * unit).abs()).sum((0, 1))
    if weight is not None:
        err["dweight"] = err["dweight"] + rounded(val["dweight"], weight.dtype)
    g, ge = g * w, ge * w.abs()
    dot = (g * unit).mean(-1, keepdim=True)
    dx = (g - unit * dot) / size
    de = ((ge + 2 * many * g.abs()) * unit.abs()).mean(-1, keepdim=True) \
        + (d + 8) * e * (g * unit).abs().mean(-1, keepdim=True)
    val["dx"] = dx
    err["dx"] = (ge + many * g.abs() + unit.abs() * (de + 2 * many * dot.abs())
                 + 2 * many * (g.abs() + (unit * dot).abs())) / size \
        + rounded(dx, dtype)
    return val, err


def lookup64(weight, index, scale, dout=None):
    flat = index.reshape(-1)
    n = weight.size(0)
    there = (flat >= 0) & (flat < n)
    rows = flat[there].long()
    w64 = weight.double()
    out = torch.zeros(flat.numel(), weight.size(1), dtype=torch.float64,
                      device=weight.device)
    out[there] = scale * w64[rows]
    val = {"out": out.view(*index.shape, weight.size(1))}
    # (scale itself goes to fp32, then one product)
    err = {"out": 2 * E * val["out"].abs() + rounded(val["out"], weight.dtype)}
    if dout is not None:
        # (on the host: many entries of one row are slow to add on the device)
        g = dout.reshape(flat.numel(), -1).double()[there].cpu()
        grad = torch.zeros(w64.shape, dtype=torch.float64)
        size = torch.zeros_like(grad)
        grad.index_add_(0, rows.cpu(), g)
        size.index_add_(0, rows.cpu(), g.abs())
        grad, size = grad.to(weight.device), size.to(weight.device)
        many = torch.bincount(rows, minlength=n).double()[:, None] + 8
        val["dweight"] = scale * grad
        err["dweight"] = abs(scale) * many * E * size \
            + rounded(val["dweight"], weight.dtype)
    return val, err


def check(got, val, err, what=""):
    """Every value within its bound; prints how much of it was used."""
    for name, x in got.items():
        x = x.detach().double()
        assert x.shape == val[name].shape, (what, name, x.shape)
        assert torch.isfinite(x).all(), (what, name, "not finite")
        diff = (x - val[name]).abs()
        ratio = (diff / err[name].clamp(min=1e-300)).max().item() \
            if x.numel() else 0.0
        assert ratio <= 1.0, (what, name, "%.3g of its bound" % ratio,
                              diff.max().item())
