"""attention in 64 bits with bounds that go by the scores, whatever the cap is
(imported by the tests of large caps, long tails, many rows and cut sides).

To first order, U half a step of the element type, E = 2^-24 that of fp32:

* product of d pairs, scale, unit of the exponent: (d + 6) E scale |q| |k|;
* a cap up to 128 with 16-bit rows: 12 roundings of numbers of the cap's size;
* any other cap: below tanh(0.35) the series: 10 roundings of the score and 2e-8 of it.
  Beyond, 1 - 2 w with w = 1 / (exp2(x) + 1) < 1/3: exp2 and what goes into x 10 E x
  2 w (1 - w) < 5 E, the sum and the reciprocal 3 E x 2 w < 2 E, the difference E; of a
  tanh of at least 0.336 that is 24 E; two products more: 26 E.  With a cap of 2^127 (a
  larger one is taken for it) scores are fractions of it below the smallest normal
  number, in steps of 2^-149: two roundings of half a step, one of them halved again by
  0.35, times 2^127 are 3 E;
* bias: differences, squares, root, product: 10 E of it;
* exponent and exponential: 4 E of the score and 4 E;
* a weight: twice what its exponent and those of the sum are off, U for its rounding;
  the exponential gives 0 in place of anything below 2^-126, the smallest normal number,
  and so does the matrix instruction with what it takes and gives.
"""
import torch

from features_common import E, half_step, rounded, spans

TINY = 2.0 ** -126


def tail(dtype):
    """Of the largest weight of a row: what rounding a weight may take off one
    that is too small for fp16."""
    return 2.0 ** -32 if dtype == torch.float16 else 0.0


def attention_bounds(q, k, v, batch_q=None, batch_k=None, pos_q=None,
                     pos_k=None, slope=None, scale=None, cap=0.0, dout=None,
                     exact_weights=False, rest=True):
    """(values, bounds): dicts of out (and dq, dk, dv).  exact_weights: the inputs
    are such that all weights of a row are powers of two, which no rounding
    changes.  rest: the backward pass has what rounding took off out."""
    dtype, e = q.dtype, E
    u = half_step(dtype) if dtype != torch.float32 else 0.0
    group, d = q.size(1) // k.size(1), q.size(2)
    scale = d ** -0.5 if scale is None else scale
    q64, k64, v64 = q.double(), k.double(), v.double()
    like = {"out": q64}
    if dout is not None:
        like.update(dq=q64, dk=k64, dv=v64)
    val = {n: torch.zeros_like(x) for n, x in like.items()}
    err = {n: torch.zeros_like(x) for n, x in like.items()}
    low = 0.0 if exact_weights else tail(dtype)
    for sq, sk in spans(batch_q, batch_k, q.size(0), k.size(0)):
        a, b = sq.stop - sq.start, sk.stop - sk.start
        if a == 0 or b == 0:
            continue
        qs = q64[sq].transpose(0, 1).contiguous()
        ks = k64[sk].transpose(0, 1).repeat_interleave(group, 0).contiguous()
        vs = v64[sk].transpose(0, 1).repeat_interleave(group, 0).contiguous()
        kt, vt = ks.mT.contiguous(), vs.mT.contiguous()
        s = qs @ kt * scale
        product = (d + 6) * e * abs(scale) * (qs.abs() @ kt.abs())
        wrong, flat, curve = product, torch.ones_like(s), 0.0
        if cap > 0:
            tanh = torch.tanh(s / cap)
            s = cap * tanh
            flat = 1 - tanh ** 2
            if dtype != torch.float32 and cap <= 128:
                wrong = wrong + 12 * e * cap
                curve = 12 * e
            else:
                wrong = wrong + 26 * e * s.abs()
                if cap > 1e36:
                    wrong = wrong + 3 * e
                curve = 2 * e + 52 * e * tanh ** 2
            # (flat moves by 2 tanh flat / cap with the product)
            curve = curve + 2 * tanh.abs() * flat * product / cap
        if slope is not None:
            step = pos_q[sq].double()[:, None] - pos_k[sk].double()[None]
            bias = slope.double()[:, None, None] * step.square().sum(-1).sqrt()
            s = s - bias
            wrong = wrong + 10 * e * bias.abs()
        wrong = wrong + 4 * e * s.abs() + 4 * e
        if exact_weights:
            wrong = torch.zeros_like(wrong)
        p = torch.softmax(s, -1)
        off = wrong + (wrong * p).sum(-1, keepdim=True) + (b + 20) * e
        pu = p * (2 * off + (0.0 if exact_weights else u)) + TINY
        o = p @ vs
        most = p.amax(-1, keepdim=True)
        oe = pu @ vs.abs() + low * most * vs.abs().sum(1, keepdim=True) \
            + (b + 8) * e * (p @ vs.abs())
        val["out"][sq] = o.transpose(0, 1)
        err["out"][sq] = (oe + rounded(o, dtype)).transpose(0, 1)
        if dout is None:
            continue
        do = dout[sq].double().transpose(0, 1).contiguous()
        gain = do @ vt
        delta = (p * gain).sum(-1, keepdim=True)
        ds = p * (gain - delta) * flat
        left = rounded(o, dtype)
        if rest and u:  # (rounded a second time)
            left = rounded(left, dtype)
        ge = (d + 4) * e * (do.abs() @ vt.abs())
        de = (do.abs() * (oe + left)).sum(-1, keepdim=True) \
            + (2 * d + 4) * e * (do.abs() * o.abs()).sum(-1, keepdim=True)
        less = (gain - delta).abs()
        xe = ds.abs() * (2 * off + u) + p * less * curve + TINY * (1 + less) \
            + p * (ge + de + 4 * e * (gain.abs() + delta.abs()))
        if dtype == torch.float16:  # (values far below the largest of a step)
            xe = xe + 2.0 ** -36 * ds.abs().amax((1, 2), keepdim=True)
        many = (max(a * group, b) + 8) * e
        dq = scale * (ds @ ks)
        dqe = abs(scale) * (xe @ ks.abs() + many * (ds.abs() @ ks.abs()))
        val["dq"][sq] = dq.transpose(0, 1)
        err["dq"][sq] = (dqe + rounded(dq, dtype) + TINY).transpose(0, 1)

        def fold(x):
            return x.view(-1, group, b, d).sum(1).transpose(0, 1)
        dst, pt = ds.mT.contiguous(), p.mT.contiguous()
        xet, put = xe.mT.contiguous(), pu.mT.contiguous()
        val["dk"][sk] = fold(scale * (dst @ qs))
        val["dv"][sk] = fold(pt @ do)
        dke = fold(abs(scale) * (xet @ qs.abs()
                                 + many * (dst.abs() @ qs.abs())))
        # (weights go to fp16 times 2^14: what is lost below 2^-39)
        low_v = 2.0 ** -39 if dtype == torch.float16 else 0.0
        dve = fold(put @ do.abs() + many * (pt @ do.abs())
                   + low_v * do.abs().sum(1, keepdim=True))
        err["dk"][sk] = dke + rounded(val["dk"][sk], dtype) + TINY
        err["dv"][sk] = dve + rounded(val["dv"][sk], dtype) + TINY
    return val, err
