"""Window-and-sinks and shared-prefix attention in 64 bits, straight from the definition, with bounds for a kernel's error.

The bounds count roundings.  u = 2^-24 is fp32's half step, e the half step of the operands' type (finfo.eps / 2).
  * A score is a dot product of dim terms in fp32: off by at most ds = (dim + 4) u scale sum |q_d k_d|; so a softmax weight is off by a
    relative c = 2 max ds + (keys + 32) u (its own exponential and the sum's, additions in any order, a few steps of exp2).
  * A kernel may round a weight, or a score's gradient, once to the operands' type before it multiplies: w = e, 0 in fp32.
  * A result is rounded once to the operands' type: e |result|.
  * Numbers below the smallest normal one have a step of their own: every rounded weight, score's gradient and result may be off by
    a besides, half of fp16's subnormal step 2^-24, or 2^-126 where fp32's range ends (bf16 has the same; such numbers may
    be flushed to zero).  The largest weight of a row is 1 before the division, so a is not enlarged by it.
"""
import torch


def visible(nq, nk, window, sinks, device):
    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None, :]
    return (j <= p) & ((p - j < window) | (j < sinks))


def softmax(s, seen):
    s = s.masked_fill(~seen, -float("inf"))
    top = s.amax(-1, keepdim=True)
    x = torch.exp(s - torch.where(top == -float("inf"), torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    return x / torch.where(total == 0, torch.ones_like(total), total)


def one_sequence(q, k, v, seen, scale, dout=None):
    """q [nq, heads, dim], k, v [nk, kv_heads, dim] of a call's type, seen [nq, nk]: {name: (value, bound)} in 64 bits."""
    u = 2.0 ** -24
    e = torch.finfo(q.dtype).eps / 2
    w = 0.0 if q.dtype == torch.float32 else e
    a = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -126
    nq, heads, dim = q.shape
    nk, kv_heads, _ = k.shape
    group = heads // kv_heads
    if nq == 0 or nk == 0:
        zq, zk = torch.zeros(nq, heads, dim, dtype=torch.float64, device=q.device), torch.zeros(nk, kv_heads, dim, dtype=torch.float64, device=q.device)
        out = {"out": (zq, zq)}
        if dout is not None:
            out.update(dq=(zq, zq), dk=(zk, zk), dv=(zk, zk))
        return out
    Q = q.double().transpose(0, 1)                                          # [heads, nq, dim]
    K = k.double().transpose(0, 1).repeat_interleave(group, 0)
    V = v.double().transpose(0, 1).repeat_interleave(group, 0)
    P = softmax(Q @ K.transpose(1, 2) * scale, seen)
    ds = (dim + 4) * u * abs(scale) * (Q.abs() @ K.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    c = 2 * ds + (nk + 32) * u                                              # [heads, nq, 1]
    O = P @ V
    out_tol = e * O.abs() + (w + c) * (P @ V.abs()) + a * (seen.double() @ V.abs()) + a
    back = lambda x: x.transpose(0, 1)
    res = {"out": (back(O), back(out_tol))}
    if dout is None:
        return res
    G = dout.double().transpose(0, 1)
    dP = G @ V.transpose(1, 2)
    delta = (G * O).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    # delta is taken from the rounded result; dP and delta are fp32 sums of dim terms
    off = (G.abs() * out_tol).sum(-1, keepdim=True) + (dim + 4) * u * (G.abs() * O.abs()).sum(-1, keepdim=True)
    dS_off = P * ((w + c + 4 * u) * (dP - delta).abs() + off + (dim + 4) * u * (G.abs() @ V.abs().transpose(1, 2)))
    dS_off = dS_off + a * seen * ((dP - delta).abs() + 1)
    terms = (nk + nq * group + 32) * u
    per_head = lambda x: back(x.reshape(kv_heads, group, nk, dim).sum(1))
    dQ, dK, dV = scale * (dS @ K), per_head(scale * (dS.transpose(1, 2) @ Q)), per_head(P.transpose(1, 2) @ G)
    s = abs(scale)
    tq = a + e * dQ.abs() + s * (dS_off @ K.abs()) + terms * s * (dS.abs() @ K.abs())
    tk = a + e * dK.abs() + s * per_head(dS_off.transpose(1, 2) @ Q.abs()) + terms * s * per_head(dS.abs().transpose(1, 2) @ Q.abs())
    tv = a + e * dV.abs() + per_head(((w + c) * P + a * seen).transpose(1, 2) @ G.abs()) + terms * per_head(P.transpose(1, 2) @ G.abs())
    res.update(dq=(back(dQ), back(tq)), dk=(dK, tk), dv=(dV, tv))
    return res


def packed(q, k, v, q_lens, k_lens, window, sinks, scale, dout=None, q_start=0, k_start=0):
    """All sequences; rows of none are zero with a bound of zero."""
    names = {"out": q, "dq": q, "dk": k, "dv": k}
    if dout is None:
        names = {"out": q}
    res = {n: (torch.zeros(x.shape, dtype=torch.float64, device=q.device), torch.zeros(x.shape, dtype=torch.float64, device=q.device)) for n, x in names.items()}
    a, b = q_start, k_start
    for nq, nk in zip(q_lens, k_lens):
        one = one_sequence(q[a:a + nq], k[b:b + nk], v[b:b + nk], visible(nq, nk, window, sinks, q.device), scale,
                           None if dout is None else dout[a:a + nq])
        for n, (x, t) in one.items():
            at = slice(a, a + nq) if n in ("out", "dq") else slice(b, b + nk)
            res[n][0][at], res[n][1][at] = x, t
        a, b = a + nq, b + nk
    return res


def check(got, want, name=""):
    value, bound = want
    assert got.shape == value.shape
    err = (got.double() - value).abs()
    bad = ~(err <= bound)
    if bool(bad.any()):
        worst = (err / (bound + 1e-300)).nan_to_num(float("inf")).masked_fill(~bad, 0.0).argmax()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, worst at {worst.item()} of {list(got.shape)}: "
                             f"{got.flatten()[worst].item()!r}, not {value.flatten()[worst].item()!r} +- {bound.flatten()[worst].item()!r}")
