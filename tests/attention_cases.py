"""The two attentions over series written out in 64 bits, dense, on the CPU, with bounds on what the kernels'
roundings may add up to.

u is half a step of the row type relative to a value (2^-8 for bfloat16, 2^-24 for float32): every
result is rounded to it once, and where a product's operand is (softmax weights, decayed scores, states, dS),
each term of that product is off by u of itself at most.  Sums of m terms in 32 bits are off by m 2^-24 of the
sum of their magnitudes at most."""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gamma(m):
    return m * E32


def series_of(n, offsets):
    """(series id or -1, place in the series) of each row."""
    sid = torch.full((n,), -1, dtype=torch.int64)
    pos = torch.zeros(n, dtype=torch.int64)
    for s in range(len(offsets) - 1):
        a, b = offsets[s], offsets[s + 1]
        sid[a:b] = s
        pos[a:b] = torch.arange(b - a)
    return sid, pos


def window_mask(n, offsets, window, sinks):
    sid, pos = series_of(n, offsets)
    same = (sid[:, None] == sid[None, :]) & (sid[:, None] >= 0)
    return same & (pos[None, :] <= pos[:, None]) & ((pos[None, :] > pos[:, None] - window) | (pos[None, :] < sinks))


def window_reference(q, k, v, dout, offsets, window, sinks, scale):
    """{name: (value, bound)} of out, lse, dq, dk, dv; rows of no series are zeros (lse -inf)."""
    dtype, n = q.dtype, q.shape[0]
    u = half_step(dtype)
    heads, kv = q.shape[1], k.shape[1]
    g = heads // kv
    mask = window_mask(n, offsets, window, sinks)
    live = mask.any(1)
    # what no series holds is not read: rows of no series may hold anything
    Q, K, V, DO = (torch.where(live[:, None, None], x.double(), 0.0).transpose(0, 1) for x in (q, k, v, dout))
    K, V = K.repeat_interleave(g, 0), V.repeat_interleave(g, 0)
    dk, seen = q.shape[2], int(mask.sum(1).max()) if n else 0
    S = (Q @ K.transpose(1, 2)) * scale
    S = torch.where(mask, S, -math.inf)
    top = torch.where(live, S.amax(2), 0.0)
    ex = torch.exp(S - top[..., None])
    l = torch.where(live, ex.sum(2), 1.0)
    P = ex / l[..., None]
    lse = torch.where(live, top + torch.log(l), -math.inf)
    absS = torch.where(mask, (Q.abs() @ K.abs().transpose(1, 2)) * scale, 0.0).amax(2)
    # a score is off by its sum's error, its exponent's rounding and the base change; a weight by e times that,
    # and by two steps of the exponential
    relP = 2 * (gamma(dk + 8) * absS + 4 * E32 * absS) + 8 * E32
    relP = (relP + gamma(seen))[..., None]
    O = P @ V
    A = P @ V.abs()
    out = {"out": (O, u * O.abs() + (u + relP + gamma(seen)) * A), "lse": (lse, relP[..., 0] + 8 * E32 * top.abs() + 1e-6)}
    dP = DO @ V.transpose(1, 2)
    delta = (DO * O).sum(2, keepdim=True)
    dS = torch.where(mask, P * (dP - delta), 0.0)
    # do.o uses the rounded out; dP and do.o are sums of dim_v terms
    eD = (DO.abs() * out["out"][1]).sum(2, keepdim=True) + gamma(v.shape[2] + 4) * (DO.abs() * O.abs()).sum(2, keepdim=True)
    edP = gamma(v.shape[2] + 4) * (DO.abs() @ V.abs().transpose(1, 2))
    eS = torch.where(mask, P * (edP + eD) + dS.abs() * (u + relP + 4 * E32), 0.0)
    eP = P * (u + relP)
    dq, bq = dS @ K * scale, (eS + gamma(seen) * dS.abs()) @ K.abs() * scale
    m = gamma(int(mask.sum(0).max()) * g if n else 0)
    dkh, bk = dS.transpose(1, 2) @ Q * scale, (eS + m * dS.abs()).transpose(1, 2) @ Q.abs() * scale
    dvh, bv = P.transpose(1, 2) @ DO, (eP + m * P).transpose(1, 2) @ DO.abs()
    fold = lambda x: x.reshape(kv, g, n, -1).sum(1)  # noqa: E731
    dkh, bk, dvh, bv = (fold(x) for x in (dkh, bk, dvh, bv))
    for name, x, b in (("dq", dq, bq), ("dk", dkh, bk), ("dv", dvh, bv)):
        out[name] = (x, 1.01 * b + u * x.abs())
    done = {}
    for name, (x, b) in out.items():
        x, b = (x.transpose(0, 1), b.transpose(0, 1))
        done[name] = (x, b + 1e-30)
    return done


def decay_reference(q, k, v, log_decay, offsets, scale, state=None, dout=None, dstate=None):
    """{name: (value, bound)} of out, state, and with dout dq, dk, dv, dstate, by the definition row by row pair."""
    dtype, n = q.dtype, q.shape[0]
    u = half_step(dtype)
    sid, pos = series_of(n, offsets)
    live = sid >= 0
    ns = len(offsets) - 1
    zero = lambda x: torch.where(live[:, None, None], x.double(), 0.0).transpose(0, 1)  # noqa: E731
    Q, K, V = zero(q), zero(k), zero(v)
    h, dk, dv = Q.shape[0], q.shape[2], v.shape[2]
    ld = log_decay.double()

    def power(m):  # [h, ...] lambda^m, 0^0 = 1
        m = m.double()
        x = ld.reshape(-1, *([1] * m.dim())) * m
        return torch.where(m == 0, 1.0, torch.exp(torch.where(m == 0, 0.0, x)))

    same = (sid[:, None] == sid[None, :]) & live[:, None] & (pos[None, :] <= pos[:, None])
    gap = (pos[:, None] - pos[None, :]).clamp(min=0)
    W = torch.where(same, power(gap), 0.0)
    lens = torch.tensor([offsets[s + 1] - offsets[s] for s in range(ns)])
    longest = int(lens.max()) if ns else 0
    # a power of lambda is off by the rounding of its exponent (at most |log2 lambda^m| 2^-23, beyond 2^-126 nothing is left)
    eW = 8 * E32 + 90 * 2 ** -22 * (ld < 0).double()[:, None, None]
    # bfloat16: decayed scores or states are rounded once (u), the terms of a state to 2^-17 of themselves
    term = u + 2.0 ** -17 if dtype != torch.float32 else 2 * E32
    S0 = torch.zeros(ns, h, dk, dv, dtype=torch.float64) if state is None else state.double()
    into = torch.where(live[None], power(pos + 1), 0.0)[..., None]

    def through(A, B, C, W):  # sum_j W_ij (a_i.b_j) c_j, and the same of magnitudes
        return (A @ B.transpose(1, 2) * W) @ C, (A.abs() @ B.abs().transpose(1, 2) * W) @ C.abs()

    def past(A, S):  # a_i S_series
        out = torch.zeros(h, n, S.shape[3], dtype=torch.float64)
        for s in range(ns):
            a, b = offsets[s], offsets[s + 1]
            out[:, a:b] = A[:, a:b] @ S[s]
        return out

    def make(x, b, by):
        err = term + eW + gamma(longest + max(dk, dv) + 8)
        return (x * by, (u * x.abs() + 1.01 * err * b) * by)

    def rows(pair):
        return pair[0].transpose(0, 1), pair[1].transpose(0, 1) + 1e-30

    o, ob = through(Q, K, V, W)
    o, ob = o + into * past(Q, S0), ob + into * past(Q.abs(), S0.abs())
    res = {"out": rows(make(o, ob, scale))}
    last, lb = torch.zeros_like(S0), torch.zeros_like(S0)
    for s in range(ns):
        a, b = offsets[s], offsets[s + 1]
        w = power(lens[s] - 1 - pos[a:b])[..., None] if b > a else torch.zeros(h, 0, 1, dtype=torch.float64)
        f = power(lens[s])[:, None, None]
        last[s] = (K[:, a:b] * w).transpose(1, 2) @ V[:, a:b] + f * S0[s]
        lb[s] = (K[:, a:b] * w).abs().transpose(1, 2) @ V[:, a:b].abs() + f * S0[s].abs()
    fine = 2.0 ** -24 + eW.reshape(1, h, 1, 1) + gamma(longest + 8)
    res["state"] = (last, fine * lb + 1e-30)
    if dout is None:
        return res
    DO = zero(dout)
    DS = torch.zeros_like(S0) if dstate is None else dstate.double()
    tail = torch.where(live[None], power(torch.where(live, lens[sid.clamp(min=0)] - 1 - pos, 0)), 0.0)[..., None]
    T = lambda S: S.transpose(2, 3)  # noqa: E731
    x, b = through(DO, V, K, W)
    x, b = x + into * past(DO, T(S0)), b + into * past(DO.abs(), T(S0).abs())
    res["dq"] = rows(make(x, b, scale))
    Wt = W.transpose(1, 2)
    x, b = through(V, DO, Q, Wt)
    x, b = x * scale + tail * past(V, T(DS)), b * scale + tail * past(V.abs(), T(DS).abs())
    res["dk"] = rows(make(x, b, 1.0))
    x, b = through(K, Q, DO, Wt)
    x, b = x * scale + tail * past(K, DS), b * scale + tail * past(K.abs(), DS.abs())
    res["dv"] = rows(make(x, b, 1.0))
    d0, d0b = torch.zeros_like(S0), torch.zeros_like(S0)
    for s in range(ns):
        a, b = offsets[s], offsets[s + 1]
        f = power(lens[s])[:, None, None]
        d0[s] = scale * (Q[:, a:b] * into[:, a:b]).transpose(1, 2) @ DO[:, a:b] + f * DS[s]
        d0b[s] = scale * (Q[:, a:b] * into[:, a:b]).abs().transpose(1, 2) @ DO[:, a:b].abs() + f * DS[s].abs()
    # where the state itself is not returned its terms enter to 2^-18; with it to 2^-27
    res["dstate"] = (d0, fine * d0b + 1e-30)
    return res


def check(name, got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)}, expected {tuple(want.shape)}"
    same = (got == want) | ((got - want).abs() <= bound)
    if not bool(same.all()):
        bad = torch.nonzero(~same)
        at = tuple(bad[0].tolist())
        worst = float(((got - want).abs() / bound).nan_to_num(nan=math.inf)[~same].max())
        raise AssertionError(f"{name}: {len(bad)} of {got.numel()} out of bounds (worst {worst:.2f} of the bound), first at "
                             f"{at}: {float(got[at])} for {float(want[at])} +- {float(bound.expand_as(want)[at])}")
