"""What the attention operators over ordered series are measured on.

Rows lie in (key, ts) order, one series after the other, as the ordering step leaves them; `offsets` says where each
series starts.  Two operators, each over whole series (prompt), with its gradients (train) and row by row (step):

* decay: linear attention whose state decays by one factor per head and row -- the exponential moving average with
  weights that come from queries and keys;
* window: softmax attention over the last `window` rows of a series and its first `sinks` rows.

Windows (10, 30, 600, 1000), series counts (9 users, 100 symbols) and the decay 0.2 are those of this repository's
look-back, moving-average and range workloads; head layouts are generic.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # a feature encoder over one minute of 100 symbols, a handful of rows each: latency counts
        dict(name="decay_prompt_small", op="decay_prompt", n=2_000, series=100, heads=4, dk=64, dv=64, type="bf16",
             continued=False),
        # a new slice of every user's series that continues from the states of the slice before, odd head sizes
        dict(name="decay_prompt_continued", op="decay_prompt", n=30_011, series=9, heads=8, dk=40, dv=72, type="f32",
             continued=True),
        # nine users' series whole, the largest prompt
        dict(name="decay_prompt_large", op="decay_prompt", n=131_072, series=9, heads=16, dk=128, dv=128, type="bf16",
             continued=False),
        # a training step over 100 symbols
        dict(name="decay_train", op="decay_train", n=50_000, series=100, heads=16, dk=64, dv=64, type="bf16",
             continued=False),
        # one new row for each of 100 symbols
        dict(name="decay_step_small", op="decay_step", n=100, slots=128, heads=8, dk=64, dv=64, type="bf16"),
        # one new row for each of 512 series of a serving process
        dict(name="decay_step_large", op="decay_step", n=512, slots=640, heads=16, dk=128, dv=128, type="bf16"),
        # the look-back of ten rows, 32-bit features
        dict(name="window_prompt_lookback", op="window_prompt", n=20_000, series=100, heads=4, kv_heads=4, d=32,
             type="f32", window=10, sinks=0),
        # nine users' series whole, 600 rows back, shared key/value heads, first rows kept
        dict(name="window_prompt_large", op="window_prompt", n=131_072, series=9, heads=16, kv_heads=4, d=128,
             type="bf16", window=600, sinks=4),
        # a training step: 1000 rows back
        dict(name="window_train", op="window_train", n=32_768, series=9, heads=16, kv_heads=4, d=64, type="bf16",
             window=1000, sinks=4),
        # a training step at the moving average's 30 rows, odd head size, ragged short series
        dict(name="window_train_short", op="window_train", n=9_001, series=100, heads=6, kv_heads=2, d=24, type="f32",
             window=30, sinks=2),
        # one new row for each of nine users
        dict(name="window_step_small", op="window_step", n=9, slots=12, heads=8, kv_heads=2, d=64, type="bf16",
             window=600, sinks=4),
        # one new row for each of 256 series, 1000 rows back
        dict(name="window_step_large", op="window_step", n=256, slots=300, heads=32, kv_heads=8, d=128, type="bf16",
             window=1000, sinks=8),
    ]


def draw(rng):
    """One more case: sizes spread over the logarithm of the listed ranges, at most the cost of the largest."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["decay_prompt", "decay_train", "decay_step", "window_prompt", "window_train", "window_step"])
    most = [work(c) for c in listed()]
    most = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        case = dict(op=op, type=rng.choice(["bf16", "bf16", "f32"]))
        if op.startswith("decay"):
            case |= dict(heads=rng.randint(1, 16), dk=log(8, 128), dv=log(8, 128))
            if rng.random() < 0.5:
                case["dv"] = case["dk"] = rng.choice([16, 32, 64, 96, 128])
        else:
            kv = rng.randint(1, 8)
            case |= dict(heads=kv * rng.choice([1, 2, 3, 4]), kv_heads=kv, d=rng.choice([log(8, 128), 32, 64, 128]))
            case |= dict(window=log(10, 1000), sinks=rng.choice([0, 0, 1, 4, 8]))
        if op.endswith("step"):
            case |= dict(n=log(9, 512))
            case |= dict(slots=case["n"] + rng.randint(0, 100))
        else:
            case |= dict(n=log(2_000, 131_072 if op.endswith("prompt") else 50_000))
            case |= dict(series=min(log(1, 200), case["n"] // 10))
            if op.startswith("decay"):
                case["continued"] = rng.random() < 0.3
        w = work(case)
        if w["flops"] <= most[0] and w["bytes"] <= most[1]:
            return case


def lengths_of(case):
    """Rows of each series: ragged around the mean (from half of it to one and a half), whole number of rows."""
    s, n = case["series"], case["n"]
    share = 0.5 + (np.arange(s) + 0.5) / s
    ends = np.floor(np.cumsum(share) / share.sum() * n + 0.5).astype(np.int64)
    ends[-1] = n
    return np.diff(ends, prepend=0)


def counts_of(case):
    """Rows that each slot of a step has seen: seven of eight have passed their window, the others are young."""
    i, cap = np.arange(case["slots"]), case["window"] + case["sinks"]
    return np.where(i % 8 == 3, (cap * ((i // 8) % 5)) // 5, cap + (i * 7919) % (3 * cap)).astype(np.int64)


def pairs_of(case):
    """Visible (row, earlier row) pairs of one head."""
    total, w, s = 0, case["window"], case["sinks"]
    for m in lengths_of(case):
        i = np.arange(m)
        total += int(np.minimum(i + 1, w).sum() + np.minimum(np.maximum(i + 1 - w, 0), s).sum())
    return total


def work(case):
    n, e = case["n"], BYTES[case["type"]]
    if case["op"] == "decay_step":
        h, dk, dv = case["heads"], case["dk"], case["dv"]
        return {"bytes": n * h * (2 * dk + 2 * dv) * e + 8 * n * h * dk * dv, "flops": 5 * n * h * dk * dv}
    if case["op"].startswith("decay"):
        h, dk, dv = case["heads"], case["dk"], case["dv"]
        states = 8 * case["series"] * h * dk * dv if case["continued"] else 0
        if case["op"] == "decay_prompt":
            return {"bytes": n * h * (2 * dk + 2 * dv) * e + states, "flops": 4 * n * h * dk * dv}
        return {"bytes": n * h * (4 * dk + 4 * dv) * e + states, "flops": 12 * n * h * dk * dv}
    h, kv, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "window_step":
        used = case["n"] / case["slots"] * np.minimum(counts_of(case) + 1, case["window"] + case["sinks"]).sum()
        return {"bytes": (2 * used * kv * d + 2 * n * h * d + 4 * n * kv * d) * e + 16 * n, "flops": 4 * used * h * d}
    if case["op"] == "window_prompt":
        return {"bytes": n * d * (2 * h + 2 * kv) * e, "flops": 4 * h * d * pairs_of(case)}
    return {"bytes": n * d * (4 * h + 4 * kv) * e, "flops": 14 * h * d * pairs_of(case)}


def prepare(case, seed):
    dev, t = torch.device("cuda"), TYPES[case["type"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(t)

    st = dict(case)
    n, h = case["n"], case["heads"]
    decay = case["op"].startswith("decay")
    dk, dv = (case["dk"], case["dv"]) if decay else (case["d"], case["d"])
    kv = h if decay else case["kv_heads"]
    st.update(q=normal(n, h, dk), k=normal(n, kv, dk), v=normal(n, kv, dv), scale=1.0 / math.sqrt(dk))
    if decay:  # 1 - lambda from the moving average's 0.2 down to a 64th of it, head by head
        share = 0.2 * 2.0 ** (-6.0 * torch.arange(h, device=dev, dtype=torch.float64) / max(h - 1, 1))
        st["log_decay"] = torch.log1p(-share).float()
    if case["op"].endswith("step"):
        order = rng.permutation(case["slots"])[:n].astype(np.int32)
        st["slots"] = torch.from_numpy(order).to(dev)
        if decay:
            st["state"] = torch.randn(case["slots"], h, dk, dv, generator=g, device=dev) * 2
        else:
            cap = case["window"] + case["sinks"]
            st["k_cache"], st["v_cache"] = normal(case["slots"], cap, kv, dk), normal(case["slots"], cap, kv, dv)
            st["length"] = torch.from_numpy(counts_of(case)).to(dev)
        return st
    lens = rng.permutation(lengths_of(case))
    offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    st["lens"] = lens.tolist()
    st["offsets"] = torch.from_numpy(offsets).to(dev)
    if decay and case["continued"]:
        st["state"] = torch.randn(case["series"], h, dk, dv, generator=g, device=dev) * 2
    if case["op"].endswith("train"):
        st["dout"] = normal(n, h, dv)
    of = np.repeat(np.arange(case["series"]), lens)
    st["row_series"] = torch.from_numpy(of).to(dev)
    st["row_pos"] = torch.from_numpy(np.arange(n) - offsets[of]).to(dev)
    st["longest"] = int(lens.max())
    return st


# ---- the plain forms: series side by side in a padded array, elementary operations in 32 bits ----

def _padded(x, st, block):
    """[n, heads, d] -> [series, heads, rows, d], rows a multiple of `block`, zeros behind each series' end."""
    rows = -(-st["longest"] // block) * block
    out = torch.zeros(st["series"], rows, x.shape[1], x.shape[2], device=x.device, dtype=torch.float32)
    out = out.index_put((st["row_series"], st["row_pos"]), x)
    return out.transpose(1, 2)


def _packed(x, st):
    return x.transpose(1, 2)[st["row_series"], st["row_pos"]]


def _decay(q, k, v, st, state):
    c = 64
    q, k, v = (_padded(x, st, c) for x in (q, k, v))
    s, h, rows, dk = q.shape
    dv, nc = v.shape[3], rows // c
    ld, dev = st["log_decay"], q.device
    i = torch.arange(c, device=dev, dtype=torch.float32)
    gap = i[:, None] - i[None, :]
    within = torch.where(gap >= 0, torch.exp(ld[:, None, None] * gap.clamp(min=0)), 0.0)
    qc, kc, vc = q.reshape(s, h, nc, c, dk), k.reshape(s, h, nc, c, dk), v.reshape(s, h, nc, c, dv)
    out = (qc @ kc.transpose(3, 4) * within[None, :, None]) @ vc
    to_end = torch.exp(ld[:, None] * (c - 1 - i))[None, :, None, :, None]
    gains = ((kc * to_end).transpose(3, 4) @ vc).reshape(s, h, nc, dk * dv)
    b = torch.arange(nc, device=dev, dtype=torch.float32)
    steps = b[:, None] - 1 - b[None, :]
    over = torch.where(steps >= 0, torch.exp(ld[:, None, None] * c * steps.clamp(min=0)), 0.0)
    before = (over[None] @ gains).reshape(s, h, nc, dk, dv)
    if state is not None:
        before = before + torch.exp(ld[:, None] * c * b)[None, :, :, None, None] * state[:, :, None]
    out = out + torch.exp(ld[:, None] * (i + 1))[None, :, None, :, None] * (qc @ before)
    out = _packed(out.reshape(s, h, rows, dv), st) * st["scale"]
    if state is None:
        return out, None
    lens = (st["offsets"][1:] - st["offsets"][:-1]).float()
    left = lens[:, None] - 1 - torch.arange(rows, device=dev, dtype=torch.float32)
    weight = torch.where(left[:, None] >= 0, torch.exp(ld[None, :, None] * left[:, None].clamp(min=0)), 0.0)
    last = (k * weight[..., None]).transpose(2, 3) @ v + torch.exp(ld[None] * lens[:, None])[..., None, None] * state
    return out, last


def _window(q, k, v, st):
    w, sinks, scale = st["window"], st["sinks"], st["scale"]
    c = max(w, 64)
    q, k, v = (_padded(x, st, c) for x in (q, k, v))
    s, h, rows, d = q.shape
    kv, nb = k.shape[1], rows // c
    g = h // kv
    qb = q.reshape(s, kv, g, nb, c, d).transpose(2, 3).reshape(s, kv, nb, g * c, d)

    def both(x):  # each block of rows behind the block before it
        x = x.reshape(s, kv, nb, c, d)
        return torch.cat([torch.cat([torch.zeros_like(x[:, :, :1]), x[:, :, :-1]], 2), x], 3)

    dev = q.device
    i = torch.arange(rows, device=dev).reshape(nb, c).repeat(1, g)[:, :, None]
    j = torch.arange(nb, device=dev)[:, None, None] * c - c + torch.arange(2 * c, device=dev)
    seen = (j >= 0) & (j <= i) & (j > i - w)
    scores = qb @ both(k).transpose(3, 4) * scale
    scores = torch.where(seen, scores, -math.inf)
    if sinks:
        first = min(sinks, rows)
        ks, vs = k[:, :, None, :first], v[:, :, None, :first]
        early = torch.arange(first, device=dev) <= i - w
        scores = torch.cat([scores, torch.where(early, qb @ ks.transpose(3, 4) * scale, -math.inf)], 4)
    p = torch.exp(scores - scores.amax(4, keepdim=True).detach())
    p = p / p.sum(4, keepdim=True)
    out = p[..., :2 * c] @ both(v)
    if sinks:
        out = out + p[..., 2 * c:] @ vs
    out = out.reshape(s, kv, nb, g, c, d).transpose(2, 3).reshape(s, h, rows, d)
    return _packed(out, st)


def _plain(st):
    t, op = st["q"].dtype, st["op"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if op == "decay_step":
        slots = st["slots"].long()
        s = st["state"][slots] * torch.exp(st["log_decay"])[:, None, None] + k[..., None] * v[..., None, :]
        st["state"][slots] = s
        return ((q[..., None] * s).sum(2) * st["scale"]).to(t), st["state"]
    if op == "window_step":
        slots, sinks = st["slots"].long(), st["sinks"]
        cap = st["window"] + sinks
        at = st["length"][slots]
        place = torch.where(at < sinks, at, sinks + (at - sinks) % st["window"])
        st["k_cache"][slots, place], st["v_cache"][slots, place] = st["k"], st["v"]
        st["length"][slots] = at + 1
        kc, vc = (st[x][slots].float().transpose(1, 2) for x in ("k_cache", "v_cache"))
        n, h, d = q.shape
        kv = kc.shape[1]
        scores = q.reshape(n, kv, h // kv, d) @ kc.transpose(2, 3) * st["scale"]
        seen = torch.arange(cap, device=q.device) <= at[:, None, None, None]
        scores = torch.where(seen, scores, -math.inf)
        p = torch.exp(scores - scores.amax(3, keepdim=True))
        out = (p / p.sum(3, keepdim=True)) @ vc
        return out.reshape(n, h, d).to(t), st["k_cache"], st["v_cache"], st["length"]
    if op == "decay_prompt":
        out, last = _decay(q, k, v, st, st.get("state"))
        return (out.to(t),) if last is None else (out.to(t), last)
    if op == "window_prompt":
        return (_window(q, k, v, st).to(t),)
    leaves = [q, k, v] + ([st["state"].clone()] if "state" in st else [])
    leaves = [x.detach().requires_grad_() for x in leaves]
    if op == "decay_train":
        out, _ = _decay(*leaves[:3], st, leaves[3] if len(leaves) > 3 else None)
    else:
        out = _window(*leaves, st)
    grads = torch.autograd.grad(out, leaves, st["dout"].float())
    return [out.detach().to(t)] + [x.to(t) for x in grads[:3]] + list(grads[3:])


def _calls(st):
    from tempo_amd import ops
    op, q, k, v = st["op"], st["q"], st["k"], st["v"]
    if op == "decay_step":
        out = ops.decay_attention_step(q, k, v, st["log_decay"], st["state"], slots=st["slots"], scale=st["scale"])
        return out, st["state"]
    if op == "window_step":
        out = ops.window_attention_step(q, k, v, st["k_cache"], st["v_cache"], st["length"], sinks=st["sinks"],
                                        slots=st["slots"], scale=st["scale"])
        return out, st["k_cache"], st["v_cache"], st["length"]
    if op.startswith("decay"):
        how = dict(offsets=st["offsets"], scale=st["scale"], state=st.get("state"))
        if op == "decay_prompt":
            if "state" in st:
                return ops.decay_attention(q, k, v, st["log_decay"], return_state=True, **how)
            return (ops.decay_attention(q, k, v, st["log_decay"], **how),)
        out = ops.decay_attention(q, k, v, st["log_decay"], **how)
        grads = ops.decay_attention_grad(st["dout"], q, k, v, st["log_decay"], return_dstate="state" in st, **how)
        return [out] + list(grads)
    how = dict(sinks=st["sinks"], offsets=st["offsets"], scale=st["scale"])
    if op == "window_prompt":
        return (ops.window_attention(q, k, v, st["window"], **how),)
    out, lse = ops.window_attention(q, k, v, st["window"], return_lse=True, **how)
    return [out] + list(ops.window_attention_grad(st["dout"], q, k, v, out, lse, st["window"], **how))


def run(state):
    return _calls(state) if own else _plain(state)


# ---- the definition in 64 bits, series by series and row block by row block ----

def _exact_step(st):
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    slots = st["slots"].long()
    if st["op"] == "decay_step":
        state = st["state"].double()
        fade = torch.exp(st["log_decay"].double())
        out = torch.empty(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
        for b, slot in enumerate(st["slots"].tolist()):
            s = fade[:, None, None] * state[slot] + torch.einsum("hk,hv->hkv", k[b], v[b])
            state[slot] = s
            out[b] = torch.einsum("hk,hkv->hv", q[b], s) * st["scale"]
        return out, state
    w, sinks = st["window"], st["sinks"]
    length = st["length"].clone()
    kc, vc = st["k_cache"], st["v_cache"]
    out = torch.empty(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    g = q.shape[1] // k.shape[1]
    for b, slot in enumerate(st["slots"].tolist()):
        at = int(length[slot])
        place = at if at < sinks else sinks + (at - sinks) % w
        kc[slot, place], vc[slot, place] = st["k"][b], st["v"][b]
        length[slot] = at + 1
        keys = kc[slot, :at + 1].double().repeat_interleave(g, 1)
        vals = vc[slot, :at + 1].double().repeat_interleave(g, 1)
        p = torch.softmax(torch.einsum("hd,jhd->hj", q[b], keys) * st["scale"], 1)
        out[b] = torch.einsum("hj,jhd->hd", p, vals)
    return out, kc, vc, length


def _exact_series(st):
    """Every series on its own: blocks of rows against all rows that they see, with the gradients' own formulas."""
    q, k, v = (st[x].double().transpose(0, 1) for x in ("q", "k", "v"))  # [heads, n, d]
    do = st["dout"].double().transpose(0, 1) if "dout" in st else None
    scale, decay = st["scale"], st["op"].startswith("decay")
    h, n, _ = q.shape
    g, dev = h // k.shape[0], q.device
    out = torch.zeros(h, n, v.shape[2], dtype=torch.float64, device=dev)
    dq = torch.zeros_like(q)
    dk = torch.zeros(h, n, k.shape[2], dtype=torch.float64, device=dev)
    dv = torch.zeros(h, n, v.shape[2], dtype=torch.float64, device=dev)
    state = st["state"].double() if "state" in st else None
    last = torch.zeros_like(state) if state is not None else None
    ds = torch.zeros_like(state) if state is not None else None
    ld = st["log_decay"].double() if decay else None
    start = 0
    for s, m in enumerate(st["lens"]):
        end = start + m
        for a in range(start, end, 512):
            b = min(a + 512, end)
            i = torch.arange(a, b, device=dev)[:, None]
            if decay:
                cols = torch.arange(start, b, device=dev)
                gap = (i - cols).double()
                fade = torch.where(gap >= 0, torch.exp(ld[:, None, None] * gap.clamp(min=0)), 0.0)
            else:
                lo = max(start, a - st["window"] + 1)
                cols = torch.cat([torch.arange(start, min(start + st["sinks"], lo), device=dev),
                                  torch.arange(lo, b, device=dev)])
                seen = (cols <= i) & ((cols > i - st["window"]) | (cols < start + st["sinks"]))
            kk, vv = k[:, cols].repeat_interleave(g, 0), v[:, cols].repeat_interleave(g, 0)
            x = torch.bmm(q[:, a:b], kk.transpose(1, 2).contiguous()) * scale
            p = x * fade if decay else torch.softmax(x.masked_fill(~seen, -math.inf), 2)
            out[:, a:b] += torch.bmm(p, vv)
            if do is None:
                continue
            dp = torch.bmm(do[:, a:b], vv.transpose(1, 2).contiguous())
            dx = dp * fade if decay else p * (dp - (dp * p).sum(2, keepdim=True))
            dq[:, a:b] += torch.bmm(dx, kk) * scale
            dk.index_add_(1, cols, torch.bmm(dx.transpose(1, 2).contiguous(), q[:, a:b]) * scale)
            dv.index_add_(1, cols, torch.bmm(p.transpose(1, 2).contiguous(), do[:, a:b]))
        if state is not None and m:
            rank = torch.arange(m, device=dev, dtype=torch.float64)
            into = torch.exp(ld[:, None] * (rank + 1))[..., None] * scale
            out[:, start:end] += torch.bmm(q[:, start:end] * into, state[s])
            left = torch.exp(ld[:, None] * (m - 1 - rank))[..., None]
            last[s] = torch.bmm((k[:, start:end] * left).transpose(1, 2).contiguous(), v[:, start:end])
            if do is not None:
                dq[:, start:end] += torch.bmm(do[:, start:end], state[s].transpose(1, 2).contiguous()) * into
                ds[s] = torch.bmm((q[:, start:end] * into).transpose(1, 2).contiguous(), do[:, start:end])
        if state is not None:
            last[s] += torch.exp(ld * m)[:, None, None] * state[s]
        start = end
    out, dq = out.transpose(0, 1).contiguous(), dq.transpose(0, 1).contiguous()
    if do is None:
        return (out,) if state is None else (out, last)
    dk, dv = (x.reshape(h // g, g, n, -1).sum(1).transpose(0, 1).contiguous() for x in (dk, dv))
    return [out, dq, dk, dv] + ([ds] if state is not None else [])


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_step(st) if case["op"].endswith("step") else _exact_series(st)
