"""Attention over series (tempo_amd/attention.py) against its definition in 64 bits: tests/attention_cases.py
says how far each result may be off."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import attention_cases as ref  # noqa: E402

# rows of each series, empty ones among them; (rows before the first, rows behind the last)
LENGTHS = {
    "one": [1],
    "short": [1, 1, 2, 0, 3, 1],
    "ragged": [0, 5, 0, 0, 130, 1, 63, 64, 65, 0],
    "long": [700, 0, 800],
    "many": [17, 3, 41, 29, 2, 8, 55, 31, 12, 1, 1, 90] * 3,
}


def _offsets(lens, before=0):
    o = [before]
    for m in lens:
        o.append(o[-1] + m)
    return o


def _inputs(seed, n, heads, kv, dk, dv, dtype, live=None):
    g = torch.Generator().manual_seed(seed)
    make = lambda h, d: torch.randn(n, h, d, generator=g).to(dtype)  # noqa: E731
    t = [make(heads, dk), make(kv, dk), make(kv, dv), make(heads, dv)]
    if live is not None:  # rows of no series hold anything
        for x in t:
            x[:live[0]] = math.nan
            x[live[1]:] = math.inf
    return t


WINDOW = [
    # lengths, before, behind, heads, kv_heads, dk, dv, window, sinks
    ("one", 0, 0, 1, 1, 8, 8, 1, 0),
    ("one", 0, 0, 2, 1, 64, 64, 10, 4),
    ("short", 2, 3, 4, 2, 19, 5, 2, 1),
    ("ragged", 3, 7, 2, 2, 32, 32, 10, 0),
    ("ragged", 0, 70, 4, 1, 24, 24, 30, 2),
    ("ragged", 130, 0, 6, 2, 64, 64, 64, 4),
    ("ragged", 0, 0, 3, 3, 128, 128, 1000, 0),
    ("ragged", 0, 0, 2, 1, 40, 72, 1, 32),
    ("long", 0, 5, 4, 2, 64, 64, 40, 4),
    ("long", 1, 0, 2, 1, 128, 128, 300, 32),
    ("long", 0, 0, 2, 2, 16, 100, 600, 1),
    ("long", 200, 200, 1, 1, 32, 32, 7, 7),
    ("many", 5, 5, 2, 1, 72, 72, 20, 3),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(map(str, c)))
def test_window_attention(case, dtype):
    from tempo_amd import ops
    which, before, behind, heads, kv, dk, dv, window, sinks = case
    off = _offsets(LENGTHS[which], before)
    n = off[-1] + behind
    q, k, v, do = _inputs(heads * 31 + dk + window, n, heads, kv, dk, dv, dtype, (before, off[-1]))
    scale = dk ** -0.5
    want = ref.window_reference(q, k, v, do, off, window, sinks, scale)
    d = [x.cuda() for x in (q, k, v, do)]
    o = torch.tensor(off, device="cuda")
    out, lse = ops.window_attention(*d[:3], window, sinks=sinks, offsets=o, return_lse=True)
    ref.check("out", out, *want["out"])
    ref.check("lse", lse, *want["lse"])
    for name, x in zip(("dq", "dk", "dv"), ops.window_attention_grad(d[3], *d[:3], out, lse, window, sinks=sinks, offsets=o)):
        assert x.dtype == dtype
        ref.check(name, x, *want[name])


DECAY = [
    # lengths, before, behind, heads, dk, dv, log decays, state
    ("one", 0, 0, 1, 8, 8, [-0.1], True),
    ("short", 2, 3, 2, 19, 5, [-0.2, 0.0], True),
    ("ragged", 3, 7, 2, 32, 32, [-0.22314355, -1e-3], False),
    ("ragged", 0, 70, 2, 64, 64, [-0.05, -3.0], True),
    ("ragged", 130, 0, 3, 128, 128, [-0.01, -40.0, -math.inf], True),
    ("long", 0, 5, 2, 64, 64, [-0.003, -0.2], True),
    ("long", 1, 0, 1, 128, 128, [-0.02], False),
    ("long", 0, 0, 2, 40, 72, [-0.1, -1e-4], True),
    ("long", 200, 200, 1, 100, 16, [-0.05], True),
    ("many", 5, 5, 2, 24, 24, [-0.22314355, -0.01], True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", DECAY, ids=lambda c: "-".join(map(str, c[:6])))
def test_decay_attention(case, dtype):
    from tempo_amd import ops
    which, before, behind, heads, dk, dv, decays, with_state = case
    off = _offsets(LENGTHS[which], before)
    n, ns = off[-1] + behind, len(off) - 1
    q, k, v, do = _inputs(len(which) * 7 + dk, n, heads, heads, dk, dv, dtype, (before, off[-1]))
    g = torch.Generator().manual_seed(dv)
    state = torch.randn(ns, heads, dk, dv, generator=g) if with_state else None
    dstate = torch.randn(ns, heads, dk, dv, generator=g) if with_state else None
    ld = torch.tensor(decays)
    want = ref.decay_reference(q, k, v, ld, off, dk ** -0.5, state, do, dstate)
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    d, o = [x.cuda() for x in (q, k, v, do)], torch.tensor(off, device="cuda")
    out, last = ops.decay_attention(*d[:3], ld.cuda(), offsets=o, state=dev(state), return_state=True)
    ref.check("out", out, *want["out"])
    ref.check("state", last, *want["state"])
    alone = ops.decay_attention(*d[:3], ld.cuda(), offsets=o, state=dev(state))
    ref.check("out alone", alone, *want["out"])
    grads = ops.decay_attention_grad(d[3], *d[:3], ld.cuda(), offsets=o, state=dev(state), dstate=dev(dstate),
                                     return_dstate=True)
    for name, x in zip(("dq", "dk", "dv", "dstate"), grads):
        ref.check(name, x, *want[name])


STEP = [
    # slots, rows, heads, kv, dk, dv, window, sinks
    (1, 1, 1, 1, 8, 8, 1, 0),
    (7, 4, 4, 2, 19, 5, 3, 1),
    (9, 9, 8, 1, 64, 64, 100, 4),
    (5, 3, 40, 1, 128, 128, 33, 0),
    (6, 5, 6, 3, 40, 72, 64, 32),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", STEP, ids=lambda c: "-".join(map(str, c)))
def test_steps_go_on_where_whole_series_end(case, dtype):
    """Series through the whole-series forms, their states and caches filled from them, then row by row; each row
    equals the definition over the whole series."""
    from tempo_amd import ops
    slots, rows, heads, kv, dk, dv, window, sinks = case
    lens = [(i * 37 + 3 * (i % 3)) % (window + sinks + 40) for i in range(rows)]
    new = 4
    off = _offsets([m + new for m in lens])
    q, k, v, do = _inputs(dk + rows, off[-1], heads, kv, dk, dv, dtype)
    scale = dk ** -0.5
    want = ref.window_reference(q, k, v, do, off, window, sinks, scale)["out"]
    old = torch.cat([torch.arange(off[i], off[i] + lens[i]) for i in range(rows)])
    o_old = torch.tensor(_offsets(lens), device="cuda")
    which = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:rows].to(torch.int32).cuda()
    kc = torch.full((slots, window + sinks, kv, dk), math.nan, dtype=dtype, device="cuda")
    vc = torch.full((slots, window + sinks, kv, dv), math.nan, dtype=dtype, device="cuda")
    length = torch.full((slots,), -5, dtype=torch.int64, device="cuda")
    ops.window_cache_write(k[old].cuda(), v[old].cuda(), kc, vc, length, sinks=sinks, offsets=o_old, slots=which)
    assert length[which.long()].tolist() == lens
    assert int((length == -5).sum()) == slots - rows
    for t in range(new):
        at = torch.tensor([off[i] + lens[i] + t for i in range(rows)])
        out = ops.window_attention_step(q[at].cuda(), k[at].cuda(), v[at].cuda(), kc, vc, length, sinks=sinks, slots=which)
        ref.check(f"row {t}", out, want[0][at], want[1][at])
    assert length[which.long()].tolist() == [m + new for m in lens]
    # the decay form of the same rows, key/value heads given to each query head
    g = heads // kv
    k2, v2 = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    ld = torch.linspace(-0.3, -0.001, heads)
    full = ref.decay_reference(q, k2, v2, ld, off, scale)
    _, last = ops.decay_attention(q[old].cuda(), k2[old].cuda(), v2[old].cuda(), ld.cuda(), offsets=o_old, return_state=True)
    state = torch.full((slots, heads, dk, dv), math.nan, device="cuda")
    state[which.long()] = last
    for t in range(new):
        at = torch.tensor([off[i] + lens[i] + t for i in range(rows)])
        out = ops.decay_attention_step(q[at].cuda(), k2[at].cuda(), v2[at].cuda(), ld.cuda(), state, slots=which)
        ref.check(f"decay row {t}", out, full["out"][0][at], full["out"][1][at])
    ref.check("decay state", state[which.long()], full["state"][0], full["state"][1] * 2)
