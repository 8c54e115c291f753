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
    ("many", 5, 6, 1, 1, 85, 9, 20, 3),
    ("long", 1, 0, 3, 1, 7, 121, 50, 2),
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
    # odd sizes of one head: rows that start at odd multiples of two bytes
    ("many", 5, 6, 1, 85, 9, [-0.1], False),
    ("long", 1, 0, 1, 85, 9, [-0.1], True),
    ("many", 0, 0, 3, 7, 121, [-0.1, -0.5, -0.01], True),
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


def _dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_strided_rows(dtype):
    """Slices of one projection's output, heads before rows, odd paddings, shared rows of a broadcast key."""
    from tempo_amd import ops
    n, h, kv, d = 150, 4, 2, 40
    off = [0, 70, 150]
    o = torch.tensor(off, device="cuda")
    g = torch.Generator().manual_seed(5)
    packed = torch.randn(n, h + 2 * kv, d, generator=g).to(dtype)
    q, k, v = packed[:, :h], packed[:, h:h + kv], packed[:, h + kv:]
    do = torch.randn(h, n, d + 3, generator=g).to(dtype).transpose(0, 1)[:, :, 1:d + 1]
    want = ref.window_reference(q, k, v, do, off, 30, 2, d ** -0.5)
    pc = packed.cuda()
    qd, kd, vd = pc[:, :h], pc[:, h:h + kv], pc[:, h + kv:]
    dod = torch.empty(h, n, d + 3, dtype=dtype, device="cuda").transpose(0, 1)[:, :, 1:d + 1]
    dod.copy_(do)
    out, lse = ops.window_attention(qd, kd, vd, 30, sinks=2, offsets=o, return_lse=True)
    ref.check("out", out, *want["out"])
    for name, x in zip(("dq", "dk", "dv"), ops.window_attention_grad(dod, qd, kd, vd, out, lse, 30, sinks=2, offsets=o)):
        ref.check(name, x, *want[name])
    ld = torch.tensor([-0.2, -0.01, -1.0, 0.0])
    k4, v4 = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    want = ref.decay_reference(q, k4, v4, ld, off, d ** -0.5, dout=do)
    # head order in memory reversed, rows far apart
    wide = torch.empty(n, 3, h, d, dtype=dtype, device="cuda")
    wide[:, 1].copy_(k4)
    got = ops.decay_attention(qd, wide[:, 1], v4.cuda(), ld.cuda(), offsets=o)
    ref.check("decay out", got, *want["out"])
    for name, x in zip(("dq", "dk", "dv"), ops.decay_attention_grad(dod, qd, wide[:, 1], v4.cuda(), ld.cuda(), offsets=o)):
        ref.check("decay " + name, x, *want[name])
    # one key row for all rows: rows that overlap in memory
    one = k4[:1].expand(n, h, d)
    want = ref.decay_reference(q, one, v4, ld, off, d ** -0.5)
    ref.check("broadcast", ops.decay_attention(qd, k4[:1].cuda().expand(n, h, d), v4.cuda(), ld.cuda(), offsets=o), *want["out"])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_values_that_are_not_finite_stay_where_they_are_seen(bad, dtype):
    """One bad element of each input in turn: results that do not depend on it are as without it, those that do are
    not finite."""
    from tempo_amd import ops
    lens, window, sinks, h, d = [60, 100, 45], 20, 2, 2, 32
    off = _offsets(lens)
    n = off[-1]
    o = torch.tensor(off, device="cuda")
    clean = _inputs(77, n, h, h, d, d, dtype)
    mask = ref.window_mask(n, off, window, sinks)
    sid, pos = ref.series_of(n, off)
    same = (sid[:, None] == sid[None]) & (pos[None] <= pos[:, None])
    ld = torch.tensor([-0.1, -0.02]).cuda()

    def run(ts):
        q, k, v, do = _dev(*ts)
        out, lse = ops.window_attention(q, k, v, window, sinks=sinks, offsets=o, return_lse=True)
        res = [out, *ops.window_attention_grad(do, q, k, v, out, lse, window, sinks=sinks, offsets=o)]
        res.append(ops.decay_attention(q, k, v, ld, offsets=o))
        res += ops.decay_attention_grad(do, q, k, v, ld, offsets=o)
        return [x.float().cpu() for x in res]

    base = run(clean)
    names = ["out", "dq", "dk", "dv", "decay out", "decay dq", "decay dk", "decay dv"]
    head, elem = 1, 7
    for which, row in ((0, 75), (1, 61), (1, 110), (2, 60), (2, 130), (3, 90)):
        ts = [x.clone() for x in clean]
        ts[which][row, head, elem] = bad
        got = run(ts)
        for name, see, res in (("", mask, range(0, 4)), ("decay ", same, range(4, 8))):
            rows = torch.zeros(n, dtype=torch.bool)  # query rows that the element bears on, key rows of theirs
            if which in (0, 3):
                rows[row] = True
            else:
                rows = see[:, row].clone()
            keys = see[rows].any(0)
            if which in (1, 2):
                keys[row] = True
            for i in res:
                touched = (rows if i % 4 < 2 else keys)
                if i % 4 == 0 and which == 3:
                    touched = torch.zeros(n, dtype=torch.bool)
                x, y = got[i][~touched], base[i][~touched]
                assert torch.equal(x, y), f"{names[i]} changed outside what input {which} row {row} bears on"
                assert torch.equal(got[i][:, 0], base[i][:, 0]), f"{names[i]}: another head changed"
        # the results that take the element directly
        if which == 2:
            for i in (0, 4):
                seen = (mask if i == 0 else same)[:, row]
                assert not torch.isfinite(got[i][seen, head, elem]).any()
                others = [e for e in range(d) if e != elem]
                assert torch.equal(got[i][:, head, others], base[i][:, head, others])


def test_rows_of_no_series_and_wrong_offsets():
    """Everything outside of all series is zero whatever it holds; offsets that make no sense end in some result."""
    from tempo_amd import ops
    n, h, d = 300, 2, 32
    q, k, v, do = _dev(*_inputs(3, n, h, h, d, d, torch.float32))
    ld = torch.tensor([-0.1, -0.2]).cuda()
    for off in ([n, n], [0], [0, 0, 0], [50, 50, 60, 60]):
        o = torch.tensor(off, device="cuda")
        lo, hi = off[0], off[-1] if len(off) > 1 else off[0]
        out, lse = ops.window_attention(q, k, v, 9, sinks=1, offsets=o, return_lse=True)
        res = [out, *ops.window_attention_grad(do, q, k, v, out, lse, 9, sinks=1, offsets=o),
               ops.decay_attention(q, k, v, ld, offsets=o), *ops.decay_attention_grad(do, q, k, v, ld, offsets=o)]
        for x in res:
            assert not x[:lo].any() and not x[hi:].any()
        assert torch.isinf(lse[:lo]).all() and torch.isinf(lse[hi:]).all()
    for off in ([9, 3, 200, 100, 250], [-5, 40, 1000], [400, 10], [0, 300, 0, 300], [2 ** 40, -2 ** 40]):
        o = torch.tensor(off, device="cuda")
        out, lse = ops.window_attention(q, k, v, 9, sinks=1, offsets=o, return_lse=True)
        ops.window_attention_grad(do, q, k, v, out, lse, 9, sinks=1, offsets=o)
        st = torch.zeros(len(off) - 1, h, d, d, device="cuda")
        ops.decay_attention(q, k, v, ld, offsets=o, state=st, return_state=True)
        ops.decay_attention_grad(do, q, k, v, ld, offsets=o, state=st, return_dstate=True)
        torch.cuda.synchronize()


def test_no_rows_no_series():
    from tempo_amd import ops
    ld = torch.tensor([-0.1, -0.2]).cuda()
    e = torch.empty(0, 2, 8, device="cuda")
    for o, ns in ((None, 1), (torch.tensor([0], device="cuda"), 0), (torch.zeros(4, dtype=torch.int64, device="cuda"), 3)):
        assert ops.window_attention(e, e, e, 5, offsets=o).shape == (0, 2, 8)
        st = torch.randn(ns, 2, 8, 8, device="cuda")
        out, last = ops.decay_attention(e, e, e, ld, offsets=o, state=st, return_state=True)
        assert out.shape == (0, 2, 8) and torch.equal(last, st)
        grads = ops.decay_attention_grad(e, e, e, e, ld, offsets=o, state=st, dstate=st, return_dstate=True)
        assert torch.equal(grads[3], st)
        out, last = ops.decay_attention(e, e, e, ld, offsets=o, return_state=True)
        assert not last.any()
    assert ops.decay_attention_step(e, e, e, ld, torch.zeros(3, 2, 8, 8, device="cuda"),
                                    slots=torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 2, 8)
    kc = torch.zeros(3, 4, 2, 8, device="cuda")
    ln = torch.zeros(3, dtype=torch.int64, device="cuda")
    assert ops.window_attention_step(e, e, e, kc, kc.clone(), ln, slots=torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 2, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_slots_out_of_range_and_named_twice(dtype):
    """Such rows change nothing and give NaN; the others are as without them."""
    from tempo_amd import ops
    n, slots, h, kv, d, window, sinks = 6, 4, 4, 2, 16, 5, 1
    q, k, v, _ = _dev(*_inputs(9, n, h, kv, d, d, dtype))
    which = torch.tensor([2, 7, 2, 0, -1, 0], dtype=torch.int32, device="cuda")
    good, bad = [0, 3], [1, 2, 4, 5]
    g = torch.Generator(device="cuda").manual_seed(1)
    kc = torch.randn(slots, window + sinks, kv, d, generator=g, device="cuda").to(dtype)
    vc = torch.randn(slots, window + sinks, kv, d, generator=g, device="cuda").to(dtype)
    length = torch.tensor([3, 9, 40, 0], device="cuda")
    a, b = (kc.clone(), vc.clone(), length.clone()), (kc.clone(), vc.clone(), length.clone())
    out = ops.window_attention_step(q, k, v, *a, sinks=sinks, slots=which)
    alone = ops.window_attention_step(q[good], k[good], v[good], *b, sinks=sinks, slots=which[good].contiguous())
    assert torch.equal(out[good], alone) and torch.isnan(out[bad]).all()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert a[2].tolist() == [4, 9, 41, 0]
    k4, v4 = k.repeat_interleave(2, 1).contiguous(), v.repeat_interleave(2, 1).contiguous()
    ld = torch.linspace(-0.5, 0, h).cuda()
    s1 = torch.randn(slots, h, d, d, generator=g, device="cuda")
    s2, s0 = s1.clone(), s1.clone()
    out = ops.decay_attention_step(q, k4, v4, ld, s1, slots=which)
    alone = ops.decay_attention_step(q[good], k4[good], v4[good], ld, s2, slots=which[good].contiguous())
    assert torch.equal(out[good], alone) and torch.isnan(out[bad]).all() and torch.equal(s1, s2)
    assert torch.equal(s1[[1, 3]], s0[[1, 3]])


def test_differentiable():
    """autograd calls the backward passes; inputs that need none get none."""
    from tempo_amd import ops
    off = torch.tensor([0, 33, 90], device="cuda")
    q, k, v, do = _dev(*_inputs(21, 90, 4, 2, 24, 24, torch.float32))
    for t in (q, k, v):
        t.requires_grad_()
    out, lse = ops.window_attention(q, k, v, 12, sinks=2, offsets=off, return_lse=True)
    assert not lse.requires_grad
    out.backward(do)
    want = ops.window_attention_grad(do, q.detach(), k.detach(), v.detach(), out.detach(), lse, 12, sinks=2, offsets=off)
    assert all(torch.equal(t.grad, w) for t, w in zip((q, k, v), want))
    with torch.no_grad():
        assert ops.window_attention(q, k, v, 12, offsets=off).grad_fn is None
    k4, v4 = k.detach().repeat_interleave(2, 1).requires_grad_(), v.detach().repeat_interleave(2, 1)
    st = torch.randn(2, 4, 24, 24, device="cuda", requires_grad=True)
    ld = torch.linspace(-0.5, -0.01, 4).cuda()
    q.grad = None
    out, last = ops.decay_attention(q, k4, v4, ld, offsets=off, state=st, return_state=True)
    ds = torch.randn_like(last)
    torch.autograd.backward([out, last], [do, ds])
    want = ops.decay_attention_grad(do, q.detach(), k4.detach(), v4, ld, offsets=off, state=st.detach(), dstate=ds, return_dstate=True)
    assert torch.equal(q.grad, want[0]) and torch.equal(k4.grad, want[1]) and torch.equal(st.grad, want[3])
    out = ops.decay_attention(q, k4, v4, ld, offsets=off)
    (gq,) = torch.autograd.grad(out.sum(), q)  # (a gradient that is one number repeated)
    assert torch.isfinite(gq).all()
    with pytest.raises(ValueError, match="log_decay"):
        ops.decay_attention(q, k4, v4, ld.requires_grad_(), offsets=off)


def test_captured_and_replayed():
    """A whole training step and two serving steps in one graph, replayed with eager work in between."""
    from tempo_amd import ops
    off = torch.tensor([0, 300, 700], device="cuda")
    q, k, v, do = _dev(*_inputs(4, 700, 4, 2, 64, 64, torch.bfloat16))
    k4, v4 = k.repeat_interleave(2, 1).contiguous(), v.repeat_interleave(2, 1).contiguous()
    ld = torch.linspace(-0.5, -0.01, 4).cuda()
    st0 = torch.randn(2, 4, 64, 64, device="cuda")
    state, kc, vc = st0.clone(), torch.zeros(2, 52, 2, 64, dtype=torch.bfloat16, device="cuda"), None
    vc, length = kc.clone(), torch.zeros(2, dtype=torch.int64, device="cuda")
    slots = torch.tensor([1, 0], dtype=torch.int32, device="cuda")

    def step():
        out, lse = ops.window_attention(q, k, v, 50, sinks=2, offsets=off, return_lse=True)
        grads = ops.window_attention_grad(do, q, k, v, out, lse, 50, sinks=2, offsets=off)
        o2, last = ops.decay_attention(q, k4, v4, ld, offsets=off, state=st0, return_state=True)
        g2 = ops.decay_attention_grad(do, q, k4, v4, ld, offsets=off, state=st0, return_dstate=True)
        o3 = ops.decay_attention_step(q[:2], k4[:2], v4[:2], ld, state, slots=slots)
        o4 = ops.window_attention_step(q[:2], k[:2], v[:2], kc, vc, length, sinks=2, slots=slots)
        return [out, lse, *grads, o2, last, *g2, o3, o4]

    def reset():
        state.copy_(st0)
        kc.zero_(), vc.zero_(), length.zero_()

    want = []
    for _ in range(4):
        want.append([x.clone() for x in step()])
    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    reset()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
        ops.window_attention(q, k, v, 7)
        torch.randn(1000, device="cuda").sum().item()
    assert length.tolist() == [4, 4]


def test_on_another_stream():
    from tempo_amd import ops
    q, k, v, do = _dev(*_inputs(8, 900, 2, 2, 64, 64, torch.bfloat16))
    want, lse = ops.window_attention(q, k, v, 100, return_lse=True)
    grads = ops.window_attention_grad(do, q, k, v, want, lse, 100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, l2 = ops.window_attention(q, k, v, 100, return_lse=True)
        b = ops.window_attention_grad(do, q, k, v, a, l2, 100)
    side.synchronize()
    assert torch.equal(a, want) and all(torch.equal(x, y) for x, y in zip(b, grads))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_long_series_over_many_sections(dtype):
    """Series far longer than a section of the walk, against the recurrence in 64 bits."""
    from tempo_amd import ops
    lens, h, dk, dv = [9_000, 1, 15_001], 8, 16, 12
    off = _offsets(lens)
    n = off[-1]
    q, k, v, do = _inputs(13, n, h, h, dk, dv, dtype)
    ld = -0.5 * 2.0 ** -torch.arange(h).float()
    ld[-1] = 0.0
    scale = 0.25
    Q, K, V = (x.double() for x in (q, k, v))
    lam = torch.exp(ld.double())[:, None, None]
    out = torch.empty(n, h, dv, dtype=torch.float64)
    mag = torch.empty(n, h, dv, dtype=torch.float64)
    last = []
    for s in range(len(lens)):
        S, A = torch.zeros(h, dk, dv, dtype=torch.float64), torch.zeros(h, dk, dv, dtype=torch.float64)
        for i in range(off[s], off[s + 1]):
            S = lam * S + K[i, :, :, None] * V[i, :, None, :]
            A = lam * A + (K[i, :, :, None] * V[i, :, None, :]).abs()
            out[i] = (Q[i, :, :, None] * S).sum(1) * scale
            mag[i] = (Q[i, :, :, None].abs() * A).sum(1) * scale
        last.append((S, A))
    u = ref.half_step(dtype)
    # sums are taken in pieces of 32 rows, sections and across sections: far fewer than rows, but bounded by them
    err = (u + 2.0 ** -17 if dtype != torch.float32 else 2 * ref.E32) + ref.gamma(max(lens) // 16 + 512) + 90 * 2.0 ** -22
    got, st = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), ld.cuda(), offsets=torch.tensor(off, device="cuda"),
                                  scale=scale, return_state=True)
    ref.check("out", got, out, u * out.abs() + err * mag)
    fine = ref.gamma(max(lens) // 16 + 512) + 90 * 2.0 ** -22
    for s, (S, A) in enumerate(last):
        ref.check("state", st[s], S, fine * A)


def test_tables_beyond_32_bit_offsets():
    """More than 2^31 elements: the last, short series of a large table equals the same rows alone."""
    from tempo_amd import ops
    n, h, d, tail = 1_100_000, 16, 128, 150
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(n, h, d, generator=g, device="cuda", dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31
    k, v = q.roll(1, 2), q.roll(2, 2)
    off = torch.tensor([0, 700_000, n - tail, n], device="cuda")
    ld = torch.linspace(-0.5, -0.01, h).cuda()
    sub = [x[n - tail:].cpu() for x in (q, k, v)]
    want = ref.window_reference(*sub, sub[0], [0, tail], 40, 3, d ** -0.5)
    out, lse = ops.window_attention(q, k, v, 40, sinks=3, offsets=off, return_lse=True)
    ref.check("out", out[n - tail:], *want["out"])
    grads = ops.window_attention_grad(q, q, k, v, out, lse, 40, sinks=3, offsets=off)
    for name, x in zip(("dq", "dk", "dv"), grads):
        ref.check(name, x[n - tail:], *want[name])
    del out, lse, grads
    want = ref.decay_reference(*sub, ld.cpu(), [0, tail], d ** -0.5, dout=sub[0])
    out = ops.decay_attention(q, k, v, ld, offsets=off)
    ref.check("decay out", out[n - tail:], *want["out"])
    for name, x in zip(("dq", "dk", "dv"), ops.decay_attention_grad(q, q, k, v, ld, offsets=off)):
        ref.check("decay " + name, x[n - tail:], *want[name])


def test_cache_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements and a row count beyond 2^31: the last slot equals the same rows in a small
    cache."""
    from tempo_amd import ops
    slots, window, sinks, kv, d, h = 36, 65_000, 8, 8, 128, 16
    kc = torch.zeros(slots, window + sinks, kv, d, dtype=torch.bfloat16, device="cuda")
    assert kc.numel() > 2 ** 31
    vc = torch.zeros_like(kc)
    g = torch.Generator(device="cuda").manual_seed(3)
    kc[-1].normal_(generator=g), vc[-1].normal_(generator=g)
    q, k, v, _ = _dev(*_inputs(6, 1, h, kv, d, d, torch.bfloat16))
    length = torch.full((slots,), 2 ** 33 + 5, dtype=torch.int64, device="cuda")
    small = (kc[-1:].clone(), vc[-1:].clone(), length[-1:].clone())
    out = ops.window_attention_step(q, k, v, kc, vc, length, sinks=sinks, slots=torch.tensor([slots - 1], dtype=torch.int32, device="cuda"))
    alone = ops.window_attention_step(q, k, v, *small, sinks=sinks)
    assert torch.equal(out, alone) and torch.equal(kc[-1:], small[0]) and torch.equal(vc[-1:], small[1])
    assert int(length[-1]) == 2 ** 33 + 6 and int(length[0]) == 2 ** 33 + 5
    place = sinks + (2 ** 33 + 5 - sinks) % window
    assert torch.equal(kc[-1, place], k[0])
    keys, vals = (x[0].double().repeat_interleave(2, 1) for x in small[:2])
    p = torch.softmax((q[0].double()[None] * keys).sum(2) * d ** -0.5, 0)
    want = (p[:, :, None] * vals).sum(0)
    mag = (p[:, :, None] * vals.abs()).sum(0)
    ref.check("against all rows", out[0].cpu(), want.cpu(), (ref.half_step(torch.bfloat16) * want.abs() + 2.0 ** -14 * mag).cpu())


def test_moving_average_is_a_decay_attention():
    """The table's own path: order a shuffled table, take the series' offsets, and compare with ops.ema, whose taps are
    the same weights cut off after `window` rows."""
    import numpy as np
    from tempo_amd import ops
    rng = np.random.default_rng(4)
    n, n_keys, e, window = 5_000, 7, 0.2, 200
    key, ts = torch.from_numpy(rng.integers(0, n_keys, n).astype(np.int32)).cuda(), torch.from_numpy(rng.permutation(n) * 10 ** 6).cuda()
    x = torch.from_numpy(rng.normal(size=n)).cuda()
    perm, ema = ops.ema(key, ts, x, None, n_keys, window=window, exp_factor=e)
    order = ops.sort_order(key, ts, n_keys)
    assert torch.equal(order, perm)
    off = ops.series_offsets(key[order.long()].contiguous(), n_keys)
    assert off.tolist() == [0] + np.cumsum(np.bincount(key.cpu().numpy(), minlength=n_keys)).tolist()
    v = x[order.long()].float().reshape(n, 1, 1)
    one = torch.ones_like(v)
    got = ops.decay_attention(one, one, v, torch.tensor([math.log(1 - e)]).cuda(), offsets=off, scale=e).reshape(n)
    # taps beyond the window weigh (1 - e)^200 < 2^-64; 32-bit inputs, sums and powers
    bound = (2.0 ** -24 + 8 * ref.E32 + 90 * 2.0 ** -22 + ref.gamma(600)) * float(x.abs().max())
    assert float((got.double() - ema).abs().max()) <= bound


def test_refused_on_the_device():
    from tempo_amd import ops
    q, k, v, do = _dev(*_inputs(1, 10, 4, 2, 16, 16, torch.float32))
    ld = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="share"):
        ops.window_attention(q[:, :3], k, v, 5)
    with pytest.raises(ValueError, match="window"):
        ops.window_attention(q, k, v, 0)
    with pytest.raises(ValueError, match="window"):
        ops.window_attention(q, k, v, 2.5)
    with pytest.raises(ValueError, match="scale"):
        ops.window_attention(q, k, v, 5, scale=-1.0)
    with pytest.raises(NotImplementedError, match="sinks"):
        ops.window_attention(q, k, v, 5, sinks=33)
    with pytest.raises(TypeError, match="dtype"):
        ops.window_attention(q, k.bfloat16(), v, 5)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.window_attention(q.half(), k.half(), v.half(), 5)
    with pytest.raises(ValueError, match="rows"):
        ops.window_attention(q, k[:9], v, 5)
    with pytest.raises(ValueError, match="innermost"):
        ops.window_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, 5)
    with pytest.raises(ValueError, match="offsets"):
        ops.window_attention(q, k, v, 5, offsets=torch.tensor([0, 10], dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="CUDA"):
        ops.window_attention(q, k.cpu(), v, 5)
    big = torch.zeros(4, 1, 129, device="cuda")
    with pytest.raises(NotImplementedError, match="128"):
        ops.window_attention(big, big, big, 5)
    with pytest.raises(NotImplementedError, match="128"):
        ops.decay_attention(big, big, big, ld[:1])
    with pytest.raises(ValueError, match="heads"):
        ops.decay_attention(q, k, v, ld)
    with pytest.raises(ValueError, match="log_decay"):
        ops.decay_attention(q, q, q, ld[:2].contiguous())
    with pytest.raises(ValueError, match="state"):
        ops.decay_attention(q, q, q, ld, state=torch.zeros(2, 4, 16, 16, device="cuda"))
    cache = torch.zeros(3, 8, 2, 16, device="cuda")
    length = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="slots"):
        ops.window_attention_step(q, k, v, cache, cache.clone(), length)
    with pytest.raises(ValueError, match="window"):
        ops.window_attention_step(q[:3], k[:3], v[:3], cache, cache.clone(), length, sinks=8)
    with pytest.raises(ValueError, match="length"):
        ops.window_attention_step(q[:3], k[:3], v[:3], cache, cache.clone(), length[:2].contiguous())
    with pytest.raises(ValueError, match="repeat"):
        ops.window_attention_step(q[:3], k[:3], v[:3], cache[:1].expand(3, 8, 2, 16), cache, length)
    with pytest.raises(ValueError, match="gradient"):
        ops.decay_attention_step(q.requires_grad_(), q, q, ld, torch.zeros(10, 4, 16, 16, device="cuda"))


def _among_nan(t, lead, gap):
    """t [rows, heads, dim] on the device as a view whose every neighbour in memory is NaN: `lead` elements before, `gap`
    behind each head, gap + 3 more behind each row."""
    n, h, d = t.shape
    row = h * (d + gap) + gap + 3
    flat = torch.full((lead + n * row + 16,), math.nan, dtype=t.dtype, device="cuda")
    view = flat.as_strided((n, h, d), (row, d + gap, 1), lead)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dk,dv,lead,gap", [(5, 9, 1, 1), (40, 33, 3, 0), (64, 64, 1, 0), (127, 121, 5, 2), (128, 128, 7, 3),
                                            (16, 24, 2, 6)])
def test_neighbours_in_memory_do_not_show(dk, dv, lead, gap, dtype):
    """Rows at every odd place, NaN all around them: whole forms, their gradients, and steps over such rows and caches."""
    from tempo_amd import ops
    off = [0, 1, 131, 131, 333]
    n, h, window, sinks = off[-1], 2, 40, 3
    o = torch.tensor(off, device="cuda")
    q, k, v, do = _inputs(dk * 3 + dv, n, h, h, dk, dv, dtype)
    scale = dk ** -0.5
    qd, kd, vd, dod = [_among_nan(x.cuda(), lead, gap) for x in (q, k, v, do)]
    want = ref.window_reference(q, k, v, do, off, window, sinks, scale)
    out, lse = ops.window_attention(qd, kd, vd, window, sinks=sinks, offsets=o, return_lse=True)
    ref.check("out", out, *want["out"])
    for name, x in zip(("dq", "dk", "dv"), ops.window_attention_grad(dod, qd, kd, vd, _among_nan(out, lead, gap), lse, window,
                                                                      sinks=sinks, offsets=o)):
        ref.check(name, x, *want[name])
    ld = torch.tensor([-0.2, -0.003])
    decay = ref.decay_reference(q, k, v, ld, off, scale, dout=do)
    ref.check("decay out", ops.decay_attention(qd, kd, vd, ld.cuda(), offsets=o), *decay["out"])
    for name, x in zip(("dq", "dk", "dv"), ops.decay_attention_grad(dod, qd, kd, vd, ld.cuda(), offsets=o)):
        ref.check("decay " + name, x, *decay[name])
    # caches whose every row lies among NaN, filled from all rows but each series' last, which the step adds
    rows = window + sinks
    caches = []
    for d in (dk, dv):
        step = h * (d + gap) + gap + 3
        flat = torch.full((lead + 4 * rows * step + 16,), math.nan, dtype=dtype, device="cuda")
        caches.append(flat.as_strided((4, rows, h, d), (rows * step, step, d + gap, 1), lead))
    length = torch.zeros(4, dtype=torch.int64, device="cuda")
    old = torch.cat([torch.arange(off[i], max(off[i], off[i + 1] - 1)) for i in range(4)])
    o_old = torch.tensor(_offsets([max(0, off[i + 1] - off[i] - 1) for i in range(4)]), device="cuda")
    ops.window_cache_write(kd[old.cuda()], vd[old.cuda()], *caches, length, sinks=sinks, offsets=o_old)
    has = [0, 1, 3]
    last = torch.tensor([off[i + 1] - 1 for i in has])
    got = ops.window_attention_step(*[_among_nan(x[last.cuda()], lead, gap) for x in (qd, kd, vd)], *caches, length, sinks=sinks,
                                    slots=torch.tensor(has, dtype=torch.int32, device="cuda"))
    ref.check("step", got, want["out"][0][last], want["out"][1][last])
    for c, d in zip(caches, (dk, dv)):  # nothing between the rows was written
        flat = torch.as_strided(c, (lead + 4 * c.stride(0) + 16,), (1,), 0)
        kept = torch.ones_like(flat, dtype=torch.bool)
        torch.as_strided(kept, c.shape, c.stride(), lead).fill_(False)
        assert bool(flat[kept].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,dk,dv", [(3, 64, 48), (1, 128, 70), (5, 17, 32), (2, 100, 40)])
def test_decay_gradients_without_states(heads, dk, dv, dtype):
    """Long and short series, no state given or wanted: the walks that share a launch, over several sections."""
    from tempo_amd import ops
    off = _offsets([900, 1, 0, 64, 2500, 31, 700])
    n = off[-1]
    q, k, v, do = _inputs(heads + dk, n, heads, heads, dk, dv, dtype)
    ld = torch.linspace(-0.5, -0.001, heads)
    want = ref.decay_reference(q, k, v, ld, off, dk ** -0.5, dout=do)
    d, o = _dev(q, k, v, do), torch.tensor(off, device="cuda")
    for name, x in zip(("dq", "dk", "dv"), ops.decay_attention_grad(d[3], *d[:3], ld.cuda(), offsets=o)):
        ref.check(name, x, *want[name])


@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (24, 70)])
def test_values_that_are_not_finite_and_states_between_sections(dk, dv, dtype, bad):
    """Series over many sections, whose states are strung together: a bad element shows in its series from its row on
    (in gradients of keys and values up to it) and nowhere else."""
    from tempo_amd import ops
    off = _offsets([300, 1100, 40, 700])
    n, h, head = off[-1], 2, 1
    o = torch.tensor(off, device="cuda")
    clean = _inputs(dk + dv, n, h, h, dk, dv, dtype)
    ld = torch.tensor([-0.1, -0.02]).cuda()
    sid, _ = ref.series_of(n, off)
    at = torch.arange(n)

    def run(ts):
        q, k, v, do = _dev(*ts)
        res = [ops.decay_attention(q, k, v, ld, offsets=o), *ops.decay_attention_grad(do, q, k, v, ld, offsets=o)]
        return [x.float().cpu() for x in res]

    base = run(clean)
    for which, row in ((0, 700), (1, 310), (1, 1399), (2, 655), (2, 1500), (3, 900)):
        ts = [x.clone() for x in clean]
        ts[which][row, head, 5] = bad
        got = run(ts)
        behind, before = (sid == sid[row]) & (at >= row), (sid == sid[row]) & (at <= row)
        # out, dq, dk, dv: which rows each may differ in, and which of them are certainly not finite
        reach = {0: (at == row, at == at.new_tensor(-1), before, before), 1: (behind, behind, at == row, before),
                 2: (behind, behind, before, at == row), 3: (at == at.new_tensor(-1), at == row, before, before)}[which]
        for name, x, y, rows in zip(("out", "dq", "dk", "dv"), got, base, reach):
            where = torch.zeros(n, h, dtype=torch.bool)
            where[:, head] = rows
            assert torch.equal(x[~where], y[~where]), (which, row, name)
        if which < 3:
            assert not bool(got[0][reach[0]][:, head].isfinite().all(-1).any()), (which, row)
