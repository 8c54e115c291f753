"""Attention over series at the largest tables, at calls beside the usual ones, and what a reader of its results relies on."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import attention_cases as ref  # noqa: E402


def _repeats(x, want):
    """Whether x [n, ...] is `want` [period, ...] over and over, looked at in pieces."""
    period = want.shape[0]
    whole = x.reshape(x.shape[0] // period, period, -1)
    return all(bool((part == want.reshape(1, period, -1)).all()) for part in whole.split(1 << 14))


def test_window_gradients_of_a_table_where_row_and_window_pass_32_bits():
    """1.2 * 10^9 rows in series of fifty, "all earlier rows" for a window: the same 3200 rows over and over give the same
    results everywhere, those of the first ones."""
    from tempo_amd import ops
    period, times, m = 3200, 375_000, 50
    n = period * times
    assert n > 2 ** 30
    g = torch.Generator().manual_seed(7)
    small = [torch.randn(period, 1, 1, generator=g).to(torch.bfloat16) for _ in range(4)]
    want = ref.window_reference(*small, list(range(0, period + 1, m)), 2 ** 40, 0, 1.0)
    q, k, v, do = (x.cuda().repeat(times, 1, 1) for x in small)
    off = torch.arange(0, n + 1, m, device="cuda")
    out, lse = ops.window_attention(q, k, v, 2 ** 40, offsets=off, return_lse=True)
    ref.check("out", out[:period], *want["out"])
    assert _repeats(out, out[:period])
    for name, x in zip(("dq", "dk", "dv"), ops.window_attention_grad(do, q, k, v, out, lse, 2 ** 40, offsets=off)):
        ref.check(name, x[:period], *want[name])
        assert _repeats(x, x[:period]), name


def test_decay_attention_of_the_largest_table():
    """One series of 2^31 - 65537 rows: what a section's start and its length add up to passes 2^31 in the last section (of
    a walk towards the first row: at the first rows).  With a decay of exp(-1/2) four hundred rows are all that a row
    depends on (exp(-200) of a term is nothing)."""
    from tempo_amd import ops
    n, period, look, far = 2 ** 31 - 65537, 6_400, 3_000, 400
    g = torch.Generator().manual_seed(11)
    small = [torch.randn(period, 1, 1, generator=g).to(torch.bfloat16) for _ in range(4)]
    q, k, v, do = (x.cuda().repeat(-(-n // period), 1, 1)[:n] for x in small)
    ld = torch.tensor([-0.5])
    # what memory the results get holds NaN beforehand
    junk = [torch.full((n, 1, 1), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    del junk
    out, last = ops.decay_attention(q, k, v, ld.cuda(), scale=1.0, return_state=True)
    grads = ops.decay_attention_grad(do, q, k, v, ld.cuda(), scale=1.0)
    for a, b in ((0, look + far), (n - look - far, n)):
        part = [x[a:b].cpu() for x in (q, k, v, do)]
        want = ref.decay_reference(*part[:3], ld, [0, b - a], 1.0, dout=part[3])
        # (a row far enough from the cut has all that it depends on)
        behind, before = slice(0 if a == 0 else far, look + far), slice(0, look if a == 0 else look + far)
        for name, x, rows in (("out", out, behind), ("dq", grads[0], behind), ("dk", grads[1], before), ("dv", grads[2], before)):
            ref.check(f"{name} of rows {a}..", x[a:b][rows], want[name][0][rows], want[name][1][rows])
    ref.check("state", last, *want["state"])
    for x in (out, *grads):
        assert all(bool(part.isfinite().all()) for part in x.split(1 << 28))


def test_steps_tell_autograd_what_they_change():
    """A backward pass whose saved state or rows a step has changed since raises, as with torch's own in-place operations;
    with another state's step, and in inference mode, calls go on as ever."""
    from tempo_amd import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = lambda n=6: torch.randn(n, 2, 16, generator=g, device="cuda")  # noqa: E731
    q, k, v = rows().requires_grad_(), rows(), rows()
    ld = torch.tensor([-0.1, -0.2], device="cuda")
    state, other = torch.zeros(1, 2, 16, 16, device="cuda"), torch.zeros(1, 2, 16, 16, device="cuda")
    out = ops.decay_attention(q, k, v, ld, state=state)
    ops.decay_attention_step(rows(1), rows(1), rows(1), ld, other)
    out.sum().backward(retain_graph=True)
    ops.decay_attention_step(rows(1), rows(1), rows(1), ld, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # rows of a cache, read in place as keys and values of the whole form
    kc, vc = rows(8).reshape(2, 4, 2, 16), rows(8).reshape(2, 4, 2, 16)
    length = torch.tensor([4, 4], device="cuda")
    writes = {
        "step": lambda: ops.window_attention_step(rows(2), rows(2), rows(2), kc, vc, length),
        "write": lambda: ops.window_cache_write(rows(4), rows(4), kc, vc, length, offsets=torch.tensor([0, 1, 4], device="cuda")),
    }
    for write in writes.values():
        for keys, values in ((kc[0], rows(4)), (rows(4), vc[0])):
            out = ops.window_attention(rows(4).requires_grad_(), keys, values, 3)
            counted = length._version
            write()
            assert length._version > counted
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()
    with torch.inference_mode():
        made = torch.zeros(1, 2, 16, 16, device="cuda")
        ops.decay_attention_step(rows(1), rows(1), rows(1), ld, made)
        ops.decay_attention_step(rows(1), rows(1), rows(1), ld, state)
        for write in writes.values():
            write()


def test_decays_held_as_a_parameter():
    """Without gradients such a decay is as good as any; where one is wanted it is refused, at every entry."""
    from tempo_amd import ops
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, do = (torch.randn(40, 2, 16, generator=g, device="cuda") for _ in range(4))
    ld = torch.nn.Parameter(torch.tensor([-0.1, -0.02], device="cuda"))
    state = torch.zeros(40, 2, 16, 16, device="cuda")
    with torch.no_grad():
        assert torch.equal(ops.decay_attention(q, k, v, ld), ops.decay_attention(q, k, v, ld.detach()))
        for a, b in zip(ops.decay_attention_grad(do, q, k, v, ld), ops.decay_attention_grad(do, q, k, v, ld.detach())):
            assert torch.equal(a, b)
        ops.decay_attention_step(q, k, v, ld, state)
    for call in (lambda: ops.decay_attention(q, k, v, ld), lambda: ops.decay_attention_grad(do, q, k, v, ld),
                 lambda: ops.decay_attention(q.clone().requires_grad_(), k, v, ld)):
        with pytest.raises(ValueError, match="log_decay has no gradient"):
            call()
    with pytest.raises(ValueError, match="gradient"):
        ops.decay_attention_step(q, k, v, ld, state)
    # detached it trains the rest
    leaf = q.clone().requires_grad_()
    ops.decay_attention(leaf, k, v, ld.detach()).backward(do)
    assert torch.equal(leaf.grad, ops.decay_attention_grad(do, q, k, v, ld.detach())[0]) and ld.grad is None


@pytest.mark.parametrize("dtype, few", [(torch.bfloat16, 512), (torch.float32, 256)], ids=["bf16", "f32"])
def test_one_long_series_among_empty_ones(dtype, few):
    """Sections of a long series are walked side by side however many empty series there are besides; up to `few` rows
    every block walks what it needs in one launch.  Either way results are the definition's."""
    from tempo_amd import _lib, ops
    h, dk, dv = 2, 24, 40
    ld = torch.tensor([-0.1, -0.004])
    for n, launches in ((few - 1, 1), (few, 1), (few + 1, 3), (1500, 3), (4096, 3)):
        g = torch.Generator().manual_seed(n)
        q, k, v, do = (torch.randn(n, h, d, generator=g).to(dtype) for d in (dk, dk, dv, dv))
        off = [0] * 60 + [n] * 61
        d, o = [x.cuda() for x in (q, k, v, do)], torch.tensor(off, device="cuda")
        want = ref.decay_reference(q, k, v, ld, off, dk ** -0.5, dout=do)
        _lib.profile_enable(True)
        try:
            _lib.profile_reset()
            out = ops.decay_attention(*d[:3], ld.cuda(), offsets=o)
            torch.cuda.synchronize()
            assert len(_lib.profile_read()) == launches, n
        finally:
            _lib.profile_enable(False)
        ref.check("out", out, *want["out"])
        for name, x in zip(("dq", "dk", "dv"), ops.decay_attention_grad(d[3], *d[:3], ld.cuda(), offsets=o)):
            ref.check(name, x, *want[name])


@pytest.mark.parametrize("d, heads, kv, sinks", [(32, 2, 2, 0), (64, 4, 2, 0), (128, 4, 2, 4)])
@pytest.mark.parametrize("window", [60, 64, 65, 70, 600])
def test_errors_of_bfloat16_training_do_not_depend_on_the_window(window, d, heads, kv, sinks):
    """Root mean square errors against 64 bits, in units of what rounding the exact result once gives.  Independent roundings
    add in squares: the result alone is 1, one more of the same size (an operand of a product that is rounded once, as
    the weights are for out and dv) sqrt(2), two more sqrt(3).  dS is not rounded to eight bits anywhere, so that dq and
    dk have the result's rounding and, smaller than that over sixty rows, that of out within do.o."""
    from tempo_amd import ops
    n = 1500
    q, k, v, do = (torch.randn(n, h, d, generator=torch.Generator().manual_seed(d + i)).bfloat16()
                   for i, h in enumerate((heads, kv, kv, heads)))
    off = [0, 700, n]
    want = ref.window_reference(q, k, v, do, off, window, sinks, d ** -0.5)
    a, o = [x.cuda() for x in (q, k, v, do)], torch.tensor(off, device="cuda")
    out, lse = ops.window_attention(*a[:3], window, sinks=sinks, offsets=o, return_lse=True)
    got = (out, *ops.window_attention_grad(a[3], *a[:3], out, lse, window, sinks=sinks, offsets=o))
    for name, x, most in zip(("out", "dq", "dk", "dv"), got, (1.5, 1.2, 1.2, 1.5)):
        exact = want[name][0]
        alone = float((exact.bfloat16().double() - exact).norm())
        assert float((x.cpu().double() - exact).norm()) < most * alone, name


def _recurrence(q, k, v, ld, off, scale, state, do=None, dstate=None):
    """The definition row by row in 64 bits: {name: (value, sum of magnitudes)} of out, state, dq, dk, dv, dstate."""
    n, h, dk = q.shape
    lam = torch.exp(ld.double())[:, None, None]
    res = {}
    for which, of in (("value", lambda x: x), ("size", torch.abs)):
        Q, K, V, S0 = (of(x.double()) for x in (q, k, v, state))
        out, last = torch.zeros(n, h, v.shape[2], dtype=torch.float64), torch.zeros_like(S0)
        dq, dk_, dv_ = torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V)
        ds = torch.zeros_like(S0)
        for s in range(len(off) - 1):
            S = S0[s]
            for i in range(off[s], off[s + 1]):
                S = lam * S + K[i, :, :, None] * V[i, :, None, :]
                out[i] = (Q[i, :, :, None] * S).sum(1) * scale
                if do is not None:
                    dq[i] = (S * of(do[i].double())[:, None, :]).sum(2) * scale
            last[s] = S
            if do is None:
                continue
            G = of(dstate[s].double())  # dG/dS behind row i: what the state there is worth
            for i in range(off[s + 1] - 1, off[s] - 1, -1):
                G = G + scale * Q[i, :, :, None] * of(do[i].double())[:, None, :]
                dk_[i] = (G * V[i, :, None, :]).sum(2)
                dv_[i] = (G * K[i, :, :, None]).sum(1)
                G = lam * G
            ds[s] = G
        res[which] = dict(out=out, state=last, dq=dq, dk=dk_, dv=dv_, dstate=ds)
    return {name: (res["value"][name], res["size"][name]) for name in res["value"]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_states_strung_together_over_several_sweeps(dtype):
    """40 000 rows of one head make 625 sections, of which a sweep of the scan takes 256; one series reaches over 560 of
    them, slowly fading, with a state before it and a gradient of the one behind it."""
    from tempo_amd import ops
    off, h, dk, dv, scale = [0, 1_900, 37_900, 37_900, 40_000], 1, 16, 12, 0.25
    n = off[-1]
    g = torch.Generator().manual_seed(17)
    q, k, v, do = (torch.randn(n, h, d, generator=g).to(dtype) for d in (dk, dk, dv, dv))
    state, dstate = (torch.randn(4, h, dk, dv, generator=g) for _ in range(2))
    ld = torch.tensor([-2e-5])
    want = _recurrence(q, k, v, ld, off, scale, state, do, dstate)
    a, o = [x.cuda() for x in (q, k, v, do)], torch.tensor(off, device="cuda")
    out, last = ops.decay_attention(*a[:3], ld.cuda(), offsets=o, scale=scale, state=state.cuda(), return_state=True)
    grads = ops.decay_attention_grad(a[3], *a[:3], ld.cuda(), offsets=o, scale=scale, state=state.cuda(), dstate=dstate.cuda(),
                                     return_dstate=True)
    got = dict(zip(("out", "state", "dq", "dk", "dv", "dstate"), (out, last, *grads)))
    # rows in parts of 32, sections of 64, 625 sections: no term passes through more sums than these; powers of the decay as
    # in the definition's bounds; bfloat16 terms are rounded once, those of a state to 2^-17
    u = ref.half_step(dtype)
    sums = ref.gamma(32 + 64 + 2 * 625 + dk) + 8 * ref.E32 + 90 * 2.0 ** -22
    term = u + 2.0 ** -17 if dtype != torch.float32 else 2 * ref.E32
    for name, x in got.items():
        exact, size = want[name]
        fine = name in ("state", "dstate")
        ref.check(name, x, exact, (0 if fine else u * exact.abs()) + (sums + (0 if fine else term)) * size)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_gradients_that_depend_on_a_value_that_is_not_finite(dtype, bad):
    """One bad element of an input in turn.  Where a gradient is a sum that has it, or a weight made of it, as a term, the
    gradient is not finite: of the window's, dq of the rows whose weights it makes, dk and dv of the keys that these see, the
    bad element of dv for dout; of the decay's, every sum with it as a factor.  (A key whose score is minus infinity has the
    weight zero: the row's other weights are as finite as ever, and zero times the key is not.)"""
    from tempo_amd import ops
    lens, window, sinks, h, d, head, e = [60, 300, 45], 20, 2, 2, 32, 1, 7
    off = [0, 60, 360, 405]
    n = off[-1]
    o = torch.tensor(off, device="cuda")
    g = torch.Generator().manual_seed(78)
    clean = [torch.randn(n, h, d, generator=g).to(dtype) for _ in range(4)]
    ld = torch.tensor([-0.1, -0.02]).cuda()
    seen = ref.window_mask(n, off, window, sinks)
    sid, pos = ref.series_of(n, off)
    past = (sid[:, None] == sid[None]) & (pos[None] <= pos[:, None])
    none = torch.zeros(n, dtype=torch.bool)
    for which, row in ((0, 100), (0, 61), (1, 60), (1, 61), (1, 200), (2, 60), (2, 201), (3, 150), (3, 62)):
        ts = [x.clone() for x in clean]
        ts[which][row, head, e] = bad
        q, k, v, do = (x.cuda() for x in ts)
        out, lse = ops.window_attention(q, k, v, window, sinks=sinks, offsets=o, return_lse=True)
        grads = [x.float().cpu()[:, head] for x in ops.window_attention_grad(do, q, k, v, out, lse, window, sinks=sinks, offsets=o)]
        at = none.clone()
        at[row] = True
        rows = at if which in (0, 3) else seen[:, row]  # query rows with a weight, or a gradient of one, that is not finite
        if which == 1:
            assert not bool(grads[0][rows][:, e].isfinite().any()), (which, row)
            rows = rows & ~(ts[0][:, head, e].float() * bad == -float("inf"))
        keys = seen[rows].any(0)
        for i, (name, x) in enumerate(zip(("dq", "dk", "dv"), grads)):
            touched = rows if i == 0 else keys
            if which == 2 and i == 2:
                continue  # (weights do not depend on v: dv stays finite)
            part = x[touched][:, e] if i == 2 and which == 3 else x[touched]
            assert not bool(part.isfinite().any()), (name, which, row)
        # S_i of rows behind, G_i of rows before: element e is a row or a column of them
        grads = [x.float().cpu()[:, head] for x in ops.decay_attention_grad(do, q, k, v, ld, offsets=o)]
        behind, before = past[:, row], past[row]
        bad_part = {  # input: (gradient, rows, elements)
            0: [(1, before, [e]), (2, before, slice(None))],
            1: [(0, behind, [e]), (2, at, slice(None))],
            2: [(0, behind, slice(None)), (1, at, slice(None))],
            3: [(0, at, slice(None)), (1, before, slice(None)), (2, before, [e])],
        }[which]
        for i, rows, elems in bad_part:
            assert not bool(grads[i][rows][:, elems].isfinite().any()), ("decay", i, which, row)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [1e-39, 2.0 ** -100, 1e-3, 1e20])
def test_gradients_of_states_at_every_scale(scale, dtype):
    """The gradient of a returned state passes the backward walk as it is: a scale that is small, or no normal number, does
    not make it overflow on its way."""
    from tempo_amd import ops
    off, h, dk, dv = [0, 40, 40, 400], 2, 24, 40
    n = off[-1]
    g = torch.Generator().manual_seed(19)
    q, k, v, do = (torch.randn(n, h, d, generator=g).to(dtype) for d in (dk, dk, dv, dv))
    state, dstate = (torch.randn(3, h, dk, dv, generator=g) for _ in range(2))
    dstate *= 2.0 ** 40
    ld = torch.tensor([-0.1, -0.004])
    scale = float(torch.tensor(scale))  # (as the kernels take it)
    want = ref.decay_reference(q, k, v, ld, off, scale, state, do, dstate)
    a, o = [x.cuda() for x in (q, k, v, do)], torch.tensor(off, device="cuda")
    grads = ops.decay_attention_grad(a[3], *a[:3], ld.cuda(), offsets=o, scale=scale, state=state.cuda(), dstate=dstate.cuda(),
                                     return_dstate=True)
    for name, x in zip(("dk", "dv", "dstate"), grads[1:]):
        ref.check(name, x, *want[name])
    if scale >= 2.0 ** -100:  # (below, products of two small factors are no normal numbers)
        ref.check("dq", grads[0], *want["dq"])


def test_more_series_than_a_launch_has_blocks():
    """States of 2^24 + 100 series, nearly all of them without rows: each keeps its own, or zeros without one."""
    from tempo_amd import ops
    ns, h, d = 2 ** 24 + 100, 1, 2
    counts = torch.zeros(ns, dtype=torch.int64, device="cuda")
    full = torch.tensor([0, 5, 65_535, 65_536, 2 ** 24 - 1, 2 ** 24, ns - 1], device="cuda")
    counts[full] = 3
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    n = int(off[-1])
    g = torch.Generator(device="cuda").manual_seed(23)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda") for _ in range(3))
    ld = torch.tensor([-0.5], device="cuda")
    state = torch.randn(ns, h, d, d, generator=g, device="cuda")
    empty = torch.ones(ns, dtype=torch.bool, device="cuda")
    empty[full] = False
    _, last = ops.decay_attention(q, k, v, ld, offsets=off, state=state, return_state=True)
    assert torch.equal(last[empty], state[empty])
    small = torch.arange(0, n + 1, 3, device="cuda")
    assert torch.equal(last[full], ops.decay_attention(q, k, v, ld, offsets=small, state=state[full].contiguous(), return_state=True)[1])
    _, last = ops.decay_attention(q, k, v, ld, offsets=off, return_state=True)
    assert not bool(last[empty].any())


def test_sizes_beyond_32_bits_are_refused():
    """Numbers that the library is told in 32 bits do not come out as others."""
    from tempo_amd import ops
    a = torch.zeros(3, 1, 8, device="cuda")
    ld = torch.zeros(1, device="cuda")
    for sinks in (2 ** 32, 2 ** 32 + 2, 2 ** 70):
        with pytest.raises(NotImplementedError, match="sinks"):
            ops.window_attention(a, a, a, 5, sinks=sinks)
    wide = torch.zeros(3, 1, 1, device="cuda").expand(3, 2 ** 32 + 1, 1)
    for call in (lambda: ops.window_attention(wide, wide, wide, 5), lambda: ops.window_attention(wide, a[..., :1], a[..., :1], 5),
                 lambda: ops.decay_attention(wide, wide, wide, ld)):
        with pytest.raises(NotImplementedError, match="heads"):
            call()
    long = torch.empty(2 ** 32 + 8, device="cuda", dtype=torch.bfloat16).reshape(1, 1, -1)
    with pytest.raises(NotImplementedError, match="elements"):
        ops.window_attention(long, long, long, 5)
    cache = long.reshape(1, -1, 1, 1)  # 2^32 + 8 rows
    b = torch.zeros(1, 1, 1, device="cuda", dtype=torch.bfloat16)
    length = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="window"):
        ops.window_attention_step(b, b, b, cache, cache, length)
    with pytest.raises(ValueError, match="window"):
        ops.window_cache_write(b, b, cache, cache, length)
    del cache, long
    some = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, 1, 1, device="cuda")
    state = torch.empty(2 ** 31, 1, 1, 1, device="cuda")
    with pytest.raises(ValueError, match="slots"):
        ops.decay_attention_step(one, one, one, ld, state, slots=some)
    with pytest.raises(ValueError, match="series"):
        ops.window_attention(one, one, one, 5, offsets=torch.empty(2 ** 31, dtype=torch.int64, device="cuda"))


def test_a_table_captured_from_its_keys_on():
    """Offsets from the key column and both operators in one graph, replayed over other tables of the same size with eager
    work in between."""
    from tempo_amd import ops
    n, n_keys, h, d = 900, 12, 2, 32
    g = torch.Generator(device="cuda").manual_seed(29)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda") for _ in range(3))
    ld = torch.tensor([-0.1, -0.01], device="cuda")
    key = torch.zeros(n, dtype=torch.int32, device="cuda")
    tables = [torch.sort(torch.randint(0, n_keys, (n,), generator=g, device="cuda", dtype=torch.int32)).values for _ in range(4)]

    def step():
        off = ops.series_offsets(key, n_keys)
        return off, ops.window_attention(q, k, v, 20, sinks=1, offsets=off), ops.decay_attention(q, k, v, ld, offsets=off)

    want = []
    for t in tables:
        key.copy_(t)
        want.append([x.clone() for x in step()])
        assert want[-1][0].tolist() == [0] + torch.bincount(t.long(), minlength=n_keys).cumsum(0).tolist()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in (0, 1, 2, 3, 1, 0):
        key.copy_(tables[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
        ops.key_counts(tables[2], n_keys)
        torch.randn(1000, device="cuda").sum().item()


def test_window_attention_of_the_largest_table():
    """2^31 - 65537 rows in series of a million, a few rows of window and two that stay visible: the last rows' results are
    those of a short series that holds what they see."""
    from tempo_amd import ops
    n, m, window, sinks, look = 2 ** 31 - 65537, 1_000_000, 5, 2, 3_000
    period = 6_400
    g = torch.Generator().manual_seed(31)
    small = [torch.randn(period, 1, 1, generator=g).to(torch.bfloat16) for _ in range(4)]
    q, k, v, do = (x.cuda().repeat(-(-n // period), 1, 1)[:n] for x in small)
    off = torch.cat([torch.arange(0, n, m, device="cuda"), torch.tensor([n], device="cuda")])
    start = (n - 1) // m * m
    junk = [torch.full((n, 1, 1), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    del junk
    out, lse = ops.window_attention(q, k, v, window, sinks=sinks, offsets=off, return_lse=True)
    grads = ops.window_attention_grad(do, q, k, v, out, lse, window, sinks=sinks, offsets=off)
    rows = torch.cat([torch.arange(start, start + sinks), torch.arange(n - look, n)]).cuda()
    want = ref.window_reference(*(x[rows].cpu() for x in (q, k, v, do)), [0, len(rows)], window, sinks, 1.0)
    whole = slice(sinks + window, None)  # (before them the short series lacks rows; its first rows' dk, dv too)
    for name, x in (("out", out), ("lse", lse), *zip(("dq", "dk", "dv"), grads)):
        ref.check(name, x[rows][whole], want[name][0][whole], want[name][1][whole])
    for x in (out, *grads):
        assert all(bool(part.isfinite().all()) for part in x.split(1 << 28))


def test_steps_of_the_most_rows():
    """Close to as many rows x heads as a step takes: every row is added and read."""
    from tempo_amd import ops
    n, h, d = 2 ** 20 - 1, 16, 4
    g = torch.Generator(device="cuda").manual_seed(37)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda") for _ in range(3))
    state = torch.randn(n, h, d, d, generator=g, device="cuda")
    ld = torch.linspace(-0.5, -0.01, h, device="cuda")
    s = state.double() * torch.exp(ld.double())[:, None, None] + k.double()[..., None] * v.double()[..., None, :]
    size = state.double().abs() + k.double().abs()[..., None] * v.double().abs()[..., None, :]
    out = ops.decay_attention_step(q, k, v, ld, state, scale=0.5)
    # (a sum of two, its power off by three steps at most; then four terms, the scale and a rounding)
    assert bool(((state - s).abs() <= 6 * ref.E32 * size).all())
    want = (q.double()[..., None] * s).sum(2) * 0.5
    assert bool(((out - want).abs() <= 14 * ref.E32 * (q.double().abs()[..., None] * size).sum(2) * 0.5).all())
    del state, s, size, want, out
    h, window = 32, 3
    q = torch.randn(n, h, d, generator=g, device="cuda")
    k, v = (torch.randn(n, 1, d, generator=g, device="cuda") for _ in range(2))
    kc, vc = (torch.randn(n, window, 1, d, generator=g, device="cuda") for _ in range(2))
    length = torch.arange(n, device="cuda") % 7
    seen = (length + 1).clamp(max=window)
    keys, vals = kc.clone(), vc.clone()
    at = torch.arange(n, device="cuda")
    keys[at, length % window], vals[at, length % window] = k, v
    out = ops.window_attention_step(q, k, v, kc, vc, length, scale=0.5)
    assert torch.equal(kc, keys) and torch.equal(vc, vals) and torch.equal(length, at % 7 + 1)
    for a in range(0, n, 1 << 18):
        b = slice(a, a + (1 << 18))
        scores = (q[b].double()[:, :, None] * keys[b, None, :, 0].double()).sum(3) * 0.5
        on = torch.arange(window, device="cuda") < seen[b, None, None]
        p = torch.softmax(scores.masked_fill(~on, -float("inf")), 2)
        want = (p[..., None] * vals[b, None, :, 0].double()).sum(2)
        size = (p[..., None] * vals[b, None, :, 0].double().abs()).sum(2)
        # weights: a score of four terms, its scale, the change of base and the exponential's two steps
        rel = 16 * ref.E32 * (1 + scores.abs().amax(2, keepdim=True)) + 8 * ref.E32
        assert bool(((out[b] - want).abs() <= 2 * rel * size + ref.E32 * want.abs()).all())
