"""Attention over series without a GPU: the gradients' formulas against differences, and what is refused before
anything is launched."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import attention_cases as ref  # noqa: E402


def _differences(f, t, picks, step=1e-6):
    """Central differences of f() at some elements of t."""
    out = []
    flat = t.view(-1)
    for i in picks:
        keep = flat[i].item()
        flat[i] = keep + step
        hi = f()
        flat[i] = keep - step
        lo = f()
        flat[i] = keep
        out.append((hi - lo) / (2 * step))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("window, sinks", [(1, 0), (3, 0), (4, 2), (100, 1)])
def test_window_gradients_against_differences(window, sinks):
    g = torch.Generator().manual_seed(window)
    off, n, h, kv, d = [1, 8, 8, 20], 22, 4, 2, 3
    # float64 inputs: the reference computes in 64 bits whatever it is given, differences need the inputs in them too
    make = lambda a, b: torch.randn(n, a, b, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, do = make(h, d), make(kv, d), make(kv, d), make(h, d)
    ref_of = lambda: ref.window_reference(q, k, v, do, off, window, sinks, 0.7)  # noqa: E731
    want = ref_of()
    f = lambda: float((ref_of()["out"][0] * do).sum())  # noqa: E731
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        picks = torch.randperm(t.numel(), generator=g)[:12].tolist()
        assert torch.allclose(_differences(f, t, picks), want[name][0].reshape(-1)[picks], rtol=1e-6, atol=1e-8)


def test_decay_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    off, n, h, dk, dv = [2, 9, 9, 21], 22, 2, 3, 4
    make = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, do = make(n, h, dk), make(n, h, dk), make(n, h, dv), make(n, h, dv)
    st, ds = make(3, h, dk, dv), make(3, h, dk, dv)
    ld = torch.tensor([-0.3, -1.5], dtype=torch.float64)
    ref_of = lambda: ref.decay_reference(q, k, v, ld, off, 0.6, st, do, ds)  # noqa: E731
    want = ref_of()

    def f():
        r = ref_of()
        return float((r["out"][0] * do).sum() + (r["state"][0] * ds).sum())

    for name, t in (("dq", q), ("dk", k), ("dv", v), ("dstate", st)):
        picks = torch.randperm(t.numel(), generator=g)[:12].tolist()
        assert torch.allclose(_differences(f, t, picks), want[name][0].reshape(-1)[picks], rtol=1e-6, atol=1e-8)


def test_decay_reference_is_the_recurrence():
    g = torch.Generator().manual_seed(2)
    n, h, dk, dv = 30, 2, 3, 4
    q, k, v = (torch.randn(n, h, d, generator=g, dtype=torch.float64) for d in (dk, dk, dv))
    st = torch.randn(2, h, dk, dv, generator=g, dtype=torch.float64)
    ld = torch.tensor([-0.3, -math.inf], dtype=torch.float64)
    off = [0, 12, 30]
    want = ref.decay_reference(q, k, v, ld, off, 0.5, st)
    for s in range(2):
        S = st[s].clone()
        for i in range(off[s], off[s + 1]):
            S = torch.exp(ld)[:, None, None] * S + k[i, :, :, None] * v[i, :, None, :]
            assert torch.allclose((q[i, :, :, None] * S).sum(1) * 0.5, want["out"][0][i], atol=1e-12)
        assert torch.allclose(S, want["state"][0][s], atol=1e-12)


def _struct(cls, **kw):
    a = cls()
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_argument_errors_need_no_gpu():
    from tempo_amd import _lib
    h = _lib.lib()
    rows = _lib.RowsRef(4096, 64, 16)
    good = dict(n=10, n_series=1, type=0, heads=4, kv_heads=2, dim_k=16, dim_v=16, window=5, sinks=1, scale=0.25, q=rows,
                k=rows, v=rows, out=rows)
    cases = [(dict(n=-1), -1, b"row count"), (dict(n=2 ** 31), -1, b"row count"), (dict(type=7), -4, b"type"),
             (dict(heads=0), -1, b"heads"), (dict(heads=3), -1, b"multiple"), (dict(dim_k=0), -1, b"head sizes"),
             (dict(dim_v=129), -4, b"128"), (dict(window=0), -1, b"window"), (dict(sinks=-1), -1, b"sinks"),
             (dict(sinks=33), -4, b"sinks"), (dict(scale=0.0), -1, b"scale"), (dict(scale=math.inf), -1, b"scale"),
             (dict(scale=math.nan), -1, b"scale"), (dict(n_series=-1), -1, b"series"), (dict(n_series=5), -1, b"series"),
             (dict(q=_lib.RowsRef()), -1, b"null"), (dict(k=_lib.RowsRef(4096, 8, 16)), -4, b"stride"),
             (dict(v=_lib.RowsRef(4096, 2 ** 22, 16)), -4, b"stride")]
    for change, rc, text in cases:
        a = _struct(_lib.WindowAttentionArgs, **{**good, **change})
        assert h.tmp_window_attention(C.byref(a), None) == rc, change
        assert text in h.tmp_last_error(), (change, h.tmp_last_error())
    assert h.tmp_window_attention(None, None) == -1
    a = _struct(_lib.WindowAttentionArgs, **good)
    assert h.tmp_window_attention_grad(C.byref(a), None, 0, None) == -1 and b"null" in h.tmp_last_error()
    for name in ("dout", "dq", "dk", "dv"):
        setattr(a, name, rows)
    a.lse = 4096
    assert h.tmp_window_attention_grad(C.byref(a), None, 0, None) == -2 and b"workspace" in h.tmp_last_error()
    assert h.tmp_window_attention_grad_workspace_bytes(C.byref(a)) >= 10 * 4 * 4
    assert h.tmp_window_attention(C.byref(_struct(_lib.WindowAttentionArgs, **{**good, "n": 0})), None) == 0

    good = dict(n=10, n_series=1, type=1, heads=4, dim_k=16, dim_v=16, scale=0.25, log_decay=4096, q=rows, k=rows, v=rows, out=rows)
    cases = [(dict(n=-1), -1, b"row count"), (dict(type=2), -4, b"type"), (dict(heads=0), -1, b"heads"),
             (dict(dim_k=200), -4, b"128"), (dict(dim_v=0), -1, b"head sizes"), (dict(scale=-1.0), -1, b"scale"),
             (dict(log_decay=None), -1, b"null"), (dict(n_series=2), -1, b"series")]
    for change, rc, text in cases:
        a = _struct(_lib.DecayAttentionArgs, **{**good, **change})
        assert h.tmp_decay_attention(C.byref(a), None, 0, None) == rc, change
        assert text in h.tmp_last_error(), (change, h.tmp_last_error())
    a = _struct(_lib.DecayAttentionArgs, **good)
    assert h.tmp_decay_attention(C.byref(a), None, 0, None) == -2
    assert h.tmp_decay_attention_grad(C.byref(a), None, 0, None) == -1
    assert h.tmp_decay_attention_workspace_bytes(C.byref(a)) > 0

    cache = _lib.CacheRef(4096, 640, 64, 16)
    good = dict(n=2, n_slots=3, slots=4096, type=0, heads=4, kv_heads=2, dim_k=16, dim_v=16, window=8, sinks=1, scale=0.25, q=rows,
                k=rows, v=rows, out=rows, k_cache=cache, v_cache=cache, length=4096)
    cases = [(dict(n=-1), -1, b"row count"), (dict(slots=None, n=4), -1, b"slots"), (dict(window=0), -1, b"window"),
             (dict(sinks=40), -4, b"sinks"), (dict(heads=5), -1, b"multiple"), (dict(length=None), -1, b"null"),
             (dict(scale=0.0), -1, b"scale")]
    for change, rc, text in cases:
        a = _struct(_lib.WindowAttentionStepArgs, **{**good, **change})
        assert h.tmp_window_attention_step(C.byref(a), None, 0, None) == rc, change
        assert text in h.tmp_last_error(), (change, h.tmp_last_error())
    a = _struct(_lib.WindowAttentionStepArgs, **good)
    assert h.tmp_window_attention_step(C.byref(a), None, 0, None) == -2
    a = _struct(_lib.DecayAttentionStepArgs, n=2, n_slots=1, type=0, heads=1, dim_k=8, dim_v=8, scale=1.0)
    assert h.tmp_decay_attention_step(C.byref(a), None) == -1 and b"slots" in h.tmp_last_error()
    a = _struct(_lib.WindowCacheWriteArgs, n=4, n_series=2, type=0, kv_heads=1, dim_k=8, dim_v=8, window=4, n_slots=4)
    assert h.tmp_window_cache_write(C.byref(a), None) == -1 and b"series" in h.tmp_last_error()


def test_what_a_step_cannot_take():
    """Rows that would look through too many slots, arrays that do not lie at multiples of their type's size, scales."""
    from tempo_amd import _lib
    h = _lib.lib()
    rows, cache = _lib.RowsRef(4096, 64, 16), _lib.CacheRef(4096, 640, 64, 16)
    many = 65537
    a = dict(n=many, n_slots=many, slots=4096, type=0, heads=1, dim_k=16, dim_v=16, scale=1.0, log_decay=4096, q=rows, k=rows,
             v=rows, out=rows, state=4096)
    for change, rc, text in [({}, -4, b"65536"), (dict(n=2, scale=0.0), -1, b"scale"), (dict(n=2, scale=math.nan), -1, b"scale"),
                             (dict(n=2, k=_lib.RowsRef(4097, 64, 16)), -4, b"aligned"),
                             (dict(n=2, type=1, v=_lib.RowsRef(4098, 64, 16)), -4, b"aligned")]:
        assert h.tmp_decay_attention_step(C.byref(_struct(_lib.DecayAttentionStepArgs, **{**a, **change})), None) == rc, change
        assert text in h.tmp_last_error(), (change, h.tmp_last_error())
    a = dict(n=many, n_slots=many, slots=4096, type=0, heads=1, kv_heads=1, dim_k=16, dim_v=16, window=8, sinks=1, scale=1.0,
             q=rows, k=rows, v=rows, out=rows, k_cache=cache, v_cache=cache, length=4096)
    assert h.tmp_window_attention_step(C.byref(_struct(_lib.WindowAttentionStepArgs, **a)), None, 0, None) == -4
    assert b"65536" in h.tmp_last_error()
    a = dict(n=4, n_series=many, offsets=4096, n_slots=many, slots=4096, type=0, kv_heads=1, dim_k=16, dim_v=16, window=8, k=rows,
             v=rows, k_cache=cache, v_cache=cache, length=4096)
    assert h.tmp_window_cache_write(C.byref(_struct(_lib.WindowCacheWriteArgs, **a)), None) == -4
    assert b"65536" in h.tmp_last_error()
    a.update(n_series=2, v_cache=_lib.CacheRef(4097, 640, 64, 16))
    assert h.tmp_window_cache_write(C.byref(_struct(_lib.WindowCacheWriteArgs, **a)), None) == -4
    assert b"aligned" in h.tmp_last_error()


def test_host_tensors_are_refused():
    from tempo_amd import ops
    t = torch.zeros(4, 2, 8)
    with pytest.raises(TypeError, match="no CPU path"):
        ops.window_attention(t, t, t, 3)
    with pytest.raises(TypeError, match="no CPU path"):
        ops.decay_attention(t, t, t, torch.zeros(2))
    with pytest.raises(TypeError, match="no CPU path"):
        ops.decay_attention_step(t, t, t, torch.zeros(2), torch.zeros(4, 2, 8, 8))


def test_one_section_carries_nothing():
    from tempo_amd import _lib
    h = _lib.lib()
    a = _struct(_lib.DecayAttentionArgs, n=64, heads=4096, dim_k=128, dim_v=128, dout=_lib.RowsRef(4096, 64, 16))
    assert h.tmp_decay_attention_workspace_bytes(C.byref(a)) < 1 << 12
    a.n, a.heads = 100_000, 2
    assert h.tmp_decay_attention_workspace_bytes(C.byref(a)) >= 3 * 2 * 2 * 128 * 128 * 4
