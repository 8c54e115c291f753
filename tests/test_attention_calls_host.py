"""Attention over series without a GPU: calls that are refused before anything is launched."""
import pytest

torch = pytest.importorskip("torch")


def _calls(q, k, v, do, ld, state, cache, length):
    from tempo_amd import ops
    out, lse = torch.zeros_like(do), torch.zeros(q.shape[:2])
    return {
        "window_attention": lambda: ops.window_attention(q, k, v, 3),
        "window_attention_grad": lambda: ops.window_attention_grad(do, q, k, v, out, lse, 3),
        "decay_attention": lambda: ops.decay_attention(q, k, v, ld, state=state),
        "decay_attention_grad": lambda: ops.decay_attention_grad(do, q, k, v, ld, state=state),
        "decay_attention_step": lambda: ops.decay_attention_step(q, k, v, ld, state),
        "window_attention_step": lambda: ops.window_attention_step(q, k, v, cache, cache.clone(), length),
        "window_cache_write": lambda: ops.window_cache_write(k, v, cache, cache.clone(), length),
    }


def test_forward_mode_is_refused():
    """A tangent on any array of rows or states, with and without a gradient wanted besides; without one calls go on to
    the check of the device."""
    from torch.autograd import forward_ad
    rows, state = lambda: torch.randn(4, 2, 8), torch.randn(1, 2, 8, 8)  # noqa: E731
    plain = dict(q=rows(), k=rows(), v=rows(), do=rows(), ld=torch.zeros(2), state=state, cache=torch.randn(4, 3, 2, 8),
                 length=torch.zeros(4, dtype=torch.int64))
    takes = {"window_attention": "qkv", "window_attention_grad": "qkvd", "decay_attention": "qkvls",
             "decay_attention_grad": "qkvdls", "decay_attention_step": "qkvls", "window_attention_step": "qkvc",
             "window_cache_write": "kvc"}
    with forward_ad.dual_level():
        for which in ("q", "k", "v", "do", "ld", "state", "cache"):
            dual = forward_ad.make_dual(plain[which], torch.ones_like(plain[which]))
            for name, call in _calls(**{**plain, which: dual}).items():
                if which[0] not in takes[name]:
                    continue
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        for call in _calls(**plain).values():
            with pytest.raises(TypeError, match="no CPU path"):
                call()


def test_series_offsets_runs_on_the_device_of_its_keys(monkeypatch):
    """key_counts launches on the current device's stream: the keys' device is made the current one around it."""
    import contextlib
    from tempo_amd import attention, ops
    entered = []

    @contextlib.contextmanager
    def current(device):
        entered.append(device)
        yield
        entered.append(None)

    def key_counts(key, n_keys):
        assert entered == [key.device]
        return torch.tensor([2, 0, 3])

    monkeypatch.setattr(attention, "_current", current)
    monkeypatch.setattr(attention, "_on_device", lambda t, *_: t)
    monkeypatch.setattr(ops, "key_counts", key_counts)
    assert ops.series_offsets(torch.zeros(5, dtype=torch.int32), 3).tolist() == [0, 2, 2, 5]
    assert len(entered) == 2
    monkeypatch.undo()
    with pytest.raises(TypeError, match="no CPU path"):
        ops.series_offsets(torch.zeros(5, dtype=torch.int32), 3)


def _args(cls, **kw):
    a = cls()
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_more_than_a_launch_holds_is_refused():
    """Fewer than 2^32 threads fit a launch: what would need more is refused before the first one, so that no call ends
    half done."""
    import ctypes as C
    from tempo_amd import _lib
    h = _lib.lib()
    rows = _lib.RowsRef(4096, 64, 16)
    most = (1 << 24) - 8
    a = dict(n=2 ** 31 - 65537, n_series=1, type=0, heads=2, kv_heads=2, dim_k=16, dim_v=16, window=5, sinks=1, scale=0.25, q=rows,
             k=rows, v=rows, out=rows, dout=rows, dq=rows, dk=rows, dv=rows, lse=4096)
    a = _args(_lib.WindowAttentionArgs, **a)
    assert h.tmp_window_attention(C.byref(a), None) == -4 and b"rows x heads" in h.tmp_last_error()
    assert h.tmp_window_attention_grad(C.byref(a), None, 0, None) == -4 and b"rows x heads" in h.tmp_last_error()
    assert h.tmp_window_attention_grad_workspace_bytes(C.byref(a)) == 0
    a.heads = a.kv_heads = 1  # the largest table of one head fits
    assert h.tmp_window_attention_grad_workspace_bytes(C.byref(a)) > 0
    for n, heads in ((most // 4 + 1, 8), (1 << 24, 2), (2 ** 16, 512)):
        a = _args(_lib.DecayAttentionStepArgs, n=n, n_slots=n, type=0, heads=heads, dim_k=16, dim_v=16, scale=1.0, log_decay=4096,
                  q=rows, k=rows, v=rows, out=rows, state=4096)
        assert h.tmp_decay_attention_step(C.byref(a), None) == -4 and b"rows x heads" in h.tmp_last_error()
        cache = _lib.CacheRef(4096, 640, 64, 16)
        a = _args(_lib.WindowAttentionStepArgs, n=n, n_slots=n, type=0, heads=heads, kv_heads=heads, dim_k=16, dim_v=16, window=8,
                  sinks=1, scale=1.0, q=rows, k=rows, v=rows, out=rows, k_cache=cache, v_cache=cache, length=4096)
        assert h.tmp_window_attention_step(C.byref(a), None, 0, None) == -4 and b"rows x heads" in h.tmp_last_error()
        assert h.tmp_window_attention_step_workspace_bytes(C.byref(a)) == 0
    a.n = a.n_slots = most  # (blocks of 128 threads join the parts: twice as many rows x heads as above)
    a.heads = a.kv_heads = 2
    assert h.tmp_window_attention_step_workspace_bytes(C.byref(a)) > 0
    a = _args(_lib.DecayAttentionStepArgs, n=most + 1, n_slots=most + 1, type=0, heads=1, dim_k=16, dim_v=16, scale=1.0)
    assert h.tmp_decay_attention_step(C.byref(a), None) == -4 and b"rows x heads" in h.tmp_last_error()
    a = _args(_lib.WindowCacheWriteArgs, n=100, n_series=600_000, offsets=4096, n_slots=600_000, type=0, kv_heads=1, dim_k=16,
              dim_v=16, window=1000, sinks=0, k=rows, v=rows, k_cache=cache, v_cache=cache, length=4096)
    assert h.tmp_window_cache_write(C.byref(a), None) == -4 and b"series x rows" in h.tmp_last_error()


def test_numbers_of_series():
    """Without offsets there is one series, with them any number whose arithmetic fits 32 bits."""
    import ctypes as C
    from tempo_amd import _lib
    h = _lib.lib()
    rows, cache = _lib.RowsRef(4096, 64, 16), _lib.CacheRef(4096, 640, 64, 16)
    common = dict(n=0, type=0, dim_k=16, dim_v=16, q=rows, k=rows, v=rows)
    calls = {
        "tmp_window_attention": (_args(_lib.WindowAttentionArgs, **common, heads=2, kv_heads=2, window=5, scale=1.0, out=rows), (None,)),
        "tmp_decay_attention": (_args(_lib.DecayAttentionArgs, **common, heads=2, scale=1.0, log_decay=4096, out=rows, state_out=4096),
                                (None, 0, None)),
        "tmp_window_cache_write": (_args(_lib.WindowCacheWriteArgs, n=0, type=0, dim_k=16, dim_v=16, kv_heads=2, window=5, n_slots=9,
                                         k=rows, v=rows, k_cache=cache, v_cache=cache, length=4096), (None,)),
    }
    for name, (a, rest) in calls.items():
        for offsets, n_series in ((None, -1), (None, 2), (4096, -1), (4096, 2 ** 31 - 65536), (4096, 2 ** 31 - 1)):
            a.offsets, a.n_series = offsets, n_series
            assert getattr(h, name)(C.byref(a), *rest) == -1, (name, offsets, n_series)
            assert b"series" in h.tmp_last_error()
    a, rest = calls["tmp_window_attention"]
    for offsets, n_series in ((None, 0), (None, 1), (4096, 0)):  # (no rows: nothing is launched)
        a.offsets, a.n_series = offsets, n_series
        assert h.tmp_window_attention(C.byref(a), *rest) == 0


def test_no_workspace_for_what_is_refused():
    import ctypes as C
    from tempo_amd import _lib
    h = _lib.lib()
    for change in (dict(dim_k=2 ** 20), dict(dim_v=129), dict(heads=65537), dict(n=2 ** 31 - 65536), dict(n=-1)):
        a = _args(_lib.DecayAttentionArgs, **{**dict(n=10 ** 6, n_series=1, heads=8, dim_k=64, dim_v=64), **change})
        assert h.tmp_decay_attention_workspace_bytes(C.byref(a)) == 0, change
