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
