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
