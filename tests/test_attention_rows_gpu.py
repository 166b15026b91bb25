"""Attention row by row: how far a value that is not finite reaches, and that a row's accuracy is its own, not its batch's."""
import pytest
import torch

from test_attention_gpu import _inputs, _run

pytestmark = pytest.mark.gpu


def _same(a, b):
    return torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("hd, nq, nkv", [(64, 2, 1), (128, 3, 1)])
@pytest.mark.parametrize("window, sinks, at", [(200, 4, 100), (200, 4, 700), (200, 140, 200), (300, 3, 127), (50, 0, 300), (64, 128, 200)])
def test_a_value_that_is_not_finite_stays_within_reach(window, sinks, at, hd, nq, nkv, value):
    """Products are made of blocks of 128 tokens, in which zero times what is not finite is not zero: rows up to 512 tokens beyond the window may become NaN, of dk
    and dv also those in blocks that hold sinks. All others are the same bits."""
    s = 2200
    clean = dict(zip("qkvd", _inputs(1, s, nq, nkv, hd, seed=at)))
    want = _run(*clean.values(), window=window, sinks=sinks)
    row = torch.arange(s, device="cuda")
    sees = (row >= at) & (row - at < window)
    beyond = (row < at - window - 512) | (row >= at + window + 512)
    no_sinks = row >= (sinks + 127) // 128 * 128
    for which in "qkvd":
        bad = {n: t.clone() for n, t in clean.items()}
        bad[which][0, at, 0, 5] = value
        got = _run(*bad.values(), window=window, sinks=sinks)
        if which in "kv":
            for n in ("out", "dq"):
                assert _same(got[n][:, beyond], want[n][:, beyond]), (which, n)
            if value != value:
                assert (got["out"][0, sees].isnan().any(-1)).all()
        else:   # a query's own row; 32 neighbours move their maxima together, which rounds otherwise
            for n in ("out", "dq"):
                assert got[n][:, row != at].isfinite().all() and _same(got[n][:, row // 32 != at // 32], want[n][:, row // 32 != at // 32]), (which, n)
        for n in ("dk", "dv"):
            assert _same(got[n][:, beyond & no_sinks], want[n][:, beyond & no_sinks]), (which, n)
