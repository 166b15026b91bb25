"""Attention row by row: how far a value that is not finite reaches, and that a row's accuracy is its own, not its batch's."""
import pytest
import torch

from test_attention_gpu import _check, _expected, _inputs, _run

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


@pytest.mark.parametrize("hd, nq, nkv", [(64, 4, 2), (128, 3, 1)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (200, 20), (129, 0), (90, 60), (300, 3)])
def test_a_sequence_is_the_same_alone_and_in_a_padded_batch(window, sinks, hd, nq, nkv):
    """However far its batch is padded: output and gradients of a short sequence are the same bits."""
    lengths = (3, 40, 90, 128, 1, 127)
    ts = _inputs(len(lengths), 128, nq, nkv, hd, seed=window + hd)
    for s in (128, 129, 700, 1400):
        padded = [torch.nn.functional.pad(t, (0, 0, 0, 0, 0, s - 128)) for t in ts]
        got = _run(*padded, window=window, sinks=sinks, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        for b, n in enumerate(lengths):
            alone = _run(*(t[b:b + 1, :n] for t in ts), window=window, sinks=sinks)
            for name in alone:
                assert torch.equal(alone[name][0], got[name][b, :n]), (s, n, name)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(0, 0), (200, 20), (120, 30)])
def test_short_sequences_of_a_long_batch_are_rounded_once(window, sinks, hd):
    """Every row of at most 128 keys, whatever its batch is padded to: probabilities and gradients of scores have 16 bits of mantissa, and beside the results' own
    rounding 2^-10 is left (test_rows_of_few_keys_are_rounded_once says of what)."""
    lengths = torch.tensor([3, 40, 90, 128], dtype=torch.int32, device="cuda")
    _check(*_inputs(4, 700, 4, 2, hd, seed=window), window=window, sinks=sinks, lengths=lengths, inner=2.0 ** -10)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(0, 0), (300, 20)])
def test_first_rows_of_a_long_sequence_are_those_of_a_short_one(window, sinks, hd):
    ts = _inputs(2, 900, 4, 2, hd, seed=11)
    whole, part = _run(*ts, window=window, sinks=sinks), _run(*(t[:, :128] for t in ts), window=window, sinks=sinks)
    for name in ("out", "dq"):
        assert torch.equal(whole[name][:, :128], part[name]), name


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("s, window, sinks", [(1100, 0, 0), (1500, 300, 4), (1500, 140, 150), (129, 0, 0)])
def test_two_roundings_in_the_mean(s, window, sinks, hd):
    """Rows of many keys: one rounding of an operand (P or dS) and the result's own, in the Frobenius norm.

    Rounding a value m 2^e, 1 <= m < 2, to 8 bits of mantissa is off by at most half a step of 2^(e-7) and, over values whose further bits are even, by its root mean
    square, 2^(e-7) / sqrt(12): relative to the value at most 2^-7 / sqrt(12) = 2.26e-3. An operand's errors are independent of each other and of what it is multiplied with, whose signs are
    random here, so a product's relative norm is off by as much as the operand is. Two of them make sqrt(2) 2.26e-3 at most."""
    ts = _inputs(2, s, 4, 2, hd, seed=s + hd)
    got = _run(*ts, window=window, sinks=sinks)
    for name, (want, _) in _expected(*ts, window, sinks, None).items():
        off = ((got[name].double() - want).norm() / want.norm()).item()
        assert off <= (2 / 12) ** 0.5 * 2.0 ** -7, (name, off)
