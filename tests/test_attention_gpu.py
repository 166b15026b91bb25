"""Attention with a window and sinks against its definition in 64 bits: values and gradients, element by element.

The tolerances follow from what is rounded. With u = 2^-8 (half a step of bf16, relative): probabilities are rounded as operands, so out is off by
u sum(p |v|) beside its own rounding u |out|; dv likewise by u sum(p |dout|) + u |dv|. delta is made of the rounded out, so a score's gradient
dS = p (dp - delta) is off by u |dS| as an operand and by p sum(|dout| * out's error); dq and dk sum that times |k| or |q|, beside their own rounding.
What 32 bits lose (scores, exponentials by the unit, sums: less than 2^-12 of the same sums) is a factor 1 + 2^-4 of all that.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = 2.0 ** -8
MORE = 1 + 2.0 ** -4
TINY = 2.0 ** -100


def _inputs(b, s, nq, nkv, hd, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda h: (torch.randn(b, s, h, hd, device="cuda", generator=g) * std).to(BF)   # noqa: E731
    return make(nq), make(nkv), make(nkv), make(nq)


def _expected(q, k, v, do, window, sinks, lengths, scale=None, inner=None):
    """name -> (value, bound) in 64 bits; rows behind a sequence's end do not take part. inner: what operands and delta are off by instead of u."""
    B, S, nq, hd = q.shape
    nkv, scale = k.shape[2], scale or hd ** -0.5
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None]
    sees = j <= i
    if window:
        sees = sees & ((i - j < window) | (j < sinks))
    n = lengths.long().clamp(0, S) if lengths is not None else torch.full((B,), S, device="cuda")
    there = torch.arange(S, device="cuda")[None] < n[:, None]                     # [B, S]
    sees = sees[None, None] & there[:, None, :, None] & there[:, None, None, :]   # [B, 1, S, S]
    clean = lambda x: torch.where(there[:, :, None, None], x.double(), 0.0).transpose(1, 2)   # noqa: E731
    G = nq // nkv
    Q, D = clean(q), clean(do)
    K, V = clean(k).repeat_interleave(G, 1), clean(v).repeat_interleave(G, 1)
    x = (Q @ K.transpose(2, 3) * scale).masked_fill(~sees, -torch.inf)
    p = torch.where(sees, torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e300)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ V
    w = inner or U
    err_out = w * (p @ V.abs()) + U * out.abs()
    err_delta = (D.abs() * (w * (p @ V.abs()) if inner else err_out)).sum(-1, keepdim=True)
    dp = D @ V.transpose(2, 3)
    ds = p * (dp - (D * out).sum(-1, keepdim=True)) * scale
    err_ds = w * ds.abs() + scale * p * err_delta
    group = lambda x: x.view(B, nkv, G, S, hd).sum(2)   # noqa: E731
    dv, dk, dq = group(p.transpose(2, 3) @ D), group(ds.transpose(2, 3) @ Q), ds @ K
    bounds = dict(out=err_out, dv=w * group(p.transpose(2, 3) @ D.abs()) + U * dv.abs(),
                  dk=group(err_ds.transpose(2, 3) @ Q.abs()) + U * dk.abs(), dq=err_ds @ K.abs() + U * dq.abs())
    return {name: (value.transpose(1, 2), bounds[name].transpose(1, 2) * MORE + TINY) for name, value in dict(out=out, dq=dq, dk=dk, dv=dv).items()}


def _run(q, k, v, do, **kw):
    from aws_ofi_nccl_b200.ops.attention import attention

    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves, **kw)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))))


def _check(q, k, v, do, window=0, sinks=0, lengths=None, scale=None, inner=None):
    got = _run(q, k, v, do, window=window, sinks=sinks, lengths=lengths, scale=scale)
    for name, (value, bound) in _expected(q, k, v, do, window, sinks, lengths, scale, inner).items():
        assert got[name].dtype == BF and got[name].shape == value.shape
        off = (got[name].double() - value).abs()
        worst = (off / bound).max().item()
        assert (off <= bound).all(), (name, worst, off.max().item())
    return got


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("s", [1, 2, 63, 64, 65, 127, 128, 129, 257, 500])
def test_every_key_up_to_the_query(s, hd):
    _check(*_inputs(2, s, 4, 2, hd, seed=s))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (2, 3), (63, 0), (64, 64), (65, 5), (128, 4), (129, 129), (200, 0), (299, 300), (300, 0), (5000, 7), (100, 299)])
def test_windows_and_sinks(window, sinks, hd):
    _check(*_inputs(1, 300, 2, 1, hd, seed=window + sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("nq, nkv", [(1, 1), (3, 1), (7, 7), (6, 2), (5, 1), (16, 2)])
def test_heads_that_share_keys(nq, nkv):
    _check(*_inputs(2, 333, nq, nkv, 64, seed=nq), window=100, sinks=3)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(1, 1), (32, 4), (70, 130), (200, 260)])
def test_sinks_seen_from_far_away(window, sinks, hd):
    """The queries that see a tile of keys only through its sinks are shared out to several CTAs."""
    _check(*_inputs(1, 1500, 4, 2, hd, seed=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 3), (64, 140)])
@pytest.mark.parametrize("lengths", [(400, 0, 1, 399), (64, 128, 129, 200), (-5, 700, 65, 63)])
def test_rows_behind_a_sequence_are_zeros_whatever_they_hold(lengths, window, sinks):
    q, k, v, do = _inputs(4, 400, 6, 2, 64, seed=3)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b, at in enumerate(lengths):
        for t in (q, k, v, do):
            t[b, min(max(at, 0), 400):] = float("nan") if b % 2 else float("inf")
    got = _check(q, k, v, do, window=window, sinks=sinks, lengths=n)
    for b, at in enumerate(lengths):
        assert all((t[b, min(max(at, 0), 400):] == 0).all() for t in got.values())


def test_large_scores():
    """Scores of some hundreds: maxima grow from tile to tile, and almost all of a row lies on one key."""
    q, k, v, do = _inputs(1, 700, 2, 2, 128, seed=5)
    k = (k * torch.linspace(0.1, 20, 700, device="cuda")[None, :, None, None]).to(BF)
    _check(q, k, v, do)
    _check(q, k, v, do, window=260, sinks=9, scale=0.02)


def test_a_key_that_is_minus_infinity_weighs_nothing():
    q, k, v, do = _inputs(1, 200, 1, 1, 64, seed=6)
    q = q.abs()
    k[0, 150] = -torch.inf
    from aws_ofi_nccl_b200.ops.attention import attention
    out = attention(q, k, v)
    left = [t for t in range(200) if t != 150]
    want = attention(q[:, left].contiguous(), k[:, left].contiguous(), v[:, left].contiguous())
    # the same probabilities, summed in another order: each side is off by its own rounding and its operands'
    p_v = v.abs().double().amax()
    assert ((out[:, 151:].double() - want[:, 150:].double()).abs() <= 4 * U * p_v).all() and out[:, :150].isfinite().all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("b, s, nq, nkv, window, sinks", [(1, 2, 1, 1, 0, 0), (2, 3, 4, 2, 0, 0), (3, 32, 6, 2, 0, 0), (1, 700, 4, 4, 1, 0), (2, 700, 4, 2, 1, 1),
                                                          (1, 1000, 2, 1, 20, 12), (4, 300, 3, 3, 2, 30), (40, 130, 8, 8, 3, 0), (2, 64, 2, 1, 0, 0), (1, 600, 4, 2, 33, 31), (2, 128, 3, 1, 0, 0), (1, 900, 4, 4, 100, 28)])
@pytest.mark.parametrize("ragged", [False, True])
def test_rows_of_few_keys_are_rounded_once(b, s, nq, nkv, window, sinks, hd, ragged):
    """Up to 128 keys a row, probabilities and gradients of scores are operands of 16 bits of mantissa (2^-17): what is left beside the results' rounding are
    exponentials by a cubic (2^-13.7) and delta, of the output and five bits of its rest (2^-8 of it, off by at most 2^-3: 2^-11). Together below 2^-10."""
    lengths = torch.tensor([s - n * s // 3 % s for n in range(b)], dtype=torch.int32, device="cuda") if ragged else None
    _check(*_inputs(b, s, nq, nkv, hd, seed=s), window=window, sinks=sinks, lengths=lengths, inner=2.0 ** -10)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(40, 150), (300, 161), (130, 290), (10, 400), (500, 130)])
def test_sinks_of_several_tiles(window, sinks, hd):
    """Walks with several tiles far from the window, of which some of the last one's columns are sinks."""
    lengths = torch.tensor([1700, 0, 1031], dtype=torch.int32, device="cuda")
    _check(*_inputs(3, 1700, 6, 2, hd, seed=window), window=window, sinks=sinks, lengths=lengths)
