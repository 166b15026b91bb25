"""Tokens sorted by expert and back: the order against a stable sort on the host, rows bit by bit, sums and gradients against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F = 2.0 ** -8, 2.0 ** -24   # half a step of bf16 and of fp32, relative


def _order(idx, experts):
    flat = idx.cpu().long().reshape(-1)
    live = (flat >= 0) & (flat < experts)
    key = torch.where(live, flat, experts)
    slot = torch.sort(key, stable=True).indices
    row = torch.empty_like(slot)
    row[slot] = torch.arange(slot.numel())
    offsets = torch.cat((torch.zeros(1, dtype=torch.long), torch.bincount(key, minlength=experts + 1).cumsum(0)[:experts]))
    return torch.where(live, row, ~row).view(idx.shape), offsets, slot


def _choices(T, k, E, seed=0, lost=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * T + k)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    return torch.where(torch.rand(T, k, device="cuda", generator=g) < lost, -1, idx)


# one warp's part of a batch of loads, whole batches and one more; a CTA, two, four and eight; several batches; the fewest and the most experts
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 64), (3, 5, 7), (16, 8, 256), (511, 1, 3), (2048, 1, 1000), (2049, 1, 40), (4096, 1, 60), (4097, 1, 60), (1025, 8, 128),
                                   (2731, 3, 1024), (5000, 8, 1023), (20011, 7, 256), (65536, 8, 33), (333, 2, 1024)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_order_is_a_stable_sort(T, k, E, kind):
    from aws_ofi_nccl_b200.ops import moe

    idx = _choices(T, k, E).to(kind)
    row_of, offsets, _ = _order(idx, E)
    for _ in range(2):   # the same in every run
        order = moe.expert_order(idx, E)
        assert torch.equal(order.row_of.cpu().long(), row_of)
        assert torch.equal(order.offsets.cpu().long(), offsets)


@pytest.mark.parametrize("T,k,E", [(700, 3, 9), (9000, 2, 100)])
def test_order_of_one_expert_none_and_numbers_out_of_range(T, k, E):
    from aws_ofi_nccl_b200.ops import moe

    far = torch.tensor([-1, E, E + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 32, -2 ** 63, 2 ** 62], device="cuda")
    for idx in (torch.full((T, k), E - 1, device="cuda"), torch.full((T, k), -1, device="cuda"),
                far[torch.arange(T * k, device="cuda") % 8].view(T, k), torch.where(_choices(T, k, E) < 0, far[5], 1).long()):
        row_of, offsets, _ = _order(idx, E)
        order = moe.expert_order(idx, E)
        assert torch.equal(order.row_of.cpu().long(), row_of) and torch.equal(order.offsets.cpu().long(), offsets)


def test_no_tokens():
    from aws_ofi_nccl_b200.ops import moe

    order = moe.expert_order(torch.empty(0, 4, device="cuda", dtype=torch.int32), 5)
    assert order.row_of.shape == (0, 4) and order.offsets.tolist() == [0] * 6
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(0, 4, device="cuda", requires_grad=True)
    rows = moe.permute_tokens(x, order)
    out = moe.unpermute_tokens(rows, order, w)
    assert rows.shape == (0, 64) and out.shape == (0, 64)
    out.sum().backward()
    assert x.grad.shape == (0, 64) and w.grad.shape == (0, 4)


def _check(T, k, E, H, dtype, x=None, y=None, lost=0.2):
    """One pass of everything; y: the experts' rows, of which those of lost choices hold NaN"""
    from aws_ofi_nccl_b200.ops import moe

    g = torch.Generator(device="cuda").manual_seed(T + k + H)
    idx = _choices(T, k, E, lost=lost)
    row_of, offsets, slot = (t.cuda() for t in _order(idx, E))
    n = int(offsets[-1])
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    x = (rnd(T, H).to(dtype) if x is None else x).requires_grad_(True)
    y = rnd(T * k, H).to(dtype) if y is None else y
    y[n:] = math.nan
    y.requires_grad_(True)
    w = rnd(T, k).requires_grad_(True)
    drows, dout = rnd(T * k, H).to(dtype), rnd(T, H).to(dtype)
    drows[n:] = math.inf
    order = moe.expert_order(idx, E)
    rows, out = moe.permute_tokens(x, order), moe.unpermute_tokens(y, order, w)
    dx, dy, dw = torch.autograd.grad((rows, out), (x, y, w), (drows, dout))
    plain = moe.unpermute_tokens(y, order)
    (dplain,) = torch.autograd.grad(plain, (y,), dout)

    token = (slot // k)[:n]
    want_rows = torch.zeros(T * k, H, device="cuda", dtype=dtype)
    want_rows[:n] = x.detach()[token]
    assert torch.equal(rows.detach(), want_rows)
    half = BF if dtype == torch.bfloat16 else F
    W, Y, D = w.detach().double().view(-1)[slot][:n, None], y.detach().double()[:n], dout.double()

    def summed(rows64):
        total, mag = (torch.zeros(T, H, device="cuda", dtype=torch.float64).index_add_(0, token, r) for r in (rows64, rows64.abs()))
        # k sums in 32 bits, each off by half a step of at most the magnitudes' sum, and the result's rounding
        return total, half * total.abs() + (k + 1) * F * mag * (1 + half) + 1e-37

    for got, terms in ((out, W * Y), (plain, Y), (dx, drows.double()[:n])):
        want, most = summed(terms)
        assert ((got.detach().double() - want).abs() <= most).all()
    want = W * D[token]
    assert ((dy.double()[:n] - want).abs() <= (half + 2 * F) * want.abs() + 1e-37).all() and (dy[n:] == 0).all()
    assert torch.equal(dplain[:n], dout[token]) and (dplain[n:] == 0).all()
    prod = D[token] * Y
    want = torch.zeros(T * k, device="cuda", dtype=torch.float64)
    mag = torch.zeros_like(want)
    want[slot[:n]], mag[slot[:n]] = prod.sum(-1), prod.abs().sum(-1)
    # H products and sums in some order, each off by half a step of at most the magnitudes' sum
    assert ((dw.double().view(-1) - want).abs() <= (H + 8) * F * mag + 1e-37).all()
    assert (dw.view(-1)[slot[n:]] == 0).all()


# a row of one element, less than a warp, a team of one warp, of several, of the whole CTA; rows that are no whole number of vectors
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 1), (1, 8, 64, 4096), (5, 2, 3, 8), (37, 3, 5, 72), (64, 4, 8, 1000), (50, 5, 8, 1001), (130, 8, 16, 2048),
                                     (33, 9, 12, 4104), (20, 8, 256, 7168), (3, 2, 4, 16392), (3001, 3, 60, 131), (2000, 2, 8, 520)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_there_and_back(T, k, E, H, dtype):
    _check(T, k, E, H, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lost", [0.0, 1.0])
def test_all_choices_kept_and_all_lost(dtype, lost):
    _check(70, 4, 6, 264, dtype, lost=lost)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows(dtype):
    """Columns of a wider matrix, on and off a 16-byte boundary, and rows whose elements do not lie together"""
    T, k, H = 45, 3, 128
    for width, at in ((256, 0), (256, 128), (131, 0), (131, 3), (136, 8)):
        _check(T, k, 7, H, dtype, x=torch.randn(T, width, device="cuda").to(dtype)[:, at:at + H].detach(),
               y=torch.randn(T * k, width, device="cuda").to(dtype)[:, at:at + H].detach())
    _check(T, k, 7, H, dtype, x=torch.randn(H, T, device="cuda").to(dtype).t(), y=torch.randn(H, T * k, device="cuda").to(dtype).t())


@pytest.mark.parametrize("T,k,H,groups", [(1, 1, 16, 0), (40, 3, 48, 0), (40, 3, 256, 2), (33, 2, 130, 130), (200, 8, 4096, 32), (7, 4, 33, 0), (9, 2, 64, 8)])
def test_rows_in_8_bits_take_their_scales_along(T, k, H, groups):
    from aws_ofi_nccl_b200.ops import moe

    idx = _choices(T, k, 5)
    _, offsets, slot = (t.cuda() for t in _order(idx, 5))
    n = int(offsets[-1])
    x = torch.randint(0, 256, (T, H), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)   # NaN codes too: they are moved, not read
    scale = torch.rand(T, groups, device="cuda") if groups else torch.rand(T, device="cuda")
    order = moe.expert_order(idx, 5)
    rows, row_scale = moe.permute_tokens(x, order, scale)
    assert rows.dtype == x.dtype and torch.equal(rows.view(torch.uint8)[:n], x.view(torch.uint8)[(slot // k)[:n]])
    assert (rows.view(torch.uint8)[n:] == 0).all()
    assert torch.equal(row_scale[:n], scale[(slot // k)[:n]]) and (row_scale[n:] == 0).all()
    assert torch.equal(moe.permute_tokens(x, order).view(torch.uint8), rows.view(torch.uint8))


def test_gradients_against_differences():
    """The sums are linear in rows and in weights: a difference of two passes is the gradient but for their rounding."""
    from aws_ofi_nccl_b200.ops import moe

    T, k, E, H = 6, 3, 4, 40
    idx = _choices(T, k, E, seed=3)
    order = moe.expert_order(idx, E)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w, d = (torch.randn(*s, device="cuda", generator=g) for s in ((T, H), (T, k), (T, H)))
    f = lambda x, w: (moe.unpermute_tokens(moe.permute_tokens(x, order), order, w).double() * d.double()).sum().item()   # noqa: E731
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(moe.unpermute_tokens(moe.permute_tokens(x, order), order, w), (x, w), d)
    step = 0.25
    # each of the T * H sums is off by at most (k + 1) half steps of its magnitude, in both passes; the gradient by (H + 8) of its own
    most = 2 * T * H * (k + 1) * F * 60 / (2 * step)
    with torch.no_grad():
        for t in range(T):
            for j in range(k):
                e = torch.zeros_like(w)
                e[t, j] = step
                assert abs((f(x, w + e) - f(x, w - e)) / (2 * step) - dw[t, j].item()) <= most
            e = torch.zeros_like(x)
            e[t, 5] = step
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * step) - dx[t, 5].item()) <= most


def test_only_the_gradients_that_are_asked_for():
    from aws_ofi_nccl_b200.ops import _lib, moe

    idx = _choices(30, 2, 4)
    order = moe.expert_order(idx, 4)
    y, w, d = torch.randn(60, 64, device="cuda"), torch.randn(30, 2, device="cuda"), torch.randn(30, 64, device="cuda")
    both = [t.clone().requires_grad_(True) for t in (y, w)]
    dy, dw = torch.autograd.grad(moe.unpermute_tokens(both[0], order, both[1]), both, d)
    (only,) = torch.autograd.grad(moe.unpermute_tokens(both[0], order, w), both[:1], d)
    assert torch.equal(only, dy)
    before = _lib.launch_count
    (only,) = torch.autograd.grad(moe.unpermute_tokens(y, order, both[1]), both[1:], d)
    assert torch.equal(only, dw) and _lib.launch_count - before == 2
    e = torch.autograd.grad(moe.unpermute_tokens(both[0], order, both[1]).sum(), both)   # an expanded gradient
    ones = torch.autograd.grad(moe.unpermute_tokens(both[0], order, both[1]), both, torch.ones_like(d))
    assert torch.equal(e[0], ones[0]) and torch.equal(e[1], ones[1])


def test_an_order_of_other_numbers_is_read_within_bounds():
    """What no expert_order made (rows beyond the last) is skipped: it neither reads nor writes elsewhere."""
    from aws_ofi_nccl_b200.ops import moe

    row_of = torch.tensor([[0, 7], [2 ** 31 - 1, -2 ** 31], [3, -200], [1, -3]], device="cuda", dtype=torch.int32)
    order = moe.ExpertOrder(row_of, torch.zeros(2, device="cuda", dtype=torch.int32))
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(4, 2, device="cuda", requires_grad=True)
    rows = moe.permute_tokens(x, order)
    for r, t in ((0, 0), (7, 0), (3, 2), (1, 3)):
        assert torch.equal(rows[r], x[t])
    assert (rows[2] == 0).all()
    y = torch.randn(8, 64, device="cuda", requires_grad=True)
    out = moe.unpermute_tokens(y, order, w)
    assert torch.equal(out[1], torch.zeros_like(out[1])) and torch.equal(out[2], y[3])
    dy, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert (dy[[0, 7, 3, 1]] == 1).all() and (dw[1] == 0).all() and dw[2, 1] == 0


def test_captured_and_replayed_with_other_choices():
    from aws_ofi_nccl_b200.ops import moe

    T, k, E, H = 300, 4, 16, 520
    idx, x, w = _choices(T, k, E), torch.randn(T, H, device="cuda"), torch.randn(T, k, device="cuda")

    def step():
        order = moe.expert_order(idx, E)
        return order, moe.unpermute_tokens(moe.permute_tokens(x, order), order, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        order, out = step()
    for seed in (1, 2):
        idx.copy_(_choices(T, k, E, seed=seed))
        x.normal_()
        graph.replay()
        want_order, want = step()
        assert torch.equal(order.row_of, want_order.row_of) and torch.equal(order.offsets, want_order.offsets) and torch.equal(out, want)


def test_two_streams_at_once():
    from aws_ofi_nccl_b200.ops import moe

    streams = [torch.cuda.Stream() for _ in range(2)]
    work = [(_choices(4000, 4, 64, seed=s), torch.randn(4000, 512, device="cuda")) for s in range(2)]
    want = [moe.permute_tokens(x, moe.expert_order(i, 64)) for i, x in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(moe.permute_tokens(work[n][1], moe.expert_order(work[n][0], 64)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[n]) for n in range(2) for g in got[n])


def test_second_derivatives():
    """Of the plain sum and of the rows, which are linear; with weights it is refused instead of left out."""
    from aws_ofi_nccl_b200.ops import moe

    idx = _choices(20, 3, 5)
    order = moe.expert_order(idx, 5)
    n = int(order.offsets[-1])
    x, d = torch.randn(20, 72, device="cuda", requires_grad=True), torch.randn(60, 72, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(moe.permute_tokens(x, order), x, d, create_graph=True)
    (dd,) = torch.autograd.grad(dx, d, x.detach())
    assert torch.equal(dd, moe.permute_tokens(x.detach(), order)) and (dd[n:] == 0).all()
    (dy,) = torch.autograd.grad(moe.unpermute_tokens(d, order), d, x, create_graph=True)
    (back,) = torch.autograd.grad(dy, x, d.detach())
    assert torch.equal(back, moe.unpermute_tokens(d.detach(), order))
    w = torch.rand(20, 3, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(moe.unpermute_tokens(d, order, w), (d, w), x.detach(), create_graph=True)


def test_an_inference_pass_and_changed_inputs():
    """Without gradients nothing is kept; what a graph keeps is checked when it is used."""
    from aws_ofi_nccl_b200.ops import moe

    idx = _choices(20, 3, 5)
    with torch.inference_mode():
        order = moe.expert_order(idx, 5)
        rows = moe.permute_tokens(torch.randn(20, 64, device="cuda"), order)
        assert moe.unpermute_tokens(rows, order, torch.rand(20, 3, device="cuda")).shape == (20, 64)
    order = moe.expert_order(idx, 5)
    y, w = torch.randn(60, 64, device="cuda"), torch.rand(20, 3, device="cuda", requires_grad=True)
    out = moe.unpermute_tokens(y, order, w)
    y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_threads_at_once():
    import threading

    from aws_ofi_nccl_b200.ops import llm, moe

    x, idx, failed = torch.randn(500, 264, device="cuda"), _choices(500, 4, 16), []
    want = moe.permute_tokens(x, moe.expert_order(idx, 16))
    torch.cuda.synchronize()

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    p = [torch.zeros(700, device="cuda") for _ in range(20)]
                    g = [torch.ones(700, device="cuda") for _ in range(20)]
                    llm.adamw_step_many(p, g, **llm.adamw_states(p, bits=8), lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1)
                    rows = moe.permute_tokens(x, moe.expert_order(idx, 16))
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(rows, want) and all(torch.equal(q, p[0]) and (q != 0).all() for q in p)
        except BaseException as e:   # noqa: BLE001  the test's thread raises it
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed
