"""Activations kept in 8 bits, against their definition in 64 bits.

What is kept is compared with the value of e4m3 nearest to each quotient (ties to the even one), bit by bit: the powers of two scale exactly. Products and
activations of what is kept round to bf16 once more (u = 2^-8 of a value); products add up in 32 bits (2^-24 a term, of the sum of magnitudes: below 2^-12 of that
for the lengths here), the SwiGLU's functions are within 2^-20.
"""
import math

import pytest
import torch

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -8


def _power(group):
    """The byte of a list of finite floats."""
    top = max(abs(v) for v in group)
    e = -127
    while top > 448 * 2.0 ** e:
        e += 1
    return e + 127


def _kept(x):
    """[rows, n] in 64 bits: (values, bytes)"""
    rows, n = x.shape
    out, powers = torch.empty_like(x), torch.empty(rows, -(-n // 32), dtype=torch.uint8)
    for r in range(rows):
        for c in range(0, n, 32):
            v = x[r, c:c + 32]
            ok = v.isfinite()
            b = _power(v[ok].tolist() or [0.0])
            y = v / 2.0 ** (b - 127)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
            q = torch.round(y / step) * step * 2.0 ** (b - 127)
            out[r, c:c + 32] = torch.where(ok, q, math.nan)
            powers[r, c // 32] = b
    return out, powers


def _exact(x):
    """_kept of a larger matrix, on its device, of finite values"""
    g = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    e = torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -140) / 448)).clamp_min(-127)
    for _ in range(2):   # the logarithm is rounded
        e = torch.where(g.abs().amax(-1, keepdim=True) > 448 * torch.exp2(e), e + 1, e)
    e = torch.where((g.abs().amax(-1, keepdim=True) <= 448 * torch.exp2(e - 1)) & (e > -127), e - 1, e)
    y = g / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * torch.exp2(e)).view(x.shape[0], -1)[:, :x.shape[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", [(1, 8), (3, 24), (2, 32), (5, 40), (7, 96), (33, 264), (1, 4104)])
def test_codes_and_powers(rows, n):
    from aws_ofi_nccl_b200.ops import llm

    g = torch.Generator().manual_seed(n)
    x = (torch.randn(rows, n, generator=g) * torch.exp2(torch.randint(-40, 40, (rows, n), generator=g).float())).to(BF)
    codes, powers = llm.keep_rows8(x.cuda())
    want, bytes_ = _kept(x.double())
    assert codes.dtype == F8 and codes.shape == x.shape and torch.equal(powers.cpu(), bytes_)
    scale = torch.exp2(bytes_.double() - 127).repeat_interleave(32, 1)[:, :n]
    assert torch.equal(codes.cpu().double() * scale, want)
    assert torch.equal(llm.kept_rows8(codes, powers).cpu(), want.to(BF))


@pytest.mark.gpu
def test_every_bf16_value_alone_and_beside_others():
    """All 65536 patterns: each alone with zeros, and 32 neighbours in a group."""
    from aws_ofi_nccl_b200.ops import llm

    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    alone = torch.zeros(65536, 32, dtype=BF)
    alone[torch.arange(65536), torch.arange(65536) % 32] = every
    for x in (alone, every.view(2048, 32)):
        codes, powers = llm.keep_rows8(x.cuda())
        pick = torch.arange(0, x.shape[0], 7 if x.shape[0] > 4096 else 1)
        want, bytes_ = _kept(x[pick].double())
        assert torch.equal(powers.cpu()[pick], bytes_)
        got = codes.cpu()[pick].double() * torch.exp2(bytes_.double() - 127)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        back = llm.kept_rows8(codes, powers).cpu()[pick]
        assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(), want.to(BF).nan_to_num())


@pytest.mark.gpu
def test_strided_rows_and_odd_addresses():
    from aws_ofi_nccl_b200.ops import llm

    wide = torch.randn(9, 200, device="cuda").to(BF)
    flat = torch.randn(1 + 6 * 48, device="cuda").to(BF)
    for x in (wide[:, 8:88], wide[:, 3:83], wide[::2, :64], torch.randn(64, 9, device="cuda").to(BF).t(), flat[1:].view(6, 48), wide.view(3, 3, 200)[:, :, :40], torch.empty(0, 64, device="cuda", dtype=BF)):
        codes, powers = llm.keep_rows8(x)
        assert codes.shape == x.shape and powers.shape == (*x.shape[:-1], -(-x.shape[-1] // 32))
        if x.numel():
            assert torch.equal(llm.kept_rows8(codes, powers).double().reshape(-1, x.shape[-1]), _exact(x.double().reshape(-1, x.shape[-1])))


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 8, 8), (5, 64, 40), (128, 256, 256), (300, 72, 1000), (1000, 520, 264)])
@pytest.mark.parametrize("main_grad", [False, True])
def test_linear_keeps_its_input(m, n, k, main_grad):
    from aws_ofi_nccl_b200.ops.gemm import linear

    g = torch.Generator(device="cuda").manual_seed(m)
    x, w, dy = ((torch.randn(*s, device="cuda", generator=g) * 2).to(BF) for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(True), w.requires_grad_(True)
    if main_grad:
        w.main_grad, w.grad_written = torch.zeros_like(w), False
    y = linear(x, w, keep_bits=8)
    assert torch.equal(y, linear(x.detach(), w.detach()))
    y.backward(dy)
    kept = _exact(x.detach().double())
    dw = dy.double().t() @ kept
    off = ((w.main_grad if main_grad else w.grad).double() - dw).abs()
    assert (off <= U * dw.abs() + 2.0 ** -12 * (dy.double().abs().t() @ kept.abs())).all()
    plain = x.detach().clone().requires_grad_(True)
    linear(plain, w.detach()).backward(dy)
    assert (x.grad.double() - plain.grad.double()).abs().max() <= 2 * U * plain.grad.abs().max()   # products alone or two in a launch


@pytest.mark.gpu
@pytest.mark.parametrize("t, f", [(1, 8), (3, 40), (256, 512), (17, 1376), (1001, 72)])
def test_swiglu_keeps_gate_and_up(t, f):
    from aws_ofi_nccl_b200.ops import llm

    g = torch.Generator(device="cuda").manual_seed(t)
    gu = (torch.randn(t, 2 * f, device="cuda", generator=g) * 3).to(BF).requires_grad_(True)
    d = torch.randn(t, f, device="cuda", generator=g).to(BF)
    act = llm.swiglu(gu, keep_bits=8)
    assert torch.equal(act, llm.swiglu(gu.detach()))
    act.backward(d)
    gate, up = (_exact(h.contiguous()) for h in gu.detach().double().split(f, 1))
    s = torch.sigmoid(gate)
    want = torch.cat((d.double() * up * s * (1 + gate * (1 - s)), d.double() * gate * s), 1)
    part = torch.cat((d.double() * up * s * (1 + (gate * (1 - s)).abs()), d.double() * gate * s), 1).abs()   # terms that cancel
    assert ((gu.grad.double() - want).abs() <= U * want.abs() + 2.0 ** -18 * part).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t, hidden, f", [(64, 64, 128), (300, 256, 520), (2048, 512, 1024)])
def test_mlp_is_its_parts(t, hidden, f):
    """The layer against its three parts with 8 bits each, with the gate and up that it kept: the same codes, so products of the same operands."""
    from aws_ofi_nccl_b200.ops import llm

    g = torch.Generator(device="cuda").manual_seed(t)
    make = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(BF).requires_grad_(True)   # noqa: E731
    x, wgu, wd, dy = make(t, hidden), make(2 * f, hidden, std=hidden ** -0.5), make(hidden, f, std=f ** -0.5), make(t, hidden).detach()
    y = llm.swiglu_mlp(x, wgu, wd, keep_bits=8)
    assert torch.equal(y, llm.swiglu_mlp(x.detach(), wgu.detach(), wd.detach()))
    y.backward(dy)
    with torch.no_grad():
        gu = (x.double() @ wgu.double().t())
    # what the layer kept is not seen from here; gate and up rounded to bf16 either way differ by a step of bf16 where they lie on a border, and by a step of
    # e4m3 behind that: a matrix' worth of such differences is bounded through norms, an eighth of a step of e4m3 (2^-3) in the mean
    gate, up = _exact(gu[:, :f].to(BF).double()), _exact(gu[:, f:].to(BF).double())
    s = torch.sigmoid(gate)
    dact = dy.double() @ wd.detach().double()
    dgu = torch.cat((dact * up * s * (1 + gate * (1 - s)), dact * gate * s), 1)
    for got, want in ((x.grad, dgu @ wgu.detach().double()), (wgu.grad, dgu.t() @ _exact(x.detach().double())), (wd.grad, dy.double().t() @ (gate * s * up))):
        assert (got.double() - want).norm() <= 2.0 ** -6 * want.norm()


@pytest.mark.gpu
def test_a_layer_holds_no_more_than_it_keeps():
    """Bytes asked for that live between the passes (the allocator may hand out up to a megabyte more)."""
    from aws_ofi_nccl_b200.ops import llm

    t, hidden, f = 4096, 512, 1024
    wgu, wd = (torch.randn(*s, device="cuda").to(BF).requires_grad_(True) for s in ((2 * f, hidden), (hidden, f)))
    held = {}
    for bits in (8, 16):
        x = torch.randn(t, hidden, device="cuda").to(BF)
        torch.cuda.synchronize()
        asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]   # noqa: E731
        before = asked()
        y = llm.swiglu_mlp(x, wgu, wd, keep_bits=bits)
        del x
        held[bits] = asked() - before - y.numel() * 2 + t * hidden * 2
        del y
    assert held[8] <= t * (hidden + 2 * f) * 33 // 32 + 8192 and held[16] >= t * (2 * hidden + 6 * f)


@pytest.mark.gpu
def test_only_what_is_asked_for():
    from aws_ofi_nccl_b200.ops import gemm, llm

    x, w = torch.randn(40, 64, device="cuda").to(BF), torch.randn(32, 64, device="cuda").to(BF)
    wgu, wd = torch.randn(64, 64, device="cuda").to(BF), torch.randn(16, 32, device="cuda").to(BF)
    dy = torch.ones(40, 32, device="cuda", dtype=BF)
    xg = x.clone().requires_grad_(True)
    gemm.linear(xg, w, keep_bits=8).backward(dy)
    want = x.clone().requires_grad_(True)
    gemm.linear(want, w).backward(dy)
    assert torch.equal(xg.grad, want.grad)
    for which in range(3):
        ts = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, wgu, wd))]
        llm.swiglu_mlp(*ts, keep_bits=8).backward(dy[:, :16])
        assert [t.grad is not None for t in ts] == [i == which for i in range(3)] and ts[which].grad.isfinite().all()
    assert not gemm.linear(x, w, keep_bits=8).requires_grad and not llm.swiglu(x, keep_bits=8).requires_grad


def _refused(fn, *args, error=(AssertionError, RuntimeError, ValueError, TypeError), **kw):
    with pytest.raises(error):
        fn(*args, **kw)


def test_refusals_without_a_gpu(built):
    from aws_ofi_nccl_b200.models.llama import LlamaConfig
    from aws_ofi_nccl_b200.ops import gemm, llm

    x = torch.ones(4, 64, dtype=BF)
    for fn, args in ((gemm.linear, (x, x)), (llm.swiglu, (x,)), (llm.swiglu_mlp, (x, x, x)), (llm.keep_rows8, (x,))):
        if fn is not llm.keep_rows8:
            for bits in (0, 4, 7, 32, None):
                _refused(fn, *args, keep_bits=bits, error=ValueError)
            _refused(fn, *args, keep_bits=8)
        else:
            _refused(fn, *args)
    _refused(llm.kept_rows8, x.to(F8), torch.zeros(4, 2, dtype=torch.uint8))
    _refused(LlamaConfig, keep_bits=4)


@pytest.mark.gpu
def test_refusals():
    from aws_ofi_nccl_b200.ops import gemm, llm

    x = torch.ones(4, 64, device="cuda", dtype=BF)
    for bad in (x.float(), x.half(), x[:, :60], x[:, :0], x[0, 0]):
        _refused(llm.keep_rows8, bad)
        _refused(gemm.linear, bad, x, keep_bits=8)
    _refused(llm.keep_rows8, x.clone().requires_grad_(True))
    _refused(llm.swiglu, x[:, :24], keep_bits=8)     # halves of 12
    _refused(llm.swiglu, x[:, ::2], keep_bits=8)
    _refused(llm.swiglu_mlp, x, x, x[:, :30], keep_bits=8)
    codes, powers = llm.keep_rows8(x)
    for args in ((codes, powers[:3]), (codes, powers.int()), (codes, powers.cpu()), (codes.view(torch.uint8), powers), (codes[:, ::2], powers), (codes, powers[:, :1])):
        _refused(llm.kept_rows8, *args)
    y = llm.swiglu(x.clone().requires_grad_(True), keep_bits=8)
    _refused(torch.autograd.grad, y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for fn, args in ((gemm.linear, (dual, x)), (llm.swiglu, (dual,)), (llm.keep_rows8, (dual,))):
            _refused(fn, *args, **({} if fn is llm.keep_rows8 else dict(keep_bits=8)))


@pytest.mark.gpu
def test_captured_and_replayed():
    from aws_ofi_nccl_b200.ops import gemm, llm

    x = torch.randn(100, 64, device="cuda").to(BF).requires_grad_(True)
    w = torch.randn(128, 64, device="cuda").to(BF).requires_grad_(True)
    dy = torch.randn(100, 64, device="cuda").to(BF)

    def step():
        return torch.autograd.grad(llm.swiglu(gemm.linear(x, w, keep_bits=8), keep_bits=8), (x, w), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(torch.randn(100, 64, device="cuda"))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
