"""Attention beside its values: what it refuses, layouts, streams, captured calls, two calls at once, and the model that calls it."""
import pytest
import torch

from test_attention_gpu import U, _check, _inputs, _run

BF = torch.bfloat16


def _refused(fn, *args, error=(AssertionError, RuntimeError, ValueError, TypeError), **kw):
    with pytest.raises(error):
        fn(*args, **kw)


def test_refusals_without_a_gpu(built):
    from aws_ofi_nccl_b200.models.llama import LlamaConfig
    from aws_ofi_nccl_b200.ops.attention import attention

    q = torch.ones(1, 8, 2, 64, dtype=BF)
    _refused(attention, q, q, q)
    for kw in (dict(window=-1), dict(sinks=-1, window=4), dict(sinks=2)):
        _refused(LlamaConfig, **kw)


@pytest.mark.gpu
def test_refusals():
    from aws_ofi_nccl_b200.ops.attention import attention

    q, k, v, _ = _inputs(2, 16, 4, 2, 64)
    for args in ((q.float(), k, v), (q.half(), k.half(), v.half()), (q, k.float(), v), (q[0], k, v), (q, k[0], v[0]), (q, k[:1], v[:1]), (q, k[:, :8], v[:, :8]),
                 (q, k, v[:, :, :1]), (q[..., :32], k[..., :32], v[..., :32]), (q[:, :, :3], k, v), (q[:, :, :0], k, v), (q, k[:, :, :0], v[:, :, :0]),
                 (q.cpu(), k, v), (q, k.cpu(), v), (q, k, v.cpu())):
        _refused(attention, *args)
    for kw in (dict(window=-1), dict(sinks=-1), dict(sinks=3), dict(window=2, sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(scale=1e-60), dict(lengths=torch.tensor([16, 16])), dict(lengths=torch.tensor([16, 16], device="cuda")),
               dict(lengths=torch.tensor([16], dtype=torch.int32, device="cuda")), dict(lengths=torch.tensor([[16, 16]], dtype=torch.int32, device="cuda")),
               dict(lengths=torch.tensor([16, 0, 16], dtype=torch.int32, device="cuda")[::2])):
        _refused(attention, q, k, v, **kw)
    leaf = q.clone().requires_grad_(True)
    _refused(torch.autograd.grad, attention(leaf, k, v).sum(), leaf, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        _refused(attention, torch.autograd.forward_ad.make_dual(q, q), k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_layouts(hd):
    """Views of a fused projection, heads in front of tokens, every second token, rows off 16-byte boundaries, broadcast heads and gradients."""
    b, s, nq, nkv = 2, 150, 4, 2
    fused = torch.randn(b, s, nq + 2 * nkv, hd, device="cuda").to(BF)
    q, k, v = fused.split([nq, nkv, nkv], 2)
    do = torch.randn(b, s, nq, hd, device="cuda").to(BF)
    _check(q, k, v, do, window=40, sinks=2)
    t = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)   # noqa: E731
    _check(t(q), t(k), t(v), t(do))
    _check(fused[:, ::2, :nq], fused[:, ::2, nq:nq + nkv], fused[:, ::2, nq + nkv:], do[:, ::2], window=9)
    odd = torch.randn(1 + b * s * nq * hd, device="cuda").to(BF)[1:].view(b, s, nq, hd)
    _check(odd, k, v, odd)
    wide = torch.randn(b, s, nq, hd + 4, device="cuda").to(BF)[..., :hd]     # a pitch that is no multiple of 16 bytes
    _check(wide, k, v, wide)
    _check(q, k[:, :, :1].expand(-1, -1, nkv, -1), v, do[:, :1].expand(-1, s, -1, -1), window=33, sinks=33)
    _check(torch.randn(s, b, nq, hd, device="cuda").to(BF).transpose(0, 1), k, v, do)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 4, 2, 1, 64), (2, 0, 2, 1, 128)])
def test_nothing(shape):
    b, s, nq, nkv, hd = shape
    q, k, v, do = (torch.empty(b, s, h, hd, device="cuda", dtype=BF) for h in (nq, nkv, nkv, nq))
    for name, got in _run(q, k, v, do, window=3, sinks=1).items():
        assert got.shape == (k if name in ("dk", "dv") else q).shape


@pytest.mark.gpu
def test_only_what_is_asked_for():
    from aws_ofi_nccl_b200.ops.attention import attention

    ts = _inputs(1, 200, 2, 2, 64, seed=1)
    full = _run(*ts, window=50, sinks=1)
    for which in range(3):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate(ts[:3])]
        attention(*leaves, window=50, sinks=1).backward(ts[3])
        assert [t.grad is not None for t in leaves] == [i == which for i in range(3)]
        assert torch.equal(leaves[which].grad, full[("dq", "dk", "dv")[which]])
    with torch.no_grad():
        assert torch.equal(attention(*ts[:3], window=50, sinks=1), full["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(window=64, sinks=3)])
def test_the_same_bits_in_every_run_and_any_batch(kw):
    """Also with other work on the GPU, and for a sequence alone and in a batch."""
    ts = _inputs(3, 1300, 4, 1, 128, seed=2)
    first = _run(*ts, **kw)
    for _ in range(3):
        again = _run(*ts, **kw)
        assert all(torch.equal(first[n], again[n]) for n in first)
    alone = _run(*(t[1:2] for t in ts), **kw)
    for n in ("out", "dq"):
        assert torch.equal(alone[n], first[n][1:2])
    for n in ("dk", "dv"):   # a walk is split by what else there is to do: sums in another order, each rounded once
        assert ((alone[n].double() - first[n][1:2].double()).abs() <= 2 * U * first[n][1:2].double().abs() + 2.0 ** -16 * first[n].abs().max()).all()


@pytest.mark.gpu
def test_streams_and_two_calls_at_once():
    from aws_ofi_nccl_b200.ops.attention import attention

    sets = [_inputs(2, 700, 4, 2, 64, seed=s) for s in range(3)]
    want = [_run(*ts, window=100, sinks=5) for ts in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for ts, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(_run(*ts, window=100, sinks=5))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(a[n], b[n]) for n in a)
    # a tensor of another stream, waited for as usual
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = sets[0][0].clone()
    torch.cuda.current_stream().wait_stream(side)
    q.record_stream(torch.cuda.current_stream())
    assert torch.equal(attention(q, *sets[0][1:3], window=100, sinks=5), want[0]["out"])


@pytest.mark.gpu
def test_captured_and_replayed():
    """Two graphs of one size do not share anything, and lengths are read when a graph runs."""
    ts = _inputs(2, 900, 2, 1, 64, seed=4)
    n = torch.tensor([900, 333], dtype=torch.int32, device="cuda")
    static = [t.clone() for t in ts]
    from aws_ofi_nccl_b200.ops.attention import attention
    leaves = [t.requires_grad_(True) for t in static[:3]]
    step = lambda: torch.autograd.grad(attention(*leaves, window=64, sinks=2, lengths=n), leaves, static[3])   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    n.copy_(torch.tensor([17, 900], dtype=torch.int32))
    fresh = _inputs(2, 900, 2, 1, 64, seed=5)
    with torch.no_grad():
        for a, b in zip(static, fresh):
            a.copy_(b)
    for g in graphs:
        g.replay()
    want = _run(*fresh, window=64, sinks=2, lengths=n)
    for out in outs:
        assert all(torch.equal(a, want[k]) for a, k in zip(out, ("dq", "dk", "dv")))


@pytest.mark.gpu
def test_nan_and_infinity_are_seen_by_those_that_see_them():
    from aws_ofi_nccl_b200.ops.attention import attention

    q, k, v, _ = _inputs(1, 400, 1, 1, 64, seed=7)
    for value in (float("nan"), float("inf")):
        bad = k.clone()
        bad[0, 300, 0, 5] = value
        out = attention(q, bad, v, window=50)
        clean = attention(q, k, v, window=50)
        assert torch.equal(out[:, :300], clean[:, :300]) and torch.equal(out[:, 350:], clean[:, 350:])   # keys that are not seen weigh nothing
        if value != value:
            assert out[:, 300:350].isnan().all()
    bad = v.clone()
    bad[0, 300, 0, 5] = float("nan")
    out = attention(q, k, bad, window=50)
    assert out[:, 300:350, :, 5].isnan().all() and torch.equal(out[:, :256], clean[:, :256]) and torch.equal(out[:, 512:], clean[:, 512:])


@pytest.mark.gpu
def test_a_long_sequence_is_that_of_its_windows():
    """More tokens than 2^31 bytes of q hold: with a window rows are those of a slice that begins a window earlier."""
    from aws_ofi_nccl_b200.ops.attention import attention

    s, window = 300_000, 200
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(1, s, 32, 128, device="cuda", generator=g, dtype=BF)
    k, v = (torch.randn(1, s, 1, 128, device="cuda", generator=g, dtype=BF) for _ in range(2))
    out = attention(q, k, v, window=window)
    for at in (0, 131_072 - 50, 262_144 + 77, s - 300):
        lo = max(0, at - window) // 128 * 128   # the same tiles
        part = attention(q[:, lo:at + 300], k[:, lo:at + 300], v[:, lo:at + 300], window=window)
        assert torch.equal(out[:, at:at + 300], part[:, at - lo:])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(window=40, sinks=3), dict(keep_bits=8), dict(window=17, keep_bits=8)])
def test_model(kw):
    """The tiny model with a window and with activations in 8 bits: loss and gradients against the restatement in 32 bits.

    In bf16 each of some twenty roundings between a weight and the loss adds 2^-9 at random, together below 2^-6 of a gradient; twice that is allowed. Operands in
    8 bits are off by at most 2^-4, in the mean by 2^-5; gate and up count twice, in the activation and in its slope, so 2^-4 of a gradient; twice that, too."""
    import aws_ofi_nccl_b200.models.llama as L

    class Leaf:   # what the restatement makes of a parameter is the leaf itself
        def __init__(self, p):
            self.leaf = p.detach().float().requires_grad_(True)

        def detach(self):
            return self

        def float(self):
            return self.leaf

    cfg = L.LlamaConfig(vocab_size=1024, hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn=512, max_seq=128, **kw)
    model = L.Llama(cfg, device="cuda", seed=3)
    g = torch.Generator(device="cuda").manual_seed(0)
    ids, labels = (torch.randint(0, cfg.vocab_size, (2, 128), device="cuda", generator=g) for _ in range(2))
    loss = model.forward_loss(ids, labels)
    loss.backward()
    plain = L.Llama.__new__(L.Llama)
    plain.__dict__ = dict(model.__dict__, params={k: Leaf(p) for k, p in model.params.items()})
    want = L.reference_forward_loss(plain, ids, labels)
    want.backward()
    assert abs(loss.item() - want.item()) < 2.0 ** -5
    for name, p in model.params.items():
        right = plain.params[name].leaf.grad
        off = (p.main_grad.float() - right).norm() / right.norm()
        assert off <= (2.0 ** -3 if cfg.keep_bits == 8 else 2.0 ** -5), (name, off.item())


@pytest.mark.gpu
def test_trainer_steps_with_a_window():
    from aws_ofi_nccl_b200.models.llama import LlamaConfig
    from aws_ofi_nccl_b200.parallel.engine import Trainer

    cfg = LlamaConfig(vocab_size=1024, hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn=512, max_seq=128, window=32, sinks=2, keep_bits=8)
    tr = Trainer(cfg, device="cuda")
    ids, labels = (torch.randint(0, cfg.vocab_size, (2, 128)).pin_memory() for _ in range(2))
    before = tr.model.flat_params.clone()
    losses = [tr.step(ids, labels) for _ in range(2)]
    assert all(x == x and x < 20 for x in losses) and tr.model.flat_params.isfinite().all() and not torch.equal(before, tr.model.flat_params)


@pytest.mark.gpu
def test_traced():
    """The tracer records the operators of the native layers, attention and those that keep 8 bits among them."""
    from aws_ofi_nccl_b200.ops import gemm, llm
    from aws_ofi_nccl_b200.ops.attention import attention

    q, k, v, _ = _inputs(1, 130, 2, 1, 64, seed=8)
    w = torch.randn(256, 128, device="cuda").to(BF)

    def step(q, k, v):
        o = attention(q, k, v, window=30, sinks=1).reshape(130, 128)
        return llm.swiglu(gemm.linear(o, w, keep_bits=8), keep_bits=8)

    traced = torch.jit.trace(step, (q, k, v), check_trace=False)
    other = _inputs(1, 130, 2, 1, 64, seed=9)[:3]
    assert torch.equal(traced(*other), step(*other))


@pytest.mark.gpu
@pytest.mark.parametrize("b, s, nq, nkv, window, sinks", [(1, 1100, 8, 8, 130, 3), (3, 2100, 3, 3, 0, 0), (5, 640, 8, 2, 64, 1), (40, 64, 8, 4, 20, 2), (1, 6000, 5, 1, 700, 40), (40, 700, 8, 8, 20, 2),
                                                           (1, 2000, 1, 1, 1, 1900)])
def test_more_tiles_than_ctas(b, s, nq, nkv, window, sinks):
    """CTAs that take several tiles, of ragged sequences and of full ones, empty ones among them."""
    q, k, v, do = _inputs(b, s, nq, nkv, 64, seed=s)
    _check(q, k, v, do, window=window, sinks=sinks)
    n = torch.tensor([(s * (3 * i + 1) // (2 * b + 1)) % (s + 1) if i % 4 != 2 else 0 for i in range(b)], dtype=torch.int32, device="cuda")
    for t in (q, k, v, do):
        for i, at in enumerate(n.tolist()):
            t[i, at:] = float("nan")
    _check(q, k, v, do, window=window, sinks=sinks, lengths=n)


def test_c_entries_refuse_what_they_cannot_number(built):
    """Sizes whose products pass 32 bits, null and unaligned pointers, strides off 16 bytes: the code for a bad argument in front of any launch, with addresses
    that nothing may touch."""
    import ctypes as C

    from aws_ofi_nccl_b200.ops import _lib

    class Part(C.Structure):
        _fields_ = [("data", C.c_void_p), ("batch", C.c_longlong), ("token", C.c_longlong), ("head", C.c_longlong)]

    class Args(C.Structure):
        _fields_ = ([(n, Part) for n in ("q", "k", "v", "dout")] + [(n, C.c_void_p) for n in ("out", "rest", "lse", "delta", "sums", "dq", "dk", "dv", "lengths")] +
                    [(n, C.c_int) for n in ("B", "S", "nq", "nkv", "hd", "window", "sinks")] + [("scale", C.c_float)])

    lib, bad, at = _lib.load(), 10001, 1 << 20

    def args(**kw):
        a = Args(B=1, S=16, nq=2, nkv=1, hd=64, scale=0.125)
        for n in ("q", "k", "v", "dout"):
            setattr(a, n, Part(at, 16 * 128, 128, 64))
        for n in ("out", "lse", "delta", "dq", "dk", "dv"):
            setattr(a, n, at)
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    for kw in (dict(B=1 << 20, nq=1 << 12, nkv=1 << 12), dict(B=1 << 16, nq=1 << 16, nkv=1), dict(B=1 << 15, nq=1 << 15), dict(B=1 << 10, nq=1 << 10, S=1 << 18), dict(S=0),
               dict(S=(1 << 30) + 1), dict(B=0), dict(nkv=0), dict(nq=0), dict(nq=3, nkv=2), dict(hd=96), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
               dict(scale=float("nan")), dict(out=None), dict(lse=None), dict(out=at + 2), dict(rest=at + 8), dict(q=Part(None, 2048, 128, 64)),
               dict(k=Part(at + 8, 2048, 128, 64)), dict(v=Part(at, 2048, 100, 64)), dict(v=Part(at, 2048, 0, 64))):
        a = args(**kw)
        assert lib.b200_attention_fwd(C.byref(a), None) == bad, kw
        assert lib.b200_attention_bwd(C.byref(a), None, None) == bad, kw
    for kw in (dict(delta=None), dict(dv=None), dict(dq=at + 8), dict(dout=Part(at, 2048, 128, 60))):
        a = args(**kw)
        assert lib.b200_attention_bwd(C.byref(a), None, None) == bad, kw
    vp, ll, i = C.c_void_p, C.c_longlong, C.c_int
    p, odd = vp(at), vp(at + 2)
    for rows, width in ((-1, 64), (4, 0), (4, 12), (4, -8), (4, (1 << 29) + 8)):
        assert lib.b200_keep8(p, ll(width), p, p, ll(rows), i(width), None) == bad
        for call in (lib.b200_kept8,):
            assert call(p, p, p, ll(rows), i(width), None) == bad
        for call in (lib.b200_swiglu_keep8, lib.b200_swiglu_bwd8, lib.b200_swiglu_kept8):
            assert call(p, p, p, p, ll(rows), i(width), None) == bad
    assert lib.b200_keep8(None, ll(64), p, p, ll(4), i(64), None) == bad
    assert lib.b200_keep8(p, ll(60), p, p, ll(4), i(64), None) == bad
    assert lib.b200_keep8(p, ll(64), odd, p, ll(4), i(64), None) == bad
    assert lib.b200_kept8(p, None, p, ll(4), i(64), None) == bad
    assert lib.b200_swiglu_keep8(p, odd, p, p, ll(4), i(64), None) == bad
    assert lib.b200_swiglu_bwd8(odd, p, p, p, ll(4), i(64), None) == bad


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, sinks", [(150, 3), (150, 40), (20, 17), (300, 150)])
def test_what_is_not_finite_stays_in_its_sequence(window, sinks, hd):
    """CTAs take items of several sequences one after the other: nothing of one whose keys, values or gradients are NaN is left for the next."""
    q, k, v, do = _inputs(24, 900, 4, 2, hd, seed=3)
    want = _run(q, k, v, do, window=window, sinks=sinks)
    for t in (q, k, v, do):
        t[::3] = float("nan")
    got = _run(q, k, v, do, window=window, sinks=sinks)
    for name in want:
        assert all(torch.equal(got[name][n::3], want[name][n::3]) for n in (1, 2)) and got[name][::3].isnan().all()
