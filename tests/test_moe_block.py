"""A mixture-of-experts block on one GPU as it is used: norm, tokens to their experts and back, the optimizer's step; and what its operators refuse."""
import pytest
import torch

BF = torch.bfloat16


def _refused(fn, *args, **kw):
    with pytest.raises((AssertionError, ValueError, ZeroDivisionError, TypeError)):
        fn(*args, **kw)


# ------------------------------------------------------------------ refusals, before anything is launched
def test_what_is_not_on_a_gpu_is_refused(built):
    from aws_ofi_nccl_b200.ops import llm, moe

    x, w = torch.zeros(4, 128, dtype=BF), torch.ones(128, dtype=BF)
    _refused(llm.rmsnorm_fp8, x, w)
    _refused(moe.expert_order, torch.zeros(4, 2, dtype=torch.int32), 4)
    order = moe.ExpertOrder(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(5, dtype=torch.int32))
    _refused(moe.permute_tokens, x, order)
    _refused(moe.unpermute_tokens, torch.zeros(8, 128, dtype=BF), order, torch.zeros(4, 2))
    p = [torch.zeros(64)]
    hyper = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1)
    for bits in (8, 32):
        _refused(llm.adamw_step_many, p, p, **llm.adamw_states(p, bits=bits), **hyper)
    _refused(llm.adamw_states, p, bits=16)


def test_the_layer_without_a_communicator_sends_no_fp8(built):
    from aws_ofi_nccl_b200.models.moe import MoELayer

    _refused(MoELayer, None, 8, 64, 64, 4, 2, fp8_dispatch=True, device="cpu")


def test_states_have_the_parameters_shapes():
    from aws_ofi_nccl_b200.ops import llm
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    params = [torch.zeros(3, 100, dtype=BF), torch.zeros(7), torch.zeros(0)]
    eight = llm.adamw_states(params, bits=8, master=True)
    assert [t.dtype for t in eight["m"] + eight["v"]] == [torch.float8_e4m3fn] * 6 and [t.shape for t in eight["v"]] == [p.shape for p in params]
    assert [t.numel() for t in eight["m_scale"]] == [2, 1, 0] and [t is None for t in eight["master"]] == [False, True, True]
    assert llm.adamw_states(params)["m_scale"] is None
    a, b = AdamW(params, bits=8), AdamW(params, bits=32)
    with pytest.raises(ValueError):
        a.load_state_dict(b.state_dict())
    with pytest.raises(ValueError):
        a.load_state_dict(AdamW(params[:2], bits=8).state_dict())
    a.state["m_scale"][0].fill_(3)
    a.step_count = 5
    c = AdamW(params, bits=8)
    c.load_state_dict(a.state_dict())
    assert c.step_count == 5 and (c.state["m_scale"][0] == 3).all()


@pytest.mark.gpu
def test_other_types_shapes_and_devices_are_refused():
    from aws_ofi_nccl_b200.ops import llm, moe

    x, w = torch.ones(4, 256, device="cuda", dtype=BF), torch.ones(256, device="cuda", dtype=BF)
    for args in ((x.float(), w), (x.half(), w), (x, w.float()), (x, w[:128]), (x, w.cpu()), (x[:, :100], w[:100]), (x[:, :0], w[:0])):
        _refused(llm.rmsnorm_fp8, *args)
    for kw in (dict(residual=x[:3]), dict(residual=x.float()), dict(residual=x.cpu()), dict(group=64), dict(group=-1)):
        _refused(llm.rmsnorm_fp8, x, w, **kw)
    _refused(llm.rmsnorm_fp8, x[:, :192], w[:192], group=128)
    _refused(llm.rmsnorm_fp8, torch.ones(1, 16392, device="cuda", dtype=BF), torch.ones(16392, device="cuda", dtype=BF))
    for t in (dict(x=x.clone().requires_grad_(True), weight=w), dict(x=x, weight=w.clone().requires_grad_(True))):
        _refused(llm.rmsnorm_fp8, **t)
        with torch.no_grad():
            llm.rmsnorm_fp8(**t)

    idx = torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    for args in ((idx.float(), 4), (idx.short(), 4), (idx[:, 0], 4), (idx.t(), 4), (idx[:, :0], 4), (idx, 0), (idx, -1), (idx, 1025), (idx.cpu(), 4)):
        _refused(moe.expert_order, *args)
    order = moe.expert_order(idx, 4)
    scale = torch.ones(4, 2, device="cuda")
    eight = x.to(torch.float8_e4m3fn)
    for args in ((x.half(), order), (x[:3], order), (x[0], order), (x.cpu(), order), (x[:, :0], order), (x, order, scale),
                 (eight, order, scale[:3]), (eight, order, scale.half()), (eight, order, scale.t()), (eight, order, scale.cpu()),
                 (x, order._replace(row_of=order.row_of.long())), (x, order._replace(row_of=order.row_of.t().contiguous().t())),
                 (x, order._replace(row_of=order.row_of.cpu())), (eight, order, scale.clone().requires_grad_(True))):
        _refused(moe.permute_tokens, *args)
    rows, weights = torch.ones(8, 256, device="cuda", dtype=BF), torch.ones(4, 2, device="cuda")
    for args in ((rows[:7], order, weights), (rows.half(), order, weights), (rows, order, weights[:3]), (rows, order, weights.bfloat16()),
                 (rows, order, weights.cpu()), (rows.to(torch.float8_e4m3fn), order, weights)):
        _refused(moe.unpermute_tokens, *args)


@pytest.mark.gpu
def test_optimizer_refuses_before_it_writes():
    from aws_ofi_nccl_b200.ops import llm

    hyper = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1)
    p = [torch.ones(300, device="cuda", dtype=BF), torch.ones(4, 70, device="cuda")]
    g = [torch.ones_like(t) for t in p]

    def both(bits, params=p, grads=g, **changed):
        state = llm.adamw_states(p, bits=bits, master=True)
        args = {**state, **hyper, **changed}
        _refused(llm.adamw_step_many, params, grads, **args)
        assert all((t == 1).all() for t in p + g)

    for bits in (8, 32):
        s = llm.adamw_states(p, bits=bits, master=True)
        both(bits, params=p[:1])
        both(bits, grads=g[:1])
        both(bits, params=[p[0].half(), p[1]])
        both(bits, params=[p[0], p[1].t()])
        both(bits, params=[p[0], p[1].cpu()])
        both(bits, grads=[g[0], g[1].half()])
        both(bits, grads=[g[0], g[1][:3]])
        both(bits, grads=[g[0], g[1].t()])
        both(bits, grads=[g[0].cpu(), g[1]])
        both(bits, m=s["m"][:1])
        both(bits, v=[s["v"][0], s["v"][0]])
        both(bits, m=[s["m"][0], s["m"][1].half()])
        both(bits, master=[None, p[1].clone()])          # a copy of a parameter in 32 bits
        both(bits, master=[p[0].clone(), None])          # a copy in 16
        both(bits, master=[torch.ones(299, device="cuda"), None])
        both(bits, weight_decay=[0.1])
        both(bits, step=0)
        both(bits, lr=-1.0)
        both(bits, beta1=1.0)
        both(bits, beta2=-0.1)
        # memory that is written twice
        same = torch.ones(300, device="cuda", dtype=BF)
        twin = llm.adamw_states([same, same], bits=bits)
        _refused(llm.adamw_step_many, [same, same], [same.clone(), same.clone()], **twin, **hyper)
        _refused(llm.adamw_step_many, [same[:200], same[100:]], [same[:200].clone(), same[100:].clone()],
                 **llm.adamw_states([same[:200], same[100:]], bits=bits), **hyper)
        _refused(llm.adamw_step_many, [same], [same], **llm.adamw_states([same], bits=bits), **hyper)   # its own gradient, to be zeroed
        twin["m"][1] = twin["m"][0]
        _refused(llm.adamw_step_many, [same, same.clone()], [same.clone(), same.clone()], **twin, **hyper)
        assert (same == 1).all()
    eight = llm.adamw_states(p, bits=8)
    both(32, m_scale=eight["m_scale"])
    both(32, m_scale=eight["m_scale"], v_scale=eight["v_scale"])
    both(8, m_scale=None)
    both(8, m_scale=None, v_scale=None)
    both(8, v_scale=eight["v_scale"][:1])
    both(8, m_scale=[eight["m_scale"][0][:1], eight["m_scale"][1]])
    both(8, v=llm.adamw_states(p, bits=32)["v"])


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps_of_a_layer(bits):
    """Norm, layer and optimizer: output and gradients against 64 bits from the same weights, then parameters that move."""
    from aws_ofi_nccl_b200.models.moe import MoELayer
    from aws_ofi_nccl_b200.ops import llm
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    T, H, FF, E, k = 200, 256, 128, 6, 2
    layer = MoELayer(None, T, H, FF, E, k, seed=1)
    g = torch.Generator(device="cuda").manual_seed(4)
    norm = (1 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(BF).requires_grad_(True)
    opt = AdamW([norm, *layer.parameters()], bits=bits)
    for step in range(2):
        x = torch.randn(T + step, H, device="cuda", generator=g).to(BF).requires_grad_(True)   # any number of tokens
        d = torch.randn(T + step, H, device="cuda", generator=g).to(BF)
        n, _ = llm.rmsnorm(x, norm)
        idx, w = layer.route(n)
        out = layer(n)
        out.backward(d)

        P = [p.detach().double().requires_grad_(True) for p in (x, norm, layer.router)]
        gu = [p.detach().double().requires_grad_(True) for p in layer.w_gate_up]
        dn = [p.detach().double().requires_grad_(True) for p in layer.w_down]
        N = P[0] * torch.rsqrt(P[0].square().mean(-1, keepdim=True) + 1e-5) * P[1]
        probs = torch.softmax(N @ P[2].t(), -1)
        W = probs.gather(1, idx.long())
        want = torch.zeros_like(N)
        for e in range(E):
            a, b = (N @ gu[e].t()).split(FF, -1)
            want = want + ((idx == e) * W).sum(1, keepdim=True) * ((torch.nn.functional.silu(a) * b) @ dn[e].t())
        want.backward(d.double())
        near = lambda a, b: (a.double() - b).norm() <= 0.02 * b.norm()   # noqa: E731  a dozen roundings to bf16, 2^-8 each at most: 0.047 in the worst case, 0.014 as independent ones
        assert near(out.detach(), want.detach()) and near(x.grad, P[0].grad) and near(norm.grad, P[1].grad) and near(layer.router.grad, P[2].grad)
        for got, ref in zip([*layer.w_gate_up, *layer.w_down], gu + dn):
            assert got.grad is None or near(got.grad, ref.grad)
        # what moves is the copy in 32 bits: half a step of bf16 is 2^-8 near one, of lr 3e-4 nothing is left of a norm's weight
        held = [c if c is not None else p.detach() for p, c in zip(opt.params, opt.state["master"])]
        before = [t.clone() for t in held]
        chosen = [p.grad is not None for p in opt.params]
        opt.step()
        moved = [not torch.equal(t, q) for t, q in zip(held, before)]
        assert all(torch.equal(p.detach(), t.to(p.dtype)) for p, t in zip(opt.params, held))
        assert moved == chosen and all((p.grad == 0).all() for p in opt.params if p.grad is not None)
        for p in opt.params:
            p.grad = None


@pytest.mark.gpu
@pytest.mark.parametrize("master", [False, True])
def test_trainer_with_moments_in_8_bits(tmp_path, master):
    """Each step is adamw_step_many on the flat buffers; a checkpoint holds the scales and is none of the trainer with 32 bits."""
    from aws_ofi_nccl_b200.models.llama import LlamaConfig
    from aws_ofi_nccl_b200.ops import llm
    from aws_ofi_nccl_b200.parallel.engine import OptimConfig, Trainer

    cfg = LlamaConfig.tiny()
    oc = OptimConfig(state_bits=8, master_weights=master)
    tr = Trainer(cfg, oc, device="cuda")
    assert tr.m.dtype == tr.v.dtype == torch.float8_e4m3fn and tr.m_scale.numel() == -(-tr.m.numel() // 256)
    ids, lbl = (torch.randint(0, cfg.vocab_size, (2, 128), device="cuda") for _ in range(2))
    calls = []
    step_many = llm.adamw_step_many

    def watched(params, grads, m, v, ms, vs, masters, **hyper):
        kept = [[t.clone() if t is not None else None for t in x] for x in (params, grads, m, v, ms, vs, masters)]
        step_many(params, grads, m, v, ms, vs, masters, **hyper)
        step_many(*kept, **hyper)
        for now, then in zip((params, grads, m, v, ms, vs, masters), kept):
            for a, b in zip(now, then):
                assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        calls.append(hyper["step"])

    llm.adamw_step_many = watched
    try:
        for _ in range(2):
            before = tr.model.flat_params.clone()
            assert tr.step_device(ids, lbl).isfinite()
            assert not torch.equal(before, tr.model.flat_params) and (tr.model.flat_grads == 0).all()
    finally:
        llm.adamw_step_many = step_many
    assert calls == [1, 2]
    path = tmp_path / "ckpt.pt"
    torch.save(tr.state_dict(), path)
    other = Trainer(cfg, oc, device="cuda", seed=9)
    other.load_state_dict(torch.load(path, weights_only=False))
    for name in ("m", "v", "m_scale", "v_scale"):
        assert torch.equal(getattr(tr, name).view(torch.uint8), getattr(other, name).view(torch.uint8))
    assert torch.equal(tr.model.flat_params, other.model.flat_params) and other.step_count == 2
    for a, b in ((tr, Trainer(cfg, device="cuda")), (Trainer(cfg, device="cuda"), tr)):
        with pytest.raises(ValueError):
            b.load_state_dict(a.state_dict())


@pytest.mark.gpu
def test_layer_without_a_communicator_equals_the_one_with_it():
    """The same weights and tokens: expert outputs are the same rows in another order, sums within bf16's rounding."""
    import torch.distributed as dist

    from aws_ofi_nccl_b200.models.moe import MoELayer
    from aws_ofi_nccl_b200.parallel.symm import Communicator

    own = not dist.is_initialized()
    if own:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    comm = Communicator(dist.group.WORLD, 16 << 20, torch.device("cuda", 0), wait_limit_s=2.0)
    try:
        T, H, FF, E, k = 96, 256, 128, 4, 2
        a, b = MoELayer(comm, T, H, FF, E, k, seed=3), MoELayer(None, T, H, FF, E, k, seed=3)
        x, d = (torch.randn(T, H, device="cuda").to(BF) for _ in range(2))
        outs, grads = [], []
        for layer in (a, b):
            leaf = x.clone().requires_grad_(True)
            out = layer(leaf)
            outs.append(out.detach().double())
            grads.append(torch.autograd.grad(out, [leaf, layer.router], d))
        # each sum is rounded once to bf16, 2^-8 of it at most, on either side
        assert ((outs[0] - outs[1]).abs() <= 2 * 2.0 ** -8 * outs[0].abs() + 1e-6).all()
        for one, other in zip(*grads):
            assert (one.double() - other.double()).norm() <= 2 ** -6 * one.double().norm()
    finally:
        comm.close()
        if own:
            dist.destroy_process_group()


@pytest.mark.gpu
def test_serving_in_8_bits():
    """Norm with row scales, 8-bit rows to their experts, fp8 products, back: against 64 bits of what the codes stand for."""
    from aws_ofi_nccl_b200.ops import gemm, llm, moe

    T, H, E, k = 1200, 512, 3, 1
    g = torch.Generator(device="cuda").manual_seed(2)
    x, res = (torch.randn(T, H, device="cuda", generator=g).to(BF) for _ in range(2))
    norm = torch.ones(H, device="cuda", dtype=BF)
    weights = [gemm.quantize_rows_fp8((torch.randn(256, H, device="cuda", generator=g) / H ** 0.5).to(BF)) for _ in range(E)]
    idx = (torch.arange(T, device="cuda", dtype=torch.int32) % E).view(T, k)
    idx[::50] = -1   # padding
    w = torch.rand(T, k, device="cuda", generator=g)
    q, s, h = llm.rmsnorm_fp8(x, norm, residual=res)
    order = moe.expert_order(idx, E)
    rows, row_scale = moe.permute_tokens(q, order, s)
    off = order.offsets.tolist()
    y = torch.full((T * k, 256), float("nan"), device="cuda", dtype=BF)
    for e in range(E):
        assert off[e + 1] - off[e] >= 256
        gemm.gemm_fp8(rows[off[e]:off[e + 1]], weights[e][0], row_scale[off[e]:off[e + 1]], weights[e][1], out=y[off[e]:off[e + 1]])
    out = moe.unpermute_tokens(y, order, w)
    a = q.double() * s.double()[:, None]
    want, mag = torch.zeros(T, 256, device="cuda", dtype=torch.float64), torch.zeros(T, 256, device="cuda", dtype=torch.float64)
    for e in range(E):
        b = weights[e][0].double() * weights[e][1].double()[:, None]
        gate = (idx == e) * w.double()
        want += gate * (a @ b.t())
        mag += gate * (a.abs() @ b.abs().t())
    # two roundings to bf16, and the tensor core's sums, whose terms keep 13 bits below the largest at the least
    assert ((out.double() - want).abs() <= 2.1 * 2.0 ** -8 * want.abs() + 2.0 ** -12 * mag).all()
    assert (out[::50] == 0).all()


@pytest.mark.gpu
def test_captured_forward_and_backward_pass():
    """Order, rows, sums and gradients of new inputs in a replayed graph; leaves of its own, none of which an eager graph holds."""
    from aws_ofi_nccl_b200.ops import moe

    T, k, E, H = 64, 4, 8, 256
    idx = torch.randint(0, E, (T, k), device="cuda", dtype=torch.int32)
    x, d = (torch.randn(T, H, device="cuda").to(BF) for _ in range(2))
    w = torch.rand(T, k, device="cuda")

    def step(x, w):
        order = moe.expert_order(idx, E)
        out = moe.unpermute_tokens(moe.permute_tokens(x, order), order, w)
        return out.detach(), *torch.autograd.grad(out, (x, w), d)

    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*leaves)
    for seed in range(2):
        idx.copy_(torch.randint(0, E, (T, k), device="cuda", dtype=torch.int32))
        with torch.no_grad():
            leaves[0].normal_()
            leaves[1].uniform_()
        graph.replay()
        want = step(*(t.detach().clone().requires_grad_(True) for t in leaves))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_more_than_two_to_the_31st_elements():
    """Rows, norms and parameters whose last elements lie beyond numbers of 32 bits: the same as of a slice by itself."""
    from aws_ofi_nccl_b200.ops import llm, moe

    T, k, H = 40001, 8, 8192
    idx = torch.randint(0, 5, (T, k), device="cuda", dtype=torch.int32)
    x = torch.randn(T, H, device="cuda", dtype=BF)
    order = moe.expert_order(idx, 5)
    rows = moe.permute_tokens(x, order)
    assert rows.numel() > 2 ** 31
    at = order.row_of[-3:].reshape(-1).long()
    assert torch.equal(rows[at], x[-3:].repeat_interleave(k, 0))
    token = torch.empty(T * k, device="cuda", dtype=torch.long)
    token[order.row_of.reshape(-1).long()] = torch.arange(T * k, device="cuda") // k
    assert torch.equal(rows[-5:], x[token[-5:]])
    w = torch.full((T, k), 0.125, device="cuda", requires_grad=True)
    out = moe.unpermute_tokens(rows, order, w)
    assert torch.equal(out.detach(), x)   # eighths of the same number: no rounding
    rows.requires_grad_(True)
    drows, dw = torch.autograd.grad(moe.unpermute_tokens(rows, order, w), (rows, w), x)
    assert torch.equal(drows[at], (x[-3:].float() / 8).to(BF).repeat_interleave(k, 0))
    want = x[-3:].double().square().sum(-1, keepdim=True)
    assert ((dw[-3:].double() - want).abs() <= (H + 8) * 2.0 ** -24 * want).all()
    del rows, drows, out
    wide = x.repeat(7, 1)
    assert wide.numel() > 2 ** 31
    norm = torch.ones(H, device="cuda", dtype=BF)
    for group in (0, 128):
        q, s, h = llm.rmsnorm_fp8(wide, norm, residual=wide, group=group)
        q1, s1, h1 = llm.rmsnorm_fp8(x[-3:], norm, residual=x[-3:], group=group)
        assert torch.equal(q[-3:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-3:], s1) and torch.equal(h[-3:], h1)
    del wide, q, h, x
    n, tail = 2 ** 31 + 2 ** 20 + 77, 2 ** 20 + 77
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, zero_grad=False)
    for bits in (8, 32):
        p = torch.empty(n, device="cuda", dtype=BF)
        p[-tail:].normal_()
        g = torch.empty(n, device="cuda", dtype=BF)
        g[-tail:].normal_()
        p[:-tail] = 0
        g[:-tail] = 0
        small, gs = p[-tail:].clone(), g[-tail:].clone()
        state, other = llm.adamw_states([p], bits=bits), llm.adamw_states([small], bits=bits)
        llm.adamw_step_many([p], [g], **state, **hyper, step=1)
        llm.adamw_step_many([small], [gs], **other, **hyper, step=1)
        assert torch.equal(p[-tail:], small) and (p[:1000] == 0).all() and (p[2 ** 31 - 1000:2 ** 31] == 0).all()
        if bits == 32:
            assert torch.equal(state["v"][0][-tail:], other["v"][0])
        else:
            assert torch.equal(state["v_scale"][0][-(-(-tail // 256)):], other["v_scale"][0])
        del p, g, state


@pytest.mark.gpu
def test_other_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from aws_ofi_nccl_b200.ops import llm, moe

    with torch.cuda.device(0):
        x = torch.randn(8, 256, device="cuda:1").to(BF)
        q, s, _ = llm.rmsnorm_fp8(x, torch.ones(256, device="cuda:1", dtype=BF))
        order = moe.expert_order(torch.zeros(8, 2, device="cuda:1", dtype=torch.int32), 3)
        rows = moe.permute_tokens(x, order)
        p = [torch.zeros(300, device="cuda:1")]
        llm.adamw_step_many(p, [torch.ones(300, device="cuda:1")], **llm.adamw_states(p), lr=1.0, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1)
        assert q.device == s.device == rows.device == x.device and (p[0] != 0).all()


@pytest.mark.gpu
def test_traced():
    """torch.jit.trace records the operators, not the allocation of their outputs."""
    from aws_ofi_nccl_b200.ops import llm, moe

    idx = torch.randint(0, 4, (16, 2), device="cuda", dtype=torch.int32)
    w = torch.ones(256, device="cuda", dtype=BF)

    def block(x, gate):
        order = moe.expert_order(idx, 4)
        q, s, _ = llm.rmsnorm_fp8(x, w)
        return moe.unpermute_tokens(moe.permute_tokens(x, order), order, gate), q.float() * s[:, None]

    x, gate = torch.randn(16, 256, device="cuda").to(BF), torch.rand(16, 2, device="cuda")
    traced = torch.jit.trace(block, (x, gate), check_trace=False)
    x, gate = torch.randn(16, 256, device="cuda").to(BF), torch.rand(16, 2, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(traced(x, gate), block(x, gate)))


FIRST_CALLS = """
import torch
from aws_ofi_nccl_b200.ops import _lib, llm, moe

idx = torch.randint(0, 50, (4000, 3), device="cuda", dtype=torch.int32)   # a cluster's order
x, w, norm = torch.randn(4000, 520, device="cuda").bfloat16(), torch.rand(4000, 3, device="cuda"), torch.ones(520, device="cuda").bfloat16()
p, g = ([torch.full((1000,), v, device="cuda") for _ in range(20)] for v in (0.0, 1.0))
state = llm.adamw_states(p, bits=8)


def step():
    order = moe.expert_order(idx, 50)
    rows = moe.permute_tokens(x, order)
    return (*order, rows, moe.unpermute_tokens(rows, order, w), *llm.rmsnorm_fp8(x, norm, residual=x))


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
    llm.adamw_step_many(p, g, **state, lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1, zero_grad=False)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, step()))
assert all(torch.equal(t, p[0]) and (t != 0).all() for t in p) and _lib.read_status() == 0
"""


@pytest.mark.gpu
def test_a_process_whose_first_calls_are_captured():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_chains_see_what_the_call_before_wrote(captured):
    """Every operator directly behind the one whose output it takes, over and over: as with the device idle between them."""
    from aws_ofi_nccl_b200.ops import gemm, llm, moe

    g = torch.Generator(device="cuda").manual_seed(6)
    T, H, E, k = 900, 512, 12, 3
    norm, w = torch.ones(H, device="cuda", dtype=BF), torch.rand(T, k, device="cuda", generator=g)
    weight = (torch.randn(H, H, device="cuda", generator=g) / H ** 0.5).to(BF)
    wq, ws = gemm.quantize_rows_fp8(weight)

    def run(idx, x, p, state, pause):
        for step in range(1, 6):
            q, s, h = llm.rmsnorm_fp8(x, norm, residual=x)
            pause()
            y = gemm.gemm_fp8(q, wq, s, ws)
            pause()
            order = moe.expert_order(idx, E)
            pause()
            rows = moe.permute_tokens(y, order)
            pause()
            rows = gemm.linear(rows, weight)
            pause()
            x = moe.unpermute_tokens(rows, order, w)
            pause()
            llm.adamw_step_many([p], [x], **state, lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=step, zero_grad=False)
            pause()
            idx = (idx + order.offsets[1]) % E   # of what the order has just written
            x = (x + p).to(BF)
            pause()
        return idx, x, p, state["m"][0].view(torch.uint8), state["v"][0].view(torch.uint8)

    def inputs():
        gen = torch.Generator(device="cuda").manual_seed(9)
        p = torch.randn(T, H, device="cuda", generator=gen).to(BF)
        idx = torch.randint(0, E, (T, k), device="cuda", generator=gen, dtype=torch.int32)
        return idx, torch.randn(T, H, device="cuda", generator=gen).to(BF), p, llm.adamw_states([p], bits=8)

    want = run(*inputs(), torch.cuda.synchronize)
    if captured:
        args = inputs()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*inputs(), lambda: None)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(*args, lambda: None)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    else:
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(run(*inputs(), lambda: None), want))
