"""What the operators of a mixture-of-experts block say and do at their edges: derivatives that they do not have, experts that sit steps out, and
moments in 8 bits beyond their first step."""
import math

import pytest
import torch

BF = torch.bfloat16


# ------------------------------------------------------------------ forward-mode derivatives
@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """A dual tensor requires no gradient, but its tangent would be lost: every operator that takes one says so, in a backward pass too."""
    import torch.autograd.forward_ad as fwd

    from aws_ofi_nccl_b200.ops import llm, moe

    T, k, E, H = 6, 2, 4, 256
    x, norm = torch.randn(T, H, device="cuda").to(BF), torch.ones(H, device="cuda", dtype=BF)
    order = moe.expert_order(torch.randint(0, E, (T, k), device="cuda", dtype=torch.int32), E)
    rows, w = torch.randn(T * k, H, device="cuda"), torch.rand(T, k, device="cuda")
    calls = [
        (lambda t: moe.permute_tokens(t, order), x),
        (lambda t: moe.unpermute_tokens(t, order, w), rows),
        (lambda t: moe.unpermute_tokens(t, order), rows),
        (lambda t: moe.unpermute_tokens(rows, order, t), w),
        (lambda t: llm.rmsnorm_fp8(t, norm), x),
        (lambda t: llm.rmsnorm_fp8(x, norm, residual=t), x),
        (lambda t: llm.rmsnorm_fp8(x, t), norm),
    ]
    leaf, gate, d = rows.clone().requires_grad_(True), w.clone().requires_grad_(True), torch.randn(T, H, device="cuda")
    weighted, plain = moe.unpermute_tokens(leaf, order, gate), moe.unpermute_tokens(leaf, order)
    xl = x.clone().requires_grad_(True)
    there = moe.permute_tokens(xl, order)
    calls += [(lambda t: torch.autograd.grad(weighted, (leaf, gate), t, retain_graph=True), d),
              (lambda t: torch.autograd.grad(plain, leaf, t, retain_graph=True), d),
              (lambda t: torch.autograd.grad(there, xl, t, retain_graph=True), torch.ones_like(there))]
    for fn, t in calls:
        with fwd.dual_level():
            dual = fwd.make_dual(t.detach(), torch.ones_like(t))
            with pytest.raises((RuntimeError, AssertionError, NotImplementedError)):
                fn(dual)
            with torch.no_grad(), pytest.raises((RuntimeError, AssertionError, NotImplementedError)):   # which turns backward passes off alone
                fn(dual)
            with fwd._set_fwd_grad_enabled(False):   # asked for: the value by itself
                fn(dual)
        fn(t.detach())   # outside of the level there is no tangent


# ------------------------------------------------------------------ the optimizer's sparse steps
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_experts_that_no_token_chose_stay_as_they_are(bits, master):
    """The loop as it is documented, without a gradient cleared by hand: an expert of the first step that sits out the second"""
    from aws_ofi_nccl_b200.models.moe import MoELayer
    from aws_ofi_nccl_b200.parallel.engine import AdamW, OptimConfig

    layer = MoELayer(None, 0, 256, 128, 4, 1, seed=2)
    opt = AdamW(layer.parameters(), OptimConfig(master_weights=master, lr=1e-2), bits=bits)
    x = torch.randn(64, 256, device="cuda").to(BF)

    def step(chosen):
        idx = torch.tensor(chosen, device="cuda", dtype=torch.int32).repeat(64 // len(chosen)).view(-1, 1)
        layer.route = lambda t: (idx, torch.ones(64, 1, device="cuda"))
        layer(x).backward(torch.randn(64, 256, device="cuda").to(BF))
        opt.step()

    step([0, 1])
    ones = [i for i, p in enumerate(opt.params) if p is layer.w_gate_up[1] or p is layer.w_down[1]]
    zeros = [i for i, p in enumerate(opt.params) if p is layer.w_gate_up[0] or p is layer.w_down[0]]
    assert len(ones) == len(zeros) == 2

    def kept(which):
        lists = [opt.params] + [s for s in opt.state.values() if s is not None]
        return [s[i].detach().clone() for s in lists for i in which if s[i] is not None]

    sat_out, took_part = kept(ones), kept(zeros)
    step([0])
    assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(sat_out, kept(ones)))
    assert not any(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(took_part, kept(zeros)))


@pytest.mark.gpu
def test_gradients_that_a_step_drops_are_not_reused_before_it_ran():
    """A step on another stream than the gradients' own"""
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    p = torch.zeros(1 << 20, device="cuda")
    opt = AdamW([p])
    p.grad = torch.ones(1 << 20, device="cuda")
    at = p.grad.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # 0.1 s
        opt.step()
    assert p.grad is None and torch.empty(1 << 20, device="cuda").data_ptr() != at
    torch.cuda.synchronize()
    assert (p < 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("with_backward", [False, True])
def test_captured_steps_read_gradients_where_they_were(with_backward):
    """A replay finds the gradients at their places: those that it was given, or those of its own backward pass"""
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    p, q = torch.zeros(3000, device="cuda", requires_grad=True), torch.zeros(3000, device="cuda")
    opt, other = AdamW([p]), AdamW([q])
    d = torch.randn(3000, device="cuda")
    if not with_backward:
        p.grad = torch.zeros_like(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if with_backward:
            (p * d).sum().backward()
        opt.step()
    assert p.grad is not None
    for _ in range(3):
        d.normal_()
        junk = [torch.full((3000,), 7.0, device="cuda") for _ in range(4)]   # in what memory there is
        if not with_backward:
            p.grad.copy_(d)
        graph.replay()
        q.grad, other.step_count = d.clone(), 0   # a replay repeats the step that was captured
        other.step()
        assert torch.equal(p.detach(), q) and (p.grad == 0).all() and all((t == 7).all() for t in junk)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_bias_corrections_count_a_parameters_own_steps(bits):
    """A first gradient that comes late moves its parameter as the first step does, and a step that a parameter sits out counts for the others alone."""
    from aws_ofi_nccl_b200.parallel.engine import AdamW, OptimConfig

    oc = OptimConfig(lr=1e-2, weight_decay=0.0)
    g = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(500, device="cuda", generator=g) for _ in range(4)]
    a, b, alone = (torch.zeros(500, device="cuda") for _ in range(3))
    opt, other = AdamW([a, b], oc, bits=bits), AdamW([alone], oc, bits=bits)
    for step, d in enumerate(grads):
        a.grad = d.clone()
        b.grad = None if step in (0, 2) else d.clone()
        opt.step()
        if step in (1, 3):
            alone.grad = d.clone()
            other.step()
            assert torch.equal(b, alone)
        if step == 1:   # m / (1 - b1) over the root of v / (1 - b2): lr in the direction of the gradient, whatever its size
            assert ((b + 1e-2 * grads[1].sign()).abs() <= 1e-2 * (1e-8 / grads[1].abs() + 2.0 ** -20)).all()
    assert opt.step_count == 4 and other.step_count == 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_steps_of_their_own_equal_calls_of_their_own(bits):
    from aws_ofi_nccl_b200.ops import llm

    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, zero_grad=False)
    g = torch.Generator(device="cuda").manual_seed(5)
    sizes, steps = [700, 3, 0, 256, 1000, 5, 90], (4, 1, 1, 4, 2 ** 33, 1, 7)
    params = [torch.randn(n, device="cuda", generator=g).to(BF) for n in sizes]
    grads = [torch.randn(n, device="cuda", generator=g).to(BF) for n in sizes]
    grads[5] = None
    one, state = [p.clone() for p in params], llm.adamw_states(params, bits=bits, master=True)
    for wrong in ([1] * 6, [], [1] * 6 + [0], (1, 2)):
        with pytest.raises(AssertionError):
            llm.adamw_step_many(params, grads, **state, **hyper, step=wrong)
    for wrong in (1.5, None, [1.5] * 7, "1", 2 ** 70):
        with pytest.raises(TypeError):
            llm.adamw_step_many(params, grads, **state, **hyper, step=wrong)
    with pytest.raises(AssertionError):   # before any of them is written
        llm.adamw_step_many(params, [*grads[:6], grads[6].half()], **state, **hyper, step=steps)
    assert all(torch.equal(a, b) for a, b in zip(params, one))
    llm.adamw_step_many(params, grads, **state, **hyper, step=steps)
    for i, p in enumerate(one):
        s = llm.adamw_states([p], bits=bits, master=True)
        llm.adamw_step_many([p], [grads[i]], **s, **hyper, step=steps[i])
        assert torch.equal(p, params[i])
        for name, tensors in s.items():
            assert tensors is None or torch.equal(tensors[0].view(torch.uint8), state[name][i].view(torch.uint8))


def test_checkpoints_hold_what_was_sat_out():
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    params = [torch.zeros(300), torch.zeros(7)]
    a = AdamW(params, bits=8)
    a.step_count, a.sat_out = 5, [0, 3]
    b = AdamW(params, bits=8)
    b.load_state_dict(a.state_dict())
    assert b.step_count == 5 and b.sat_out == [0, 3] and b.sat_out is not a.sat_out
    saved = a.state_dict()
    del saved["sat_out"]   # of a version that had one count for all
    b.load_state_dict(saved)
    assert b.step_count == 5 and b.sat_out == [0, 0]
    with pytest.raises(ValueError):
        b.load_state_dict({**a.state_dict(), "sat_out": [0]})


def test_a_refused_step_counts_for_nothing(built):
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    p = torch.zeros(64)
    p.grad = torch.ones(64)
    opt = AdamW([p])
    for _ in range(2):
        with pytest.raises(AssertionError):   # not on a GPU
            opt.step()
    assert opt.step_count == 0 and (p.grad == 1).all()


def test_the_configuration_says_the_moments_bits():
    from aws_ofi_nccl_b200.parallel.engine import AdamW, OptimConfig

    params = [torch.zeros(300, dtype=BF)]
    for opt, bits in ((AdamW(params), 32), (AdamW(params, OptimConfig(state_bits=8)), 8), (AdamW(params, bits=8), 8),
                      (AdamW(params, OptimConfig(), bits=8), 8), (AdamW(params, OptimConfig(state_bits=8), bits=8), 8)):
        assert opt.bits == bits and opt.state["m"][0].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32)
        assert opt.state_dict()["bits"] == bits
    with pytest.raises(ValueError):
        AdamW(params, OptimConfig(state_bits=8), bits=32)
    for optim, bits in ((None, 16), (OptimConfig(state_bits=16), None)):
        with pytest.raises(ValueError):
            AdamW(params, optim, bits=bits)


@pytest.mark.gpu
def test_gradients_over_what_is_written_are_refused():
    """A gradient is read while other CTAs write: it may be shared, but not with a parameter, a moment, a scale or a master copy."""
    from aws_ofi_nccl_b200.ops import llm

    hyper = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1, zero_grad=False)
    for bits in (8, 32):
        buf = torch.ones(4000, device="cuda")
        p = [buf[:1000], buf[2000:3000]]
        state = llm.adamw_states(p, bits=bits)
        inside = [torch.ones(1000, device="cuda"), buf[1500:2500]]
        before = buf.clone()
        for grads in (inside, inside[::-1], [buf[1000:2000], buf[2001:3001]], [buf[1:1001], buf[3000:]], [buf[:1000], buf[3000:]]):
            with pytest.raises(AssertionError):
                llm.adamw_step_many(p, grads, **state, **hyper)
        if bits == 32:
            with pytest.raises(AssertionError):
                llm.adamw_step_many(p, [state["v"][1], buf[3000:]], **state, **hyper)
        assert torch.equal(buf, before)
        llm.adamw_step_many(p, [buf[1000:2000], buf[3000:]], **state, **hyper)   # beside them
        llm.adamw_step_many(p, [buf[1000:2000]] * 2, **state, **{**hyper, "step": 2})   # one for both
        assert (buf[:1000] != 1).all() and torch.equal(buf[1000:2000], before[1000:2000]) and torch.equal(buf[:1000], buf[2000:3000])


# ------------------------------------------------------------------ the layer's backward pass
@pytest.mark.gpu
def test_experts_rows_are_cut_and_joined_once():
    """The rows' gradient is one concatenation, not a matrix of all rows for each expert"""
    from aws_ofi_nccl_b200.models.moe import MoELayer

    layer = MoELayer(None, 0, 256, 128, 16, 2, seed=1)
    x = torch.randn(200, 256, device="cuda").to(BF).requires_grad_(True)
    out = layer(x)
    seen, todo = {}, [out.grad_fn]
    while todo:
        node = todo.pop()
        if node is not None and node not in seen:
            seen[node] = node.name()
            todo += [n for n, _ in node.next_functions]
    assert not [n for n in seen.values() if "Slice" in n]
    assert sum("Split" in n for n in seen.values()) == 1


# ------------------------------------------------------------------ the norm's rows that are not finite
@pytest.mark.gpu
@pytest.mark.parametrize("H", [256, 1024, 7168])
def test_scales_of_rows_that_are_not_finite(H):
    """What the composition of rmsnorm's formula and the scales' makes of them: a NaN is in every scale of its row, an infinity in its own (its row's, or its
    128 columns'), and the rest of that row is zero times it. A finite row whose squares add up beyond 32 bits is zero, as rmsnorm's is."""
    from aws_ofi_nccl_b200.ops import llm

    x = torch.randn(4, H, device="cuda").to(BF)
    x[0, 3], x[1, 130], x[2, 130] = float("nan"), float("inf"), -float("inf")
    x[3] = 2.0 ** 90
    w = torch.ones(H, device="cuda", dtype=BF)
    least = torch.full((), 1e-12, device="cuda") * (1.0 / 448.0)
    q, scale, _ = llm.rmsnorm_fp8(x, w)
    assert scale[:3].isnan().all() and scale[3] == least and (q[3].float() == 0).all()
    q, scale, _ = llm.rmsnorm_fp8(x, w, group=128)
    assert scale[0].isnan().all()
    for row in (1, 2):
        assert scale[row, 1].isnan()
        others = torch.arange(H // 128, device="cuda") != 1
        assert (scale[row][others] == least).all() and (q[row].view(-1, 128)[others].float() == 0).all()
    assert (scale[3] == least).all() and (q[3].float() == 0).all()
    n, _ = llm.rmsnorm(x, w)
    assert n[0].isnan().all() and (n[3] == 0).all()
    for row in (1, 2):
        assert n[row, 130].isnan() and (n[row, :128] == 0).all() and (n[row, 131:] == 0).all()


# ------------------------------------------------------------------ moments in 8 bits beyond the first step
@pytest.mark.gpu
@pytest.mark.parametrize("sizes,packed", [((257,), False), ((100003, 7, 4096, 1, 65536), False), ((100003, 7, 4096, 1, 65536), True)])
@pytest.mark.parametrize("dtype,master", [(BF, False), (BF, True), (torch.float32, False)])
def test_codes_of_moments_that_are_not_zero_before(sizes, packed, dtype, master):
    """Element by element: codes and scales of both moments in the second and third step, with the rounding that m's terms leave where they cancel"""
    from aws_ofi_nccl_b200.ops import llm

    F = 2.0 ** -24
    b1, b2 = 0.9, 0.95
    g = torch.Generator(device="cuda").manual_seed(sum(sizes))
    lay = (lambda t: list(t.split(list(sizes)))) if packed else (lambda t: [s.clone() for s in t.split(list(sizes))])
    params = lay((torch.randn(sum(sizes), device="cuda", generator=g) * 0.05).to(dtype))
    state = llm.adamw_states(params, bits=8, master=master)
    checked = 0
    for step in (1, 2, 3):
        grads = lay((torch.randn(sum(sizes), device="cuda", generator=g) * 10.0 ** -step).to(dtype))
        old = [{n: (state[n][i].double(), state[n + "_scale"][i].double()) for n in "mv"} for i in range(len(sizes))]
        llm.adamw_step_many(params, grads, **state, lr=1e-3, beta1=b1, beta2=b2, eps=1e-8, weight_decay=0.1, step=step, zero_grad=False)
        for i, n in enumerate(sizes):
            block = torch.arange(n, device="cuda") // 256
            blocks = -(-n // 256)
            d = grads[i].double()
            m, v = (old[i][x][0] * old[i][x][1][block] for x in "mv")
            v = v * v
            # roundings: m's product and decoding, its scaled gradient, their sum, each of its own size; of the root half of those of v
            m_off = F * (4 * b1 * m.abs() + 4 * (1 - b1) * d.abs())
            m = b1 * m + (1 - b1) * d
            root = (b2 * v + (1 - b2) * d * d).sqrt()
            word = (torch.arange(n, device="cuda") * 0xC13FA9A9 + step * 0x91E10DA5) & 0xFFFFFFFF
            for name, z, off, dither in (("m", m, m_off, word), ("v", root, 6 * F * root, word ^ 0xFFFFFFFF)):
                most = torch.zeros(blocks, device="cuda", dtype=torch.float64).scatter_reduce_(0, block, z.abs(), "amax")
                top_off = torch.zeros(blocks, device="cuda", dtype=torch.float64).scatter_reduce_(0, block, off, "amax")
                top = most.clamp_min(1e-30) / 448
                assert ((state[name + "_scale"][i].double() - top).abs() <= top_off / 448 + 4 * F * top).all()
                share = z.abs() / top[block]
                gap = torch.exp2(torch.floor(torch.log2(share.clamp_min(2.0 ** -6))) - 3)
                place = share / gap + (dither >> 12).double() / 2 ** 20
                # what the share may be off by: of its own value, of the scale, three roundings, and half of 2^-29 of what is denormal there
                place_off = (off / top[block] + share * (top_off / most.clamp_min(1e-30))[block] + 6 * F * share) / gap + 2.0 ** -20
                near = (place - place.round()).abs() <= place_off
                near |= (share / gap - 8).abs() <= place_off   # the gap itself halves below
                want = (torch.floor(place) * gap).clamp(max=448)
                if name == "v":
                    want = torch.where(z != 0, want.clamp_min(2.0 ** -9), want)
                got = state[name][i].double()
                assert torch.equal(got.abs()[~near], want[~near])
                assert ((got.abs() - want).abs() <= gap * (1 + 1e-9))[near].all()
                sure = (z.abs() > off) & (got != 0)
                assert torch.equal(torch.signbit(got)[sure], torch.signbit(z)[sure])
                checked += int((~near).sum())
    assert checked >= 0.98 * 6 * sum(sizes)


def _odd_config():
    """Norms of 384 weights: a block of 256 elements of the flat buffer would hold two parameters"""
    from aws_ofi_nccl_b200.models.llama import LlamaConfig

    return LlamaConfig(vocab_size=512, hidden=384, n_layers=2, n_heads=6, n_kv_heads=2, ffn=640, max_seq=64)


def test_blocks_of_the_trainers_moments_are_one_parameters():
    from aws_ofi_nccl_b200.parallel.engine import OptimConfig, Trainer

    cfg = _odd_config()
    tr = Trainer(cfg, OptimConfig(state_bits=8), device="cpu")
    assert tr.m_scale.numel() == tr.v_scale.numel() == sum(-(-math.prod(s) // 256) for _, s in cfg.param_shapes())
    sd = tr.state_dict()
    Trainer(cfg, OptimConfig(state_bits=8), device="cpu", seed=3).load_state_dict(sd)
    # a checkpoint whose blocks went over the parameters' borders
    flat = {k: v for k, v in sd.items() if k != "scale_blocks"}
    with pytest.raises(ValueError):
        tr.load_state_dict(flat)
    tiny = type(cfg).tiny()   # there the borders of both are the same
    tr = Trainer(tiny, OptimConfig(state_bits=8), device="cpu")
    assert tr.m_scale.numel() == -(-tr.m.numel() // 256)
    tr.load_state_dict({k: v for k, v in tr.state_dict().items() if k != "scale_blocks"})


class _Shard:
    """What the trainer asks of a reducer in "zero" mode, of one rank among others, without the others"""
    mode, grad_scale = "zero", 0.5

    def __init__(self, lo, hi):
        self.range = (lo, hi)

    def allocate_grad_buffer(self, n):
        return torch.zeros(n, device="cuda", dtype=BF)

    def shard_range(self, n):
        return self.range

    def attach(self, model):
        pass

    def begin_step(self):
        pass

    def finish_step(self):
        pass

    def gather_params(self, flat):
        pass


@pytest.mark.gpu
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("shard", [None, (100_096, 400_000)])
def test_trainer_steps_each_parameter_by_itself(master, shard):
    """Against AdamW's step over the parameters one by one, with the numbers that the configuration names; in a shard, over what it has of each"""
    from aws_ofi_nccl_b200.ops import llm
    from aws_ofi_nccl_b200.parallel.engine import OptimConfig, Trainer

    cfg = _odd_config()
    oc = OptimConfig(lr=2e-3, beta1=0.8, beta2=0.9, eps=1e-6, weight_decay=0.3, state_bits=8, master_weights=master)
    tr = Trainer(cfg, oc, device="cuda", dp=_Shard(*shard) if shard else None)
    lo, hi = tr.shard
    pieces = []
    for off, shape in tr.model.offsets.values():
        a, b = max(off, lo), min(off + math.prod(shape), hi)
        if a < b:
            pieces.append((a, b))
    assert len(pieces) >= 3 and any((a - lo) % 256 for a, _ in pieces)
    params = [tr.model.flat_params[a:b].clone() for a, b in pieces]
    states = [llm.adamw_states([p], bits=8, master=master) for p in params]
    outside = torch.cat((tr.model.flat_params[:lo], tr.model.flat_params[hi:])).clone()
    grads = []
    step_many = llm.adamw_step_many

    def watched(*args, **kw):
        grads.append(tr.model.flat_grads.clone())
        step_many(*args, **kw)

    ids, lbl = (torch.randint(0, cfg.vocab_size, (2, 64), device="cuda") for _ in range(2))
    llm.adamw_step_many = watched
    try:
        for step in (1, 2):
            tr.step_device(ids, lbl)
            for (a, b), p, s in zip(pieces, params, states):
                step_many([p], [grads[-1][a:b].clone()], **s, lr=2e-3, beta1=0.8, beta2=0.9, eps=1e-6, weight_decay=0.3, step=step,
                          grad_scale=0.5 if shard else 1.0)
    finally:
        llm.adamw_step_many = step_many
    assert len(grads) == 2 and (tr.model.flat_grads == 0).all()
    at = 0
    for (a, b), p, s in zip(pieces, params, states):
        n = s["m_scale"][0].numel()
        assert torch.equal(tr.model.flat_params[a:b], p)
        for flat, one in ((tr.m, s["m"][0]), (tr.v, s["v"][0])):
            assert torch.equal(flat[a - lo:b - lo].view(torch.uint8), one.view(torch.uint8))
        assert torch.equal(tr.m_scale[at:at + n], s["m_scale"][0]) and torch.equal(tr.v_scale[at:at + n], s["v_scale"][0])
        assert not master or torch.equal(tr.master[a - lo:b - lo], s["master"][0])
        at += n
    assert at == tr.m_scale.numel()
    assert torch.equal(torch.cat((tr.model.flat_params[:lo], tr.model.flat_params[hi:])), outside)
