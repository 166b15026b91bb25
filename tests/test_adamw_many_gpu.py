"""AdamW over many tensors against 64 bits: moments and parameters element by element, 8-bit codes against the dither's rule."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F, BF = 2.0 ** -24, 2.0 ** -8
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8)
BLOCK = 256


def _tensors(sizes, dtype, packed, std, g, offset=0):
    """Tensors of their own, or one behind the other (on no boundary but an element's)"""
    if not packed:
        return [(torch.randn(n, device="cuda", generator=g) * std).to(dtype) for n in sizes]
    flat = (torch.randn(sum(sizes) + offset, device="cuda", generator=g) * std).to(dtype)
    return list(flat[offset:].split(list(sizes)))


def _blocks(n):
    return torch.arange(n, device="cuda") // BLOCK


def _held(values, word):
    """|values| in 64 bits, the dither -> (scale, place): the code's value is the e4m3 number at or below place, place being share + dither * step"""
    n = values.numel()
    top = torch.zeros(-(-n // BLOCK), device="cuda", dtype=torch.float64).scatter_reduce_(0, _blocks(n), values.abs(), "amax").clamp_min(1e-30) / 448
    share = values.abs() / top[_blocks(n)]
    step = torch.exp2(torch.floor(torch.log2(share.clamp_min(2.0 ** -6))) - 3)
    return top, share, step, (word >> 12).double() / 2 ** 20


def _check_held(code, scale, values, word, floor):
    top, share, step, up = _held(values, word)
    assert ((scale.double() - top).abs() <= 8 * F * top).all()
    place = share / step + up
    want = (torch.floor(place) * step).clamp(max=448)
    if floor:
        want = torch.where(values != 0, want.clamp_min(2.0 ** -9), want)
    got = code.double().abs()
    # a share that is off by a few steps of 32 bits changes the code where the place is that near to a whole number, and there to the neighbour
    near = (place - place.round()).abs() <= 16 * 64 * F
    assert torch.equal(got[~near], want[~near])
    assert ((got - want).abs() <= step * (1 + 1e-9))[near].all()
    assert near.double().mean() <= 0.01 + 8 / max(1, near.numel())


def _step(params, grads, state, decay, step, grad_scale=1.0, zero_grad=False):
    """The reference: what each tensor is after the step, in 64 bits, from what it is now"""
    out = []
    for i, (p, g) in enumerate(zip(params, grads)):
        master = state["master"][i] if state["master"] else None
        x = (master if master is not None else p).detach().double()
        if state["m_scale"]:
            m = state["m"][i].double() * state["m_scale"][i].double()[_blocks(p.numel())].view(p.shape)
            v = (state["v"][i].double() * state["v_scale"][i].double()[_blocks(p.numel())].view(p.shape)).square()
        else:
            m, v = state["m"][i].double(), state["v"][i].double()
        d = g.double() * grad_scale
        mag = HYPER["beta1"] * m.abs() + (1 - HYPER["beta1"]) * d.abs()
        m = HYPER["beta1"] * m + (1 - HYPER["beta1"]) * d
        v = HYPER["beta2"] * v + (1 - HYPER["beta2"]) * d * d
        denom = (v / (1 - HYPER["beta2"] ** step)).sqrt() + HYPER["eps"]
        lr1 = HYPER["lr"] / (1 - HYPER["beta1"] ** step)
        want = x * (1 - HYPER["lr"] * decay[i]) - lr1 * m / denom
        # the update's roundings: three in m, of its terms, and twelve in the quotient and its operands
        out.append((want, 3 * F * x.abs() + 16 * F * lr1 * mag / denom + 1e-37, m, mag, v))
    return out


def _run(sizes, bits, dtype, grad_dtype=None, master=False, packed=False, steps=2, grad_scale=1.0, zero_grad=False, offset=0):
    from aws_ofi_nccl_b200.ops import llm

    g = torch.Generator(device="cuda").manual_seed(sum(sizes) + bits)
    params = _tensors(sizes, dtype, packed, 0.05, g, offset)
    state = llm.adamw_states(params, bits=bits, master=master)
    if packed and bits == 8:   # codes on no boundary either
        for name in ("m", "v"):
            state[name] = list(torch.zeros(sum(sizes) + offset, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)[offset:].split(list(sizes)))
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    for step in range(1, steps + 1):
        grads = _tensors(sizes, grad_dtype or dtype, packed, 10.0 ** -step, g, offset)
        for t in grads:
            t[::7] = 0
        want = _step(params, grads, state, decay, step, grad_scale)
        llm.adamw_step_many(params, grads, **state, **HYPER, weight_decay=decay, step=step, grad_scale=grad_scale, zero_grad=zero_grad)
        for i, (x, most, m, mag, v) in enumerate(want):
            p = params[i].double()
            if master and dtype == torch.bfloat16:
                assert ((state["master"][i].double() - x).abs() <= most).all()
                assert torch.equal(params[i], state["master"][i].bfloat16())
            else:
                assert ((p - x).abs() <= most + (BF * (x.abs() + most) if dtype == torch.bfloat16 else 0)).all()
            if bits == 32:
                assert ((state["m"][i].double() - m).abs() <= 3 * F * mag + 1e-44).all()
                assert ((state["v"][i].double() - v).abs() <= 5 * F * v + 1e-44).all()
            else:
                word = (torch.arange(x.numel(), device="cuda") * 0xC13FA9A9 + step * 0x91E10DA5) & 0xFFFFFFFF
                # codes follow the moments of 32 bits: m's own cancellation is part of its rounding
                sure = mag <= 8 * m.abs()
                got = state["m"][i].double()
                assert (torch.signbit(got) == torch.signbit(m))[(got != 0) & sure].all()
                if sure.all():
                    _check_held(state["m"][i].reshape(-1), state["m_scale"][i], m.reshape(-1), word, False)
                _check_held(state["v"][i].reshape(-1), state["v_scale"][i], v.sqrt().reshape(-1), word ^ 0xFFFFFFFF, True)
            assert not zero_grad or (grads[i] == 0).all()


SIZES = [(1,), (255,), (256,), (257,), (8, 2048, 2049, 3), (100003, 7, 4096, 1, 65536)]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,master", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("packed", [False, True])
def test_sizes_types_and_alignments(sizes, bits, dtype, master, packed):
    _run(sizes, bits, dtype, master=master, packed=packed, offset=1 if packed else 0)


@pytest.mark.parametrize("offset", range(8))
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,master", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_every_offset_from_a_boundary(offset, bits, dtype, master):
    """Parameters, gradients and state off a boundary by as many elements, with neighbours on either side that are not touched"""
    from aws_ofi_nccl_b200.ops import llm

    sizes, room = (2000, 256, 700, 5), 16
    total = sum(sizes) + offset + room
    g = torch.Generator(device="cuda").manual_seed(offset)
    where = [offset + sum(sizes[:i]) for i in range(len(sizes))]
    cut = lambda flat: [flat[a:a + n] for a, n in zip(where, sizes)]   # noqa: E731

    def flat(make):
        t = make(total)
        return t, t.clone()

    p, p0 = flat(lambda n: (torch.randn(n, device="cuda", generator=g) * 0.05).to(dtype))
    d, d0 = flat(lambda n: torch.randn(n, device="cuda", generator=g).to(dtype))
    names = ["m", "v"] + (["master"] if master else [])
    make = {n: (lambda k: torch.zeros(k, device="cuda")) if bits == 32 or n == "master" else
            (lambda k: torch.zeros(k, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)) for n in names}
    buffers = {n: make[n](total) for n in names}
    if master:
        buffers["master"].copy_(p.float())
    scales = {f"{n}_scale": [torch.zeros(-(-k // 256), device="cuda") for k in sizes] if bits == 8 else None for n in "mv"}
    state = {"master": None, **{n: cut(b) for n, b in buffers.items()}, **scales}
    other = llm.adamw_states([t.clone() for t in cut(p)], bits=bits, master=master)
    apart = [t.clone() for t in cut(p)]
    for step in (1, 2, 3):
        llm.adamw_step_many(cut(p), cut(d), **state, **HYPER, weight_decay=0.1, step=step, zero_grad=step == 3)
        llm.adamw_step_many(apart, [t.clone() for t in cut(d0)], **other, **HYPER, weight_decay=0.1, step=step)
    as_bytes = lambda t: t.contiguous().view(torch.uint8)   # noqa: E731
    for a, b in zip(cut(p), apart):
        assert torch.equal(a, b)
    for n in names:
        for a, b in zip(state[n], other[n]):
            assert torch.equal(as_bytes(a), as_bytes(b))
    assert all((t == 0).all() for t in cut(d))
    end = where[-1] + sizes[-1]
    for now, then in ((p, p0), (d, d0)):
        assert torch.equal(as_bytes(now[:offset]), as_bytes(then[:offset])) and torch.equal(as_bytes(now[end:]), as_bytes(then[end:]))
    for n in ("m", "v"):
        assert (as_bytes(buffers[n][:offset]) == 0).all() and (as_bytes(buffers[n][end:]) == 0).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,grad_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_gradients_of_another_type(bits, dtype, grad_dtype):
    _run((3000, 513, 8), bits, dtype, grad_dtype=grad_dtype)
    _run((3000, 513, 8), bits, dtype, grad_dtype=grad_dtype, master=True, packed=True)


@pytest.mark.parametrize("bits", [8, 32])
def test_scaled_and_zeroed_gradients(bits):
    _run((5000, 300), bits, torch.bfloat16, grad_scale=0.125, zero_grad=True)
    _run((5000, 300), bits, torch.float32, grad_scale=3.7, zero_grad=True, packed=True)


# more tensors than a launch takes; and as many as each of its tables
@pytest.mark.parametrize("count", [16, 17, 128, 129, 400, 401, 1000])
@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors(count, bits):
    _run([1 + (i * 37) % 700 for i in range(count)], bits, torch.bfloat16, steps=1)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_large_tensor_among_small_ones(bits):
    """CTAs of several passes"""
    _run((40_000_003, 100, 5_000_000), bits, torch.bfloat16, steps=1)


def test_mixed_types_in_one_call_equal_calls_of_one_tensor():
    from aws_ofi_nccl_b200.ops import llm

    for bits in (8, 32):
        g = torch.Generator(device="cuda").manual_seed(8)
        params = [torch.randn(n, device="cuda", generator=g).to(t) for n, t in ((700, torch.float32), (900, torch.bfloat16), (64, torch.float32))]
        grads = [torch.randn(p.shape, device="cuda", generator=g).to(t) for p, t in zip(params, (torch.bfloat16, torch.bfloat16, torch.float32))]
        state = llm.adamw_states(params, bits=bits, master=True)
        assert [c is None for c in state["master"]] == [True, False, True]
        one = [p.clone() for p in params]
        states = [llm.adamw_states([p], bits=bits, master=True) for p in one]
        for step in (1, 2, 3):
            llm.adamw_step_many(params, grads, **state, **HYPER, weight_decay=0.1, step=step, zero_grad=False)
            for p, d, s in zip(one, grads, states):
                llm.adamw_step_many([p], [d], **s, **HYPER, weight_decay=0.1, step=step, zero_grad=False)
        assert all(torch.equal(a, b) for a, b in zip(params, one))


def test_tensors_without_a_gradient_and_without_elements_are_left_alone():
    from aws_ofi_nccl_b200.ops import llm

    params = [torch.ones(300, device="cuda"), torch.ones(300, device="cuda"), torch.empty(0, device="cuda")]
    state = llm.adamw_states(params, bits=8)
    llm.adamw_step_many(params, [torch.ones(300, device="cuda"), None, torch.empty(0, device="cuda")], **state, **HYPER, weight_decay=0.1, step=1)
    assert (params[0] != 1).all() and (params[1] == 1).all()
    assert (state["m_scale"][1] == 0).all() and (state["m"][1].float() == 0).all()
    llm.adamw_step_many([], [], [], [], **HYPER, weight_decay=0.1, step=1)
    llm.adamw_step_many(params, [None] * 3, **state, **HYPER, weight_decay=0.1, step=2)
    assert (params[1] == 1).all()


def test_matches_the_flat_buffers_step():
    """adamw_step's result to within its own roundings, which are not those of this one"""
    from aws_ofi_nccl_b200.ops import llm

    g = torch.Generator(device="cuda").manual_seed(1)
    p = (torch.randn(4096, device="cuda", generator=g) * 0.02).bfloat16()
    d = (torch.randn(4096, device="cuda", generator=g) * 1e-3).bfloat16()
    flat, m, v, master = p.clone(), torch.zeros(4096, device="cuda"), torch.zeros(4096, device="cuda"), p.float()
    state = llm.adamw_states([p], bits=32, master=True)
    for step in (1, 2, 3):
        llm.adamw_step(flat, d.clone(), m, v, master, **HYPER, weight_decay=0.1, step=step)
        llm.adamw_step_many([p], [d], **state, **HYPER, weight_decay=0.1, step=step, zero_grad=False)
    # three steps of lr each, whose bias corrections are powers in 32 bits there: 2^-24 of a power over 1 - b2^t >= 0.05
    most = 3 * HYPER["lr"] * (40 * F / 0.05 + 40 * F) + 9 * F * master.abs()
    assert ((state["master"][0] - master).abs() <= most).all()


def test_moments_in_8_bits_move_in_the_mean():
    """Gradients that vanish: roots decay by 2.5 % a step, less than half of a code's step, and m by 10 %"""
    from aws_ofi_nccl_b200.ops import llm

    n = 256 * 64
    p = torch.zeros(n, device="cuda")
    state = llm.adamw_states([p], bits=8)
    llm.adamw_step_many([p], [0.5 + torch.rand(n, device="cuda")], **state, **HYPER, weight_decay=0.0, step=1)
    blocks = _blocks(n)
    value = lambda name: (state[name][0].double() * state[name + "_scale"][0].double()[blocks])   # noqa: E731
    m0, v0 = value("m").mean(), value("v").mean()
    zero = torch.zeros(n, device="cuda")
    for step in range(2, 22):
        llm.adamw_step_many([p], [zero], **state, **HYPER, weight_decay=0.0, step=step)
    # unbiased: 20 roundings of up to a step (an eighth) each over 16384 elements, as independent ones: 0.0625 * sqrt(20 / 16384) = 0.002, and five times that
    assert abs(value("v").mean() / v0 / HYPER["beta2"] ** 10 - 1) <= 0.012
    assert abs(value("m").mean() / m0 / HYPER["beta1"] ** 20 - 1) <= 0.012


@pytest.mark.parametrize("bits", [8, 32])
def test_what_is_not_finite_stays_in_its_element(bits):
    from aws_ofi_nccl_b200.ops import llm

    params = [torch.ones(1000, device="cuda"), torch.ones(1000, device="cuda")]
    clean = torch.randn(1000, device="cuda")
    bad = clean.clone()
    bad[300], bad[301], bad[302] = float("nan"), float("inf"), -float("inf")
    state = llm.adamw_states(params, bits=bits)
    for step in (1, 2):
        llm.adamw_step_many(params, [clean, bad], **state, **HYPER, weight_decay=0.1, step=step, zero_grad=False)
    hit = torch.zeros(1000, device="cuda", dtype=torch.bool)
    hit[300:303] = True
    assert params[1][hit].isnan().all() and state["m"][1][hit].float().isnan().any() and params[1][~hit].isfinite().all()
    if bits == 32:
        assert torch.equal(params[0][~hit], params[1][~hit])
    else:   # a block's scale is that of its finite elements
        assert state["m"][1].float()[hit].isnan().all() and state["v"][1].float()[hit].isnan().all()
        assert state["m_scale"][1].isfinite().all() and state["v_scale"][1].isfinite().all()


def test_extreme_gradients_in_8_bits():
    """Blocks whose elements span more than e4m3 holds, tiny and huge ones: the update is that of moments in 32 bits, a root is never held as zero"""
    from aws_ofi_nccl_b200.ops import llm

    for low, high in ((-12, 0), (-18, -6), (0, 12)):
        g = torch.logspace(low, high, 2048, device="cuda")[torch.randperm(2048, device="cuda")]
        p = torch.zeros(2048, device="cuda")
        state = llm.adamw_states([p], bits=8)
        want = _step([p], [g], state, [0.0], 1)[0]
        llm.adamw_step_many([p], [g], **state, **HYPER, weight_decay=0.0, step=1, zero_grad=False)
        assert ((p.double() - want[0]).abs() <= want[1]).all()
        assert torch.equal(state["v"][0].float() > 0, g.square() * (1 - HYPER["beta2"]) > 0)   # squares of 1e-18 are denormal, not zero
        before = p.clone()
        llm.adamw_step_many([p], [torch.zeros_like(g)], **state, **HYPER, weight_decay=0.0, step=2)
        assert p.isfinite().all() and ((p - before).abs() <= 4 * HYPER["lr"]).all()


def test_captured_step_repeats_itself():
    from aws_ofi_nccl_b200.ops import llm

    p, d = torch.zeros(5000, device="cuda"), torch.randn(5000, device="cuda")
    state = llm.adamw_states([p], bits=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        llm.adamw_step_many([p], [d], **state, **HYPER, weight_decay=0.1, step=5, zero_grad=False)
    q, other = p.clone(), llm.adamw_states([p], bits=8)
    for _ in range(3):
        graph.replay()
        llm.adamw_step_many([q], [d], **other, **HYPER, weight_decay=0.1, step=5, zero_grad=False)
        assert torch.equal(p, q) and torch.equal(state["m"][0].view(torch.uint8), other["m"][0].view(torch.uint8))


def test_a_graph_that_kept_the_old_values_is_told():
    from aws_ofi_nccl_b200.ops import llm

    p = torch.ones(64, device="cuda", requires_grad=True)
    y = (p * p).sum()
    llm.adamw_step_many([p], [torch.ones(64, device="cuda")], **llm.adamw_states([p]), **HYPER, weight_decay=0.0, step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
