"""A mixture-of-experts block on one GPU, operator by operator: the norm in front of it with its output in 8 bits, tokens sorted by
expert and back with their gradients, and the optimizer's step over the block's many tensors.

Every case is a plain dict with a "kind"; sizes are those of the Llama-3-8B and tiny configurations of ``models/llama.py``, of
``utils/bench_moe.py`` and of the tests, plus generic odd ones. With ``own`` false ``run`` computes the operators from elementary
torch operations in 32 bits, with it true through the framework.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
BLOCK = 256           # elements of a tensor that share a scale of the optimizer's 8-bit state
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1


def listed() -> list[dict]:
    return [
        # one decoding step of eight sequences: residual, norm and row scales for the fp8 product behind it
        dict(name="norm8_decode", kind="norm8", t=8, h=4096, residual=True, group=0),
        # a prompt of 4096 tokens through the same layer
        dict(name="norm8_prompt", kind="norm8", t=4096, h=4096, residual=True, group=0),
        # a ragged batch with a scale for every 128 columns, as the expert exchange moves its rows
        dict(name="norm8_groups", kind="norm8", t=5003, h=7168, residual=False, group=128),
        # decoding: sixteen tokens to their experts and back
        dict(name="moe_decode", kind="moe", t=16, h=4096, e=64, k=8, dtype="bf16", train=False, drop=False),
        # training at the sizes of utils/bench_moe.py: both directions, and the weights' gradient
        dict(name="moe_train", kind="moe", t=4096, h=7168, e=256, k=8, dtype="bf16", train=True, drop=False),
        # odd sizes in 32 bits, with slots that go to no expert
        dict(name="moe_train_ragged", kind="moe", t=3001, h=1283, e=60, k=3, dtype="fp32", train=True, drop=True),
        # 8-bit rows and their scales for experts that multiply in fp8
        dict(name="moe_fp8", kind="moe8", t=8192, h=4096, e=128, k=4, group=128, drop=False),
        # the tiny model's tensors, states in 32 bits: launches and the host decide
        dict(name="adamw_tiny", kind="adamw", tensors=15, n=1705216, bits=32, dtype="bf16", master=False, packed=False),
        # as many parameters as a decoder layer of the 8B configuration, states in 8 bits
        dict(name="adamw_layer8", kind="adamw", tensors=6, n=218112000, bits=8, dtype="bf16", master=False, packed=False),
        # the experts of a layer as tensors of their own, 8-bit states beside a 32-bit master copy
        dict(name="adamw_experts8", kind="adamw", tensors=129, n=100663296, bits=8, dtype="bf16", master=True, packed=False),
        # the same with states in 32 bits
        dict(name="adamw_experts32", kind="adamw", tensors=129, n=100663296, bits=32, dtype="bf16", master=True, packed=False),
        # fp32 parameters of odd sizes, one behind the other without padding
        dict(name="adamw_packed8", kind="adamw", tensors=37, n=9000007, bits=8, dtype="fp32", master=False, packed=True),
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max((lo + step - 1) // step * step, min(hi // step * step, int(round(v / step)) * step))


def draw(rng) -> dict:
    kind = rng.choice(["norm8", "moe", "moe", "moe8", "adamw", "adamw"])
    if kind == "norm8":
        group = rng.choice([0, 0, 128])
        h = _log(rng, 64, 16384, 128 if group else 8)
        return dict(kind=kind, t=_log(rng, 1, min(16384, 100_000_000 // h)), h=h, residual=rng.random() < 0.7, group=group)
    if kind == "moe":
        dtype, k = rng.choice(["bf16", "bf16", "fp32"]), rng.randint(1, 8)
        h = _log(rng, 64, 8192, rng.choice([1, 8]))
        t = _log(rng, 1, min(16384, 100_000_000 // (h * k)))
        return dict(kind=kind, t=t, h=h, e=_log(rng, 4, 512), k=k, dtype=dtype, train=rng.random() < 0.7, drop=rng.random() < 0.4)
    if kind == "moe8":
        group, k = rng.choice([0, 128]), rng.randint(1, 8)
        h = _log(rng, 128, 8192, 128 if group else 16)
        return dict(kind=kind, t=_log(rng, 1, min(16384, 150_000_000 // (h * k))), h=h, e=_log(rng, 4, 512), k=k, group=group, drop=rng.random() < 0.4)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    return dict(kind=kind, tensors=_log(rng, 1, 500), n=_log(rng, 1000, 50_000_000), bits=rng.choice([8, 32]), dtype=dtype,
                master=dtype == "bf16" and rng.random() < 0.5, packed=rng.random() < 0.3)


# ------------------------------------------------------------------------------------------ inputs
class _State:
    """What the user's program holds: plain attributes."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _sizes(tensors: int, n: int) -> list[int]:
    """n elements in at most ``tensors`` tensors: every fourth is small, as norms and routers are, the others share the rest with odd remainders."""
    small = [1 + (7919 * i) % 509 for i in range(tensors // 4)]
    large = tensors - len(small)
    rest = max(large, n - sum(small))
    big = [rest // large] * large
    for i in range(0, large - 1, 2):   # pairs of a wide and a narrow one
        d = big[i] // 3
        big[i], big[i + 1] = big[i] + d, big[i + 1] - d
    big[0] += rest - sum(big)
    out, s, b = [], list(small), list(big)
    for i in range(tensors):
        out.append(s.pop() if i % 4 == 3 and s else b.pop(0) if b else s.pop())
    return out


def _views(flat: torch.Tensor, sizes: list[int], step: int) -> list[torch.Tensor]:
    """One tensor of each size in ``flat``, each from a multiple of ``step`` elements."""
    out, at = [], 0
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // step) * step
    return out


def _room(sizes: list[int], step: int) -> int:
    return sum(-(-n // step) * step for n in sizes)


def prepare(case: dict, seed: int) -> _State:
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]

    def rnd(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, device=DEV, generator=g, dtype=F32) * std).to(dtype)

    if kind == "norm8":
        t, h = case["t"], case["h"]
        return _State(kind=kind, x=rnd(t, h), res=rnd(t, h) if case["residual"] else None, w=(1 + rnd(h, std=0.1, dtype=F32)).to(BF16),
                      group=case["group"])
    if kind in ("moe", "moe8"):
        t, h, e, k = case["t"], case["h"], case["e"], case["k"]
        # tokens prefer some experts, as they do in a trained router
        scores = torch.randn(t, e, device=DEV, generator=g) + torch.randn(e, device=DEV, generator=g)
        w, idx = torch.topk(torch.softmax(scores, -1), min(k, e), dim=-1)
        w, idx = w.contiguous(), idx.to(torch.int32).contiguous()
        k = idx.shape[1]
        if case["drop"]:
            idx = torch.where(torch.rand(t, k, device=DEV, generator=g) < 0.1, -1, idx)
        if kind == "moe8":
            groups = h // case["group"] if case["group"] else 1
            x = rnd(t, h, std=100.0, dtype=F32).clamp(-448, 448).to(F8)
            scale = torch.rand(t, groups, device=DEV, generator=g) + 0.5
            return _State(kind=kind, idx=idx, e=e, x=x, scale=scale if case["group"] else scale.view(t))
        dt = BF16 if case["dtype"] == "bf16" else F32
        s = _State(kind=kind, idx=idx, e=e, train=case["train"], x=rnd(t, h, dtype=dt), w=w, y=rnd(t * k, h, dtype=dt))
        if case["drop"]:   # behind the last expert's rows nothing is to be read
            lost = (idx < 0).sum()
            s.y[torch.arange(t * k, device=DEV) >= t * k - lost] = math.nan
        if s.train:
            s.drows, s.dout = rnd(t * k, h, dtype=dt), rnd(t, h, dtype=dt)
            for v in (s.x, s.w, s.y):
                v.requires_grad_(True)
        return s
    sizes, step = _sizes(case["tensors"], case["n"]), 1 if case["packed"] else BLOCK
    room, dt = _room(sizes, step), BF16 if case["dtype"] == "bf16" else F32
    s = _State(kind=kind, bits=case["bits"], step=10, p=rnd(room, std=0.02, dtype=dt), g=rnd(room, std=1e-3, dtype=dt), master=None)
    s.params, s.grads = _views(s.p, sizes, step), _views(s.g, sizes, step)
    if case["master"]:
        s.master = s.p.float() + rnd(room, std=1e-5, dtype=F32)
    s.masters = _views(s.master, sizes, step) if case["master"] else None
    if s.bits == 32:
        s.m, s.v = rnd(room, std=3e-4, dtype=F32), rnd(room, std=1e-3, dtype=F32).square()
        s.ms = s.vs = s.m_scale = s.v_scale = None
    else:
        blocks = sum(-(-n // BLOCK) for n in sizes)
        s.m, s.v = rnd(room, std=120.0, dtype=F32).clamp(-448, 448).to(F8), rnd(room, std=120.0, dtype=F32).abs().clamp(2.0 ** -9, 448).to(F8)
        s.m_scale = (torch.rand(blocks, device=DEV, generator=g) + 0.5) * 2.5e-6
        s.v_scale = (torch.rand(blocks, device=DEV, generator=g) + 0.5) * 8e-6
        s.ms, s.vs = (_views(t, [-(-n // BLOCK) for n in sizes], 1) for t in (s.m_scale, s.v_scale))
    s.m_list, s.v_list = _views(s.m, sizes, step), _views(s.v, sizes, step)
    s.decay = [0.0 if n < 512 else DECAY for n in sizes]   # norms and the like are not decayed
    return s


# ------------------------------------------------------------------------------------------ one pass
def _rounded(y: torch.Tensor, group: int):
    """y [T, H] in 32 bits -> e4m3 and the scales of its rows or groups of columns."""
    v = y.view(y.shape[0], -1, group or y.shape[1])
    scale = v.abs().amax(-1, keepdim=True).clamp_min(1e-12) * (1.0 / 448.0)
    return (v * (1.0 / scale)).to(F8).view(y.shape), scale.view(y.shape[0], -1) if group else scale.view(-1)


def _norm8(s):
    h = s.x if s.res is None else (s.x.float() + s.res.float()).to(BF16)
    v = h.float()
    q, scale = _rounded(v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS_NORM) * s.w.float(), s.group)
    return {"q": q, "scale": scale, "h": h}


def _order(idx: torch.Tensor, e: int):
    """The row of each slot (~row where it goes to no expert), the rows where each expert begins, and the slot of each row."""
    key = idx.reshape(-1).long()
    key = torch.where((key < 0) | (key >= e), e, key)
    slot = torch.argsort(key, stable=True)
    row = torch.empty_like(slot)
    row[slot] = torch.arange(slot.numel(), device=DEV)
    counts = torch.zeros(e + 1, device=DEV, dtype=torch.int64).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)[:e])).int()
    return torch.where(key < e, row, ~row).int().view(idx.shape), offsets, slot, key < e


def _moe(s):
    row_of, offsets, slot, live = _order(s.idx, s.e)
    t, k = s.idx.shape
    there = live[slot][:, None]
    if s.kind == "moe8":
        rows = torch.where(there, s.x[slot // k].float(), 0.0).to(F8)
        scale = s.scale.view(t, -1)[slot // k]
        scale = torch.where(there, scale, 0.0)
        return {"row_of": row_of, "offsets": offsets, "rows": rows, "scale": scale.view(-1, *s.scale.shape[1:])}
    dt = s.x.dtype
    at = torch.where(row_of < 0, ~row_of, row_of).long()
    took = live.view(t, k, 1)
    rows = torch.where(there, s.x.detach()[slot // k], 0.0)
    y, w = s.y.detach(), s.w.detach()
    out = torch.where(took, w[..., None] * y[at].float(), 0.0).sum(1).to(dt)
    got = {"row_of": row_of, "offsets": offsets, "rows": rows, "out": out}
    if s.train:
        got["dx"] = torch.where(took, s.drows[at].float(), 0.0).sum(1).to(dt)
        got["dy"] = torch.where(there, (w.view(-1)[slot][:, None] * s.dout[slot // k].float()), 0.0).to(dt)
        got["dw"] = torch.where(live.view(t, k), (s.dout.float()[:, None] * torch.where(took, y[at].float(), 0.0)).sum(-1), 0.0)
    return got


def _dither(n: int, step: int) -> torch.Tensor:
    """32 bits for each element of a tensor: the R2 sequence (the plane's additive recurrence) of element and step."""
    return (torch.arange(n, device=DEV, dtype=torch.int64) * 0xC13FA9A9 + step * 0x91E10DA5) & 0xFFFFFFFF


def _blocks(x: torch.Tensor) -> torch.Tensor:
    """[n] -> [blocks, BLOCK], with zeros behind the last element."""
    n = x.numel()
    return torch.cat((x, x.new_zeros(-n % BLOCK))).view(-1, BLOCK)


def _held8(x: torch.Tensor, dither: torch.Tensor):
    """x [n] in 32 bits -> e4m3 codes of |x| and the blocks' scales. A value rounds up where the dither's top bits exceed what is missing to
    the next one: scaled by 2^-120 the bits of e4m3 and of fp32 are in the same places, below the least normal number too."""
    b = _blocks(x.abs())
    scale = b.amax(-1, keepdim=True).clamp_min(1e-30) / 448.0
    bits = (b * (1.0 / scale) * 2.0 ** -120).view(torch.int32).long().view(-1)[:x.numel()]
    return ((bits + (dither >> 12)) >> 20).clamp_max(0x7E), scale.view(-1)


def _adamw(s, i: int):
    p, g, m, v = s.params[i], s.grads[i].float(), s.m_list[i], s.v_list[i]
    n, step = p.numel(), s.step
    x = s.masters[i] if s.masters is not None else p.float()
    if s.bits == 32:
        m1, v1 = m, v
    else:
        m1 = (_blocks(m.float()) * s.ms[i][:, None]).view(-1)[:n]
        root = (_blocks(v.float()) * s.vs[i][:, None]).view(-1)[:n]
        v1 = root * root
    m1 = m1 * BETA1 + g * (1 - BETA1)
    v1 = v1 * BETA2 + (g * g) * (1 - BETA2)
    root = v1.sqrt()
    x = x * (1 - LR * s.decay[i]) - (m1 * (LR / (1 - BETA1 ** step))) / (root * (1 / math.sqrt(1 - BETA2 ** step)) + EPS)
    p.copy_(x)
    if s.masters is not None:
        s.masters[i].copy_(x)
    if s.bits == 32:
        m.copy_(m1)
        v.copy_(v1)
        return
    d = _dither(n, step)
    code, scale = _held8(m1, d)
    m.copy_((code | ((m1.view(torch.int32).long() >> 24) & 0x80)).to(torch.uint8).view(F8))
    s.ms[i].copy_(scale)
    code, scale = _held8(root, d ^ 0xFFFFFFFF)
    v.copy_(torch.maximum(code, (root > 0).long()).to(torch.uint8).view(F8))   # what is not zero is not held as zero
    s.vs[i].copy_(scale)


def _updated(s):
    got = {"p": s.p, "m": s.m, "v": s.v, "master": s.master, "m_scale": s.m_scale, "v_scale": s.v_scale}
    return {k: v for k, v in got.items() if v is not None}


def run(s: _State):
    if not own:
        with torch.no_grad():
            if s.kind == "norm8":
                return _norm8(s)
            if s.kind in ("moe", "moe8"):
                return _moe(s)
            _ = [_adamw(s, i) for i in range(len(s.params))]
            return _updated(s)
    from aws_ofi_nccl_b200.ops import llm, moe

    if s.kind == "norm8":
        q, scale, h = llm.rmsnorm_fp8(s.x, s.w, EPS_NORM, residual=s.res, group=s.group)
        return {"q": q, "scale": scale, "h": h}
    if s.kind == "adamw":
        llm.adamw_step_many(s.params, s.grads, s.m_list, s.v_list, s.ms, s.vs, s.masters, lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                            weight_decay=s.decay, step=s.step, zero_grad=False)
        return _updated(s)
    order = moe.expert_order(s.idx, s.e)
    if s.kind == "moe8":
        rows, scale = moe.permute_tokens(s.x, order, s.scale)
        return {"row_of": order.row_of, "offsets": order.offsets, "rows": rows, "scale": scale}
    rows = moe.permute_tokens(s.x, order)
    out = moe.unpermute_tokens(s.y, order, s.w)   # what the experts made of the rows is another tensor
    got = {"row_of": order.row_of, "offsets": order.offsets, "rows": rows.detach(), "out": out.detach()}
    if s.train:
        got["dx"], got["dy"], got["dw"] = torch.autograd.grad((rows, out), (s.x, s.y, s.w), (s.drows, s.dout))
    return got


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "norm8":   # x and its 8-bit rows; with a residual also that and their sum
        t, h = case["t"], case["h"]
        return {"bytes": t * h * (7 if case["residual"] else 3) + 4 * t * (h // case["group"] if case["group"] else 1) + 2 * h, "flops": 0}
    if kind in ("moe", "moe8"):
        t, h, k = case["t"], case["h"], min(case["k"], case["e"])
        sort = 8 * t * k + 4 * (case["e"] + 1)
        if kind == "moe8":
            scales = 4 * (h // case["group"] if case["group"] else 1)
            return {"bytes": sort + t * (1 + k) * (h + scales), "flops": 0}
        size = 2 if case["dtype"] == "bf16" else 4
        # x, out and the rows of both ways; backward dx, dout, drows, dy and the weights' gradient
        return {"bytes": sort + size * t * h * (2 + 2 * k) * (2 if case["train"] else 1) + 4 * t * k * (2 if case["train"] else 1), "flops": 0}
    size = 2 if case["dtype"] == "bf16" else 4
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    # p, g, the state and the master copy; beside a master copy p is only written
    n = sum(_sizes(case["tensors"], case["n"]))
    return {"bytes": n * (size + state + (size + 8 if case["master"] else 2 * size)), "flops": 0}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_moe(case, s):
    idx = s.idx.cpu().long()
    t, k = idx.shape
    e = s.e
    flat = idx.reshape(-1)
    ok = (flat >= 0) & (flat < e)
    # the rows expert by expert, a slot's place within its expert counted from the front
    kept = [torch.nonzero(ok & (flat == x)).view(-1) for x in range(e)] + [torch.nonzero(~ok).view(-1)]
    offsets = torch.tensor([0] + [q.numel() for q in kept[:e]]).cumsum(0)
    slots = torch.cat(kept)
    row = torch.empty(t * k, dtype=torch.int64)
    row[slots] = torch.arange(t * k)
    row_of = torch.where(ok, row, -1 - row).view(t, k)
    token, n = (slots // k).to(DEV), int(offsets[-1])
    head = {"row_of": row_of.int().to(DEV), "offsets": offsets.int().to(DEV)}
    if s.kind == "moe8":
        rows = s.x.double()[token]
        rows[n:] = 0
        scale = s.scale.double()[token]
        scale[n:] = 0
        return {**head, "rows": rows, "scale": scale}
    rows = s.x.detach().double()[token]
    rows[n:] = 0
    out = torch.zeros(t, s.x.shape[1], device=DEV, dtype=torch.float64)
    y, w = s.y.detach().double()[:n], s.w.detach().double().view(-1)[slots.to(DEV)][:n]
    out.index_add_(0, token[:n], y * w[:, None])
    got = {**head, "rows": rows, "out": out}
    if s.train:
        dx = torch.zeros_like(out)
        dx.index_add_(0, token[:n], s.drows.double()[:n])
        d = s.dout.double()[token]
        dw = torch.zeros(t * k, device=DEV, dtype=torch.float64)
        dw[slots.to(DEV)[:n]] = (d[:n] * y).sum(-1)
        d[:n] *= w[:, None]
        d[n:] = 0
        got |= {"dx": dx, "dy": d, "dw": dw.view(t, k)}
    return got


def _exact_e4m3(y, u):
    """The value of e4m3 below or above y >= 0, up where what is missing to the one above is less than u's share of a step."""
    step = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
    return (torch.floor(y / step + u) * step).clamp_max(448.0)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm8":
        h = s.x.double() + (s.res.double() if s.res is not None else 0)
        v = h.to(BF16).double()   # the sum is normalised as it is stored
        y = v / (v.square().mean(-1, keepdim=True) + EPS_NORM).sqrt() * s.w.double()
        group = case["group"] or case["h"]
        b = y.view(y.shape[0], -1, group)
        scale = b.abs().amax(-1) / 448
        q = (b / scale[..., None]).view(y.shape)   # unrounded: rounding is part of what is measured
        return {"q": q, "scale": scale if case["group"] else scale.view(-1), "h": h}
    if kind in ("moe", "moe8"):
        return _exact_moe(case, s)
    got = {k: v.double() for k, v in _updated(s).items()}
    sizes, pad = [p.numel() for p in s.params], 1 if case["packed"] else BLOCK
    out = {k: _views(v, [-(-n // BLOCK) for n in sizes] if k in ("m_scale", "v_scale") else sizes, 1 if k in ("m_scale", "v_scale") else pad)
           for k, v in got.items()}
    t = s.step
    for i, n in enumerate(sizes):
        g = s.grads[i].double()
        x = out["master" if s.master is not None else "p"][i].clone()
        m, v = out["m"][i], out["v"][i]
        which = torch.arange(n, device=DEV) // BLOCK
        if s.bits == 8:
            m, v = m * out["m_scale"][i][which], (v * out["v_scale"][i][which]).square()
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        x -= LR * s.decay[i] * x + LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["p"][i].copy_(x)
        if s.master is not None:
            out["master"][i].copy_(x)
        if s.bits == 32:
            out["m"][i].copy_(m)
            out["v"][i].copy_(v)
            continue
        word = torch.remainder(torch.arange(n, device=DEV) * 3242174889 + t * 2447445413, 2 ** 32)
        for name, z, word_z in (("m", m, word), ("v", v.sqrt(), 2 ** 32 - 1 - word)):
            top = torch.zeros(-(-n // BLOCK), device=DEV, dtype=torch.float64).scatter_reduce_(0, which, z.abs(), "amax") / 448
            held = _exact_e4m3(z.abs() / top[which], torch.floor(word_z / 4096) / 2 ** 20)
            if name == "v":
                held = torch.maximum(held, (z > 0) * 2.0 ** -9)
            out[name][i].copy_(torch.copysign(held, z))
            out[name + "_scale"][i].copy_(top)
    return got
