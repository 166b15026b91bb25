"""Training on long sequences, operator by operator: attention with a sliding window and first tokens that stay visible, and layers that keep
what their backward pass needs in 8 bits.

Every case is a plain dict with a "kind"; sizes are those of the Llama-3-8B and tiny configurations of ``models/llama.py`` and of the tests,
plus generic odd ones. With ``own`` false ``run`` computes the operators from elementary torch operations in 32 bits, with it true through
the framework.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
GROUP = 32            # elements of a row that share a power of two
CHUNK = 1024          # queries that the plain form takes at a time


def listed() -> list[dict]:
    return [
        # the tiny model's batch in training: launches and the host decide
        dict(name="attn_tiny", kind="attention", b=2, s=128, nq=4, nkv=2, hd=64, window=32, sinks=2, train=True, ragged=False),
        # the 8B configuration's heads over one full sequence of it, all keys visible, in training
        dict(name="attn_full_train", kind="attention", b=1, s=4096, nq=32, nkv=8, hd=128, window=0, sinks=0, train=True, ragged=False),
        # the same heads over a long document with a window, in training
        dict(name="attn_window_train", kind="attention", b=1, s=16384, nq=32, nkv=8, hd=128, window=1024, sinks=4, train=True, ragged=False),
        # evaluation of a longer one: forward only
        dict(name="attn_window_eval", kind="attention", b=1, s=32768, nq=32, nkv=8, hd=128, window=4096, sinks=4, train=False, ragged=False),
        # a padded batch of odd lengths, heads of 64, three of them to a key
        dict(name="attn_ragged_train", kind="attention", b=4, s=1777, nq=12, nkv=4, hd=64, window=300, sinks=7, train=True, ragged=True),
        # a projection of the tiny model: the smallest layer that keeps its input
        dict(name="linear8_small", kind="linear8", m=256, n=768, k=256),
        # the fused projection of the 8B configuration over one sequence
        dict(name="linear8_layer", kind="linear8", m=4096, n=6144, k=4096),
        # a packed batch with a ragged token count through a layer whose widths fill no tile and no group
        dict(name="linear8_ragged", kind="linear8", m=1000, n=2568, k=5160),
        # the tiny model's activation
        dict(name="swiglu8_small", kind="swiglu8", t=256, f=512),
        # the 8B configuration's over one sequence
        dict(name="swiglu8_layer", kind="swiglu8", t=4096, f=14336),
        # an expert's ragged rows of a width that ends inside a group
        dict(name="swiglu8_ragged", kind="swiglu8", t=5003, f=2744),
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max((lo + step - 1) // step * step, min(hi // step * step, int(round(v / step)) * step))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "attention", "linear8", "swiglu8"])
    if kind == "attention":
        while True:
            nkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
            s, hd = _log(rng, 1, 16384), rng.choice([64, 128])
            window = rng.choice([0, 0, _log(rng, 1, 4096), _log(rng, 1, 4096), _log(rng, 1, 4096)])
            sinks = rng.choice([0, rng.randint(1, 16), _log(rng, 1, 400)]) if window else 0
            case = dict(kind=kind, b=rng.randint(1, 4), s=s, nq=nkv * group, nkv=nkv, hd=hd, window=window, sinks=sinks, train=rng.random() < 0.7,
                        ragged=rng.random() < 0.4)
            if work(case)["flops"] <= 6e11 and case["b"] * s * case["nq"] * hd <= 70_000_000:
                return case
    if kind == "linear8":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 64, 14336, 8), _log(rng, 64, 14336, 8)
            if m * n * k <= 1.03e11:
                return dict(kind=kind, m=m, n=n, k=k)
    f = _log(rng, 8, 16384, 8)
    return dict(kind=kind, t=_log(rng, 1, min(65536, 58_000_000 // f)), f=f)


# ------------------------------------------------------------------------------------------ inputs
class _State:
    """What the user's program holds: plain attributes."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _lengths(case) -> list[int]:
    """How many tokens each sequence of the batch has: in a ragged one the first is full, the others are shorter by odd amounts."""
    b, s = case["b"], case["s"]
    return [max(1, s - (s * 5 * i) // (8 * b) - i) if case["ragged"] else s for i in range(b)]


def prepare(case: dict, seed: int) -> _State:
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=g, dtype=F32) * std).to(BF16)

    if kind == "attention":
        b, s, nq, nkv, hd = (case[x] for x in ("b", "s", "nq", "nkv", "hd"))
        st = _State(kind=kind, q=rnd(b, s, nq, hd, std=1.5), k=rnd(b, s, nkv, hd), v=rnd(b, s, nkv, hd), window=case["window"], sinks=case["sinks"],
                    train=case["train"], spans=_lengths(case), lengths=None, do=None)
        if case["ragged"]:
            st.lengths = torch.tensor(st.spans, dtype=torch.int32, device=DEV)
        if st.train:
            st.do = rnd(b, s, nq, hd)
            for x in (st.q, st.k, st.v):
                x.requires_grad_(True)
        return st
    if kind == "linear8":
        m, n, k = case["m"], case["n"], case["k"]
        # some channels are larger than others, as they are behind a norm
        wide = torch.exp(torch.randn(k, device=DEV, generator=g))
        x = (torch.randn(m, k, device=DEV, generator=g) * wide).to(BF16).requires_grad_(True)
        return _State(kind=kind, x=x, w=rnd(n, k, std=k ** -0.5).requires_grad_(True), dy=rnd(m, n))
    t, f = case["t"], case["f"]
    return _State(kind=kind, gu=rnd(t, 2 * f, std=1.5).requires_grad_(True), dout=rnd(t, f))


# ------------------------------------------------------------------------------------------ one pass
def _spans(s, n: int):
    """Chunks of queries [a, b) of a sequence of n tokens with the keys that any of them sees: the sinks in front, then [lo, b)."""
    for a in range(0, n, CHUNK):
        b = min(n, a + CHUNK)
        lo = max(0, a - s.window + 1) if s.window else 0
        yield a, b, lo, min(s.sinks, lo)


def _attention(s):
    q, k, v = s.q.detach(), s.k.detach(), s.v.detach()
    B, S, nq, hd = q.shape
    nkv = k.shape[2]
    G, scale = nq // nkv, hd ** -0.5
    out = torch.zeros_like(q)
    got = {"out": out}
    if s.train:
        dq, dk, dv = torch.zeros_like(q), torch.zeros(B, S, nkv, hd, device=DEV), torch.zeros(B, S, nkv, hd, device=DEV)
    for i in range(B):
        for a, b, lo, first in _spans(s, s.spans[i]):
            at = torch.cat((torch.arange(first, device=DEV), torch.arange(lo, b, device=DEV)))
            rows = torch.arange(a, b, device=DEV)[:, None]
            sees = at <= rows
            if s.window:
                sees &= (rows - at < s.window) | (at < s.sinks)

            def heads(x):   # [b - a, nq, hd] -> [nkv, G * (b - a), hd]
                return x[i, a:b].float().view(b - a, nkv, G, hd).permute(1, 2, 0, 3).reshape(nkv, G * (b - a), hd)

            def back(x):
                return x.view(nkv, G, b - a, hd).permute(2, 0, 1, 3).reshape(b - a, nq, hd)

            qf, kf, vf = heads(q), k[i, at].float().transpose(0, 1), v[i, at].float().transpose(0, 1)
            p = (qf @ kf.transpose(1, 2)).mul_(scale).view(nkv, G, b - a, -1)
            p = p.masked_fill_(~sees, -math.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True)).view(nkv, G * (b - a), -1)
            o = p @ vf
            out[i, a:b] = back(o)
            if s.train:
                do = heads(s.do)
                dv[i].index_add_(0, at, (p.transpose(1, 2) @ do).transpose(0, 1))
                ds = (do @ vf.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                dq[i, a:b] = back(ds @ kf)
                dk[i].index_add_(0, at, (ds.transpose(1, 2) @ qf).transpose(0, 1))
    if s.train:
        got |= {"dq": dq, "dk": dk.to(BF16), "dv": dv.to(BF16)}
    return got


def _kept(x: torch.Tensor) -> torch.Tensor:
    """x [rows, n] in 32 bits as 8 bits hold it: e4m3 codes times the least power of two of a group under which its largest fits."""
    rows, n = x.shape
    g = torch.cat((x, x.new_zeros(rows, -n % GROUP)), 1).view(rows, -1, GROUP)
    part, power = torch.frexp(g.abs().amax(-1, keepdim=True))   # part in [0.5, 1) times 2^power; 448 is 0.875 * 2^9
    power = torch.where(part > 0.875, power - 8, power - 9).clamp_min(-127)
    return torch.ldexp(torch.ldexp(g, -power).to(F8).float(), power).view(rows, -1)[:, :n]


def _linear8(s):
    x, w, dy = s.x.detach().float(), s.w.detach().float(), s.dy.float()
    return {"y": (x @ w.t()).to(BF16), "dx": (dy @ w).to(BF16), "dw": (dy.t() @ _kept(x)).to(BF16)}


def _swiglu8(s):
    gu, d = s.gu.detach().float(), s.dout.float()
    g, u = gu.chunk(2, 1)
    act = (g * torch.sigmoid(g) * u).to(BF16)
    g, u = _kept(g), _kept(u)
    sig = torch.sigmoid(g)
    return {"act": act, "dgu": torch.cat((d * u * sig * (1 + g * (1 - sig)), d * g * sig), 1).to(BF16)}


def run(s: _State):
    if not own:
        with torch.no_grad():
            return {"attention": _attention, "linear8": _linear8, "swiglu8": _swiglu8}[s.kind](s)
    from aws_ofi_nccl_b200.ops import attention, gemm, llm

    if s.kind == "attention":
        out = attention.attention(s.q, s.k, s.v, window=s.window, sinks=s.sinks, lengths=s.lengths)
        got = {"out": out.detach()}
        if s.train:
            got["dq"], got["dk"], got["dv"] = torch.autograd.grad(out, (s.q, s.k, s.v), s.do)
        return got
    if s.kind == "linear8":
        y = gemm.linear(s.x, s.w, keep_bits=8)
        dx, dw = torch.autograd.grad(y, (s.x, s.w), s.dy)
        return {"y": y.detach(), "dx": dx, "dw": dw}
    act = llm.swiglu(s.gu, keep_bits=8)
    return {"act": act.detach(), "dgu": torch.autograd.grad(act, s.gu, s.dout)[0]}


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(n: int, window: int, sinks: int) -> int:
    """Visible pairs of a sequence of n tokens: each query's own window, and the sinks in front of it."""
    if window == 0 or window >= n:
        return n * (n + 1) // 2
    near = window * (window + 1) // 2 + (n - window) * window
    # query i sees min(sinks, i - window + 1) keys in front of its window
    far = n - window
    few = min(sinks, far)
    return near + few * (few + 1) // 2 + (far - few) * few


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "attention":
        tokens = sum(_lengths(case))
        pairs = sum(_pairs(n, case["window"], case["sinks"]) for n in _lengths(case)) * case["nq"]
        whole = case["b"] * case["s"]
        q, kv = 2 * case["nq"] * case["hd"], 4 * case["nkv"] * case["hd"]   # bytes a token: q; k and v
        size = tokens * (q + kv) + whole * q                                # inputs; out, zeros of rows behind a sequence too
        if case["train"]:
            size += tokens * q + whole * (q + kv)
        return {"bytes": size, "flops": pairs * case["hd"] * (14 if case["train"] else 4)}
    if kind == "linear8":
        m, n, k = case["m"], case["n"], case["k"]
        kept = m * (k + -(-k // GROUP))
        # x w dy in, y dx dw out; what is kept is written and read
        return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n) + 2 * kept, "flops": 6 * m * n * k}
    t, f = case["t"], case["f"]
    return {"bytes": t * (4 * f + 2 * f + 2 * f + 4 * f + 4 * (f + -(-f // GROUP))), "flops": 0}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_attention(s):
    """Dense rows of scores with the mask as it is defined, and the derivatives that torch takes of them."""
    B, S, nq, hd = s.q.shape
    nkv = s.k.shape[2]
    q, k, v = (x.detach().double().transpose(1, 2) for x in (s.q, s.k, s.v))
    out = torch.zeros(B, nq, S, hd, device=DEV, dtype=F64)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if s.train else None
    step = max(16, min(512, 60_000_000 // (S * nq // nkv)))
    for b in range(B):
        n = s.spans[b]
        for h in range(nkv):
            own_heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            for i0 in range(0, n, step):
                i1 = min(n, i0 + step)
                i, j = torch.arange(i0, i1, device=DEV)[:, None], torch.arange(i1, device=DEV)[None]
                hidden = j > i
                if s.window > 0:
                    hidden = hidden | ((j <= i - s.window) & (j >= s.sinks))
                part = [q[b, own_heads, i0:i1], k[b, h, :i1], v[b, h, :i1]]
                with torch.set_grad_enabled(s.train):
                    if s.train:
                        part = [x.clone().requires_grad_(True) for x in part]
                    logits = torch.einsum("gid,jd->gij", part[0], part[1]) / math.sqrt(hd)
                    logits = logits.masked_fill(hidden, -math.inf)
                    o = torch.einsum("gij,jd->gid", torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True)), part[2])
                out[b, own_heads, i0:i1] = o.detach()
                if s.train:
                    d = torch.autograd.grad(o, part, s.do[b, i0:i1, own_heads].double().transpose(0, 1))
                    grads[0][b, own_heads, i0:i1] = d[0]
                    grads[1][b, h, :i1] += d[1]
                    grads[2][b, h, :i1] += d[2]
    got = {"out": out.transpose(1, 2)}
    if s.train:
        got |= {name: x.transpose(1, 2) for name, x in zip(("dq", "dk", "dv"), grads)}
    return got


def _exact_kept(x):
    """The value of e4m3 nearest to x / 2^e, ties to the even one, with the least e for which no value of the group is beyond 448."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], GROUP):
        v = x[:, c:c + GROUP]
        top = v.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -150) / 448)).clamp_min(-127)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)   # the logarithm is rounded
        e = torch.where((top <= 224 * torch.exp2(e)) & (e > -127), e - 1, e)
        y = v / torch.exp2(e)
        place = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, c:c + GROUP] = torch.round(y / place) * place * torch.exp2(e)
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s.kind == "attention":
        if case["b"] * case["s"] ** 2 * case["nq"] * case["hd"] > 6e12:   # dense rows in 64 bits
            return None
        return _exact_attention(s)
    if s.kind == "linear8":
        x, w, dy = s.x.detach().double(), s.w.detach().double(), s.dy.double()
        return {"y": torch.einsum("mk,nk->mn", x, w), "dx": torch.einsum("mn,nk->mk", dy, w), "dw": torch.einsum("mn,mk->nk", dy, _exact_kept(x))}
    gate, up = s.gu.detach().double().split(case["f"], 1)
    act = gate / (1 + torch.exp(-gate)) * up
    kg, ku, d = _exact_kept(gate), _exact_kept(up), s.dout.double()
    e = torch.exp(-kg)
    slope = (1 + e + kg * e) / (1 + e) ** 2
    return {"act": act, "dgu": torch.cat((d * ku * slope, d * kg / (1 + e)), 1)}
