"""Mixture-of-experts layer: softmax top-k router, device-initiated dispatch of the
token rows to the ranks that own their experts (optionally as block-scaled fp8), SwiGLU experts
on the tcgen05 GEMM, gate-weighted combine back to token order.  Without a communicator all experts
are on one GPU: rows are sorted by expert and summed back without a window, any number of tokens at a time."""
from __future__ import annotations

import torch

from ..ops.gemm import linear
from ..ops.llm import swiglu
from ..ops.moe import expert_order, permute_tokens, unpermute_tokens
from ..parallel.expert_parallel import ExpertParallel
from ..parallel.symm import Communicator


class MoELayer(torch.nn.Module):
    def __init__(self, comm: Communicator | None, tokens: int, hidden: int, ffn: int, experts: int, topk: int, *,
                 fp8_dispatch: bool = False, capacity_factor: float = 2.0, window_offset: int = 0, seed: int = 0,
                 device: torch.device | str | None = None):
        """comm None: all experts on ``device`` (default: the current GPU); ``tokens`` and the window's arguments then mean nothing."""
        super().__init__()
        if comm is None:
            if fp8_dispatch:
                raise ValueError("fp8_dispatch is for rows that travel between ranks: it needs a communicator")
            self.ep, world, rank = None, 1, 0
            dev = torch.device(device if device is not None else "cuda")
        else:
            asked = torch.device(device) if device is not None else comm.device
            if asked.type != comm.device.type or asked.index not in (None, comm.device.index):
                raise ValueError("the layer is on its communicator's device")
            self.ep = ExpertParallel(comm, tokens, hidden, experts, topk, capacity_factor=capacity_factor,
                                     window_offset=window_offset)
            world, rank, dev = comm.world, comm.rank, comm.device
        self.hidden, self.ffn, self.experts, self.topk, self.fp8 = hidden, ffn, experts, topk, fp8_dispatch
        el = experts // world
        g = torch.Generator(device="cpu").manual_seed(seed)
        router = torch.randn(experts, hidden, generator=g) * hidden ** -0.5
        w_gu = torch.randn(experts, 2 * ffn, hidden, generator=g) * hidden ** -0.5
        w_dn = torch.randn(experts, hidden, ffn, generator=g) * ffn ** -0.5
        lo = rank * el
        self.router = torch.nn.Parameter(router.to(dev))   # fp32, replicated
        self.w_gate_up = torch.nn.ParameterList(
            [torch.nn.Parameter(w_gu[lo + e].to(dev, torch.bfloat16)) for e in range(el)])
        self.w_down = torch.nn.ParameterList(
            [torch.nn.Parameter(w_dn[lo + e].to(dev, torch.bfloat16)) for e in range(el)])
        self._full = (router, w_gu, w_dn)  # CPU fp32 copies of all experts (reference checks only)

    def route(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        probs = torch.softmax(x.float() @ self.router.t(), dim=-1)
        w, idx = torch.topk(probs, self.topk, dim=-1)
        return idx.to(torch.int32).contiguous(), w.contiguous()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        idx, w = self.route(x)
        if self.ep is None:
            order = expert_order(idx, self.experts)
            rows, offsets = permute_tokens(x, order), order.offsets
        else:
            rows, offsets = self.ep.dispatch(x, idx, w, self.fp8), self.ep.expert_offsets
        # The per-expert row ranges live on the device; slicing the rows for the per-expert GEMM
        # calls needs them on the host.
        off = [min(n, rows.shape[0]) for n in offsets.tolist()]   # rows beyond the window's capacity have raised its status
        counts = [b - a for a, b in zip(off, off[1:])]
        outs = []
        # cut at once: the rows' gradient is one concatenation, where that of a slice would be a matrix of all rows for each expert
        for e, seg in enumerate(rows.split([*counts, rows.shape[0] - off[-1]])[:-1]):
            if counts[e]:
                outs.append(linear(swiglu(linear(seg, self.w_gate_up[e])), self.w_down[e]))
        if outs:
            y = torch.cat(outs, dim=0)
        else:
            y = rows[:0]
        return self.ep.combine(y, w) if self.ep is not None else unpermute_tokens(y, order, w)
