"""Training engine: the public entry point a user calls for a Llama training step.

``Trainer.step(ids_host, labels_host)`` runs one full optimizer step — host-to-device copy of the
batch from pinned memory, forward, backward (with the gradient all-reduce of a data-parallel job
overlapped behind it), fused AdamW — and returns the loss as a Python float (device-to-host read).
Waits in kernels are bounded; where one gave up, the step raises instead.
"""
from __future__ import annotations

import dataclasses
import math

import torch

from ..models.llama import Llama, LlamaConfig
from ..ops import _lib
from ..ops import llm as llm_ops


@dataclasses.dataclass
class OptimConfig:
    lr: float = 3e-4
    beta1: float = 0.9
    beta2: float = 0.95
    eps: float = 1e-8
    weight_decay: float = 0.1
    master_weights: bool = True
    state_bits: int = 32   # of the moments: 32, or 8 with a scale for every 256 of a parameter (six bytes less for each parameter)


class Trainer:
    def __init__(self, cfg: LlamaConfig, optim: OptimConfig | None = None, device="cuda", dp=None, seed: int = 0):
        """dp: an optional ``parallel.data_parallel.GradReducer`` (owns the symmetric gradient buffer)."""
        self.cfg = cfg
        self.optim = optim or OptimConfig()
        self.device = torch.device(device)
        self.dp = dp
        grad_buffer = dp.allocate_grad_buffer(self._padded_numel(cfg)) if dp is not None else None
        self.model = Llama(cfg, device=self.device, grad_buffer=grad_buffer, seed=seed)
        n = self.model.numel
        # a reducer in "zero" mode leaves each rank the optimizer state of its own shard only
        self.shard = dp.shard_range(n) if getattr(dp, "mode", "") == "zero" else (0, n)
        lo, hi = self.shard
        flat = self.model.flat_params[lo:hi]
        moments = llm_ops.adamw_states([flat], bits=self.optim.state_bits)
        self.m, self.v = moments["m"][0], moments["v"][0]
        self.m_scale = self.v_scale = None
        self.master = flat.float() if self.optim.master_weights else None
        if self.optim.state_bits == 8:
            self._by_parameter(lo, hi)
        self.step_count = 0
        self.kernel_launches = 0
        if dp is not None:
            dp.attach(self.model)
        self._ids_dev = None
        self._labels_dev = None

    def _by_parameter(self, lo: int, hi: int) -> None:
        """Moments in 8 bits are stepped parameter by parameter, so that no scale is that of two: a norm's moments are of another size than a matrix's."""
        spans = [(max(at, lo), min(at + math.prod(shape), hi)) for at, shape in self.model.offsets.values()]
        spans = [(a, b) for a, b in spans if a < b]
        blocks = [-(-(b - a) // llm_ops.ADAMW_BLOCK) for a, b in spans]
        self.m_scale, self.v_scale = (torch.zeros(sum(blocks), device=self.device, dtype=torch.float32) for _ in "mv")
        of_model = lambda flat: [flat[a:b] for a, b in spans]                 # noqa: E731
        of_shard = lambda flat: [flat[a - lo:b - lo] for a, b in spans]       # noqa: E731
        masters = of_shard(self.master) if self.master is not None else [None] * len(spans)
        self._pieces = (of_model(self.model.flat_params), of_model(self.model.flat_grads), of_shard(self.m), of_shard(self.v),
                        list(self.m_scale.split(blocks)), list(self.v_scale.split(blocks)), masters)
        # whether blocks of 256 counted from the shard's beginning would be the same
        self._blocks_as_flat = all((a - lo) % llm_ops.ADAMW_BLOCK == 0 for a, _ in spans)

    @staticmethod
    def _padded_numel(cfg: LlamaConfig) -> int:
        return sum((math.prod(s) + 127) // 128 * 128 for _, s in cfg.param_shapes())

    # ------------------------------------------------------------------ one optimizer step, device tensors in
    def step_device(self, ids: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        model, oc = self.model, self.optim
        launched = _lib.launch_count
        model.reset_grad_flags()
        if self.dp is not None:
            self.dp.begin_step()
        loss = model.forward_loss(ids, labels)
        loss.backward()
        if self.dp is not None:
            self.dp.finish_step()  # all buckets reduced (averaged) in place in the flat gradient buffer
        self.step_count += 1
        lo, hi = self.shard
        grad_scale = float(getattr(self.dp, "grad_scale", 1.0))   # reducers that sum leave the 1/N to the optimizer
        hyper = dict(lr=oc.lr, beta1=oc.beta1, beta2=oc.beta2, eps=oc.eps, weight_decay=oc.weight_decay, step=self.step_count,
                     grad_scale=grad_scale, zero_grad=True)
        if self.m_scale is None:
            llm_ops.adamw_step(model.flat_params[lo:hi], model.flat_grads[lo:hi], self.m, self.v, self.master, **hyper)
        else:
            llm_ops.adamw_step_many(*self._pieces, **hyper)
        if (lo, hi) != (0, model.numel):
            if lo > 0:
                model.flat_grads[:lo].zero_()
            if hi < model.numel:
                model.flat_grads[hi:].zero_()
            self.dp.gather_params(model.flat_params)
        self.kernel_launches = _lib.launch_count - launched
        return loss.detach()

    # ------------------------------------------------------------------ end to end: pinned host batch in, float out
    def step(self, ids_host: torch.Tensor, labels_host: torch.Tensor) -> float:
        if self._ids_dev is None or self._ids_dev.shape != ids_host.shape:
            self._ids_dev = torch.empty(ids_host.shape, device=self.device, dtype=torch.int64)
            self._labels_dev = torch.empty(labels_host.shape, device=self.device, dtype=torch.int64)
        self._ids_dev.copy_(ids_host, non_blocking=True)
        self._labels_dev.copy_(labels_host, non_blocking=True)
        loss = float(self.step_device(self._ids_dev, self._labels_dev).item())
        status = _lib.read_status()
        if status != 0:
            raise _lib.B200OpsError(f"a wait in a kernel gave up (status {status}): the parameters may be wrong from this step on")
        return loss

    def launches_per_step(self) -> int:
        """Number of this library's kernels that the last step launched (0 in front of the first), by their counter: how many products share a launch, and whether attention
        joins the sums of sinks, depends on the batch's shape."""
        return self.kernel_launches

    # ------------------------------------------------------------------ checkpoint / resume
    def state_dict(self) -> dict:
        scales = {} if self.m_scale is None else {"m_scale": self.m_scale, "v_scale": self.v_scale, "scale_blocks": "parameter"}
        return {
            "params": self.model.flat_params, "m": self.m, "v": self.v, "master": self.master, **scales,
            "step": self.step_count, "rng_cpu": torch.get_rng_state(),
            "rng_cuda": torch.cuda.get_rng_state(self.device) if self.device.type == "cuda" else None,
        }

    def load_state_dict(self, sd: dict) -> None:
        if ("m_scale" in sd) != (self.m_scale is not None):
            raise ValueError(f"the moments are held in {self.optim.state_bits} bits, the saved ones are not")
        if self.m_scale is not None:
            if sd.get("scale_blocks") != "parameter" and not self._blocks_as_flat:
                raise ValueError("the saved scales are of blocks that hold more than one parameter")
            self.m_scale.copy_(sd["m_scale"])
            self.v_scale.copy_(sd["v_scale"])
        self.model.flat_params.copy_(sd["params"])
        self.m.copy_(sd["m"])
        self.v.copy_(sd["v"])
        if self.master is not None and sd.get("master") is not None:
            self.master.copy_(sd["master"])
        self.step_count = int(sd["step"])
        torch.set_rng_state(sd["rng_cpu"])
        if sd.get("rng_cuda") is not None and self.device.type == "cuda":
            torch.cuda.set_rng_state(sd["rng_cuda"], self.device)


class AdamW:
    """The optimizer of parameters that are tensors of their own, such as those of ``models.moe.MoELayer``: one launch for up to 400 of them,
    with the moments in 32 bits or, for less than half of the bytes, in 8.  Parameters without a gradient (experts
    that no token chose) are left as they are, and a step that they sit out does not count in their bias corrections; parameters that have taken
    part in different numbers of steps are a launch each number.  Master copies are taken here: load the weights before, or load a state saved with them
    behind it, since a step overwrites the parameters with their copies."""

    def __init__(self, params, optim: OptimConfig | None = None, *, bits: int | None = None):
        """bits: of the moments, by default the configuration's ``state_bits``."""
        self.params = list(params)
        self.optim = optim or OptimConfig()
        if bits == 32 and self.optim.state_bits == 8:
            raise ValueError("the configuration asks for moments in 8 bits, the call for 32")
        self.bits = self.optim.state_bits if bits is None else bits
        self.state = llm_ops.adamw_states(self.params, bits=self.bits, master=self.optim.master_weights)
        self.step_count = 0
        self.sat_out = [0] * len(self.params)   # steps that a parameter had no gradient in: its bias corrections are those of its own steps

    def step(self, grad_scale: float = 1.0, zero_grad: bool = True) -> None:
        """Updates the parameters from their ``grad``, which is None afterwards unless ``zero_grad`` is false: a tensor of zeros would still be a
        gradient, whose parameter decays and moves on by its old moments. While a graph is captured they are zeroed where they are: a replay reads them there."""
        oc = self.optim
        grads = [p.grad for p in self.params]
        captured = any(g is not None and g.is_cuda for g in grads) and torch.cuda.is_current_stream_capturing()
        llm_ops.adamw_step_many(self.params, grads, **self.state, lr=oc.lr, beta1=oc.beta1, beta2=oc.beta2,
                                eps=oc.eps, weight_decay=oc.weight_decay, step=[self.step_count + 1 - n for n in self.sat_out],
                                grad_scale=grad_scale, zero_grad=zero_grad and captured)
        self.step_count += 1   # a step that was refused is none
        self.sat_out = [n + (g is None) for n, g in zip(self.sat_out, grads)]
        if zero_grad and not captured:
            _lib.native().used_here(grads)
            for p in self.params:
                p.grad = None

    def state_dict(self) -> dict:
        return {"bits": self.bits, "step": self.step_count, "sat_out": list(self.sat_out), **self.state}

    def load_state_dict(self, sd: dict) -> None:
        if sd["bits"] != self.bits:
            raise ValueError(f"the moments are held in {self.bits} bits, the saved ones in {sd['bits']}")
        sat_out = list(sd.get("sat_out") or [0] * len(self.params))
        if len(sat_out) != len(self.params):
            raise ValueError("the saved steps are those of other parameters")
        for name, mine in self.state.items():
            saved = sd[name]
            if (mine is None) != (saved is None) or (mine is not None and [t is None or t.shape for t in mine] != [t is None or t.shape for t in saved]):
                raise ValueError(f"the saved {name} is that of other parameters")
        for name, mine in self.state.items():
            for to, t in zip(mine or (), sd[name] or ()):
                if to is not None:
                    to.copy_(t)
        self.step_count, self.sat_out = int(sd["step"]), sat_out
