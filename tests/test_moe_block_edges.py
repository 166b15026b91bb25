"""What the operators of a mixture-of-experts block say and do at their edges: derivatives that they do not have, experts that sit steps out, and
moments in 8 bits beyond their first step."""
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


def test_a_refused_step_counts_for_nothing(built):
    from aws_ofi_nccl_b200.parallel.engine import AdamW

    p = torch.zeros(64)
    p.grad = torch.ones(64)
    opt = AdamW([p])
    for _ in range(2):
        with pytest.raises(AssertionError):   # not on a GPU
            opt.step()
    assert opt.step_count == 0 and (p.grad == 1).all()
