"""Training on long sequences beside the operators' values: sizes that layers with 8 bits refuse, and what the model and the trainer make of their options."""
import pytest
import torch

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _refused(fn, *args, error=(AssertionError, RuntimeError, ValueError), **kw):
    with pytest.raises(error):
        fn(*args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [(1 << 29) + 8, (1 << 31) + 64, (1 << 32) + 64])
def test_rows_that_are_too_long_are_refused(width):
    """Also those whose number has the low 32 bits of a short row's; no row is there, so that none needs memory."""
    from aws_ofi_nccl_b200.ops import gemm, llm

    rows = lambda n, t=BF: torch.empty(0, n, device="cuda", dtype=t)   # noqa: E731
    x = rows(width)
    _refused(llm.keep_rows8, x)
    _refused(llm.kept_rows8, rows(width, F8), rows((width + 31) // 32, torch.uint8))
    for grad in (False, True):
        _refused(llm.swiglu, rows(2 * width).requires_grad_(grad), keep_bits=8)
        _refused(gemm.linear, rows(width).requires_grad_(grad), rows(width), keep_bits=8)
        _refused(llm.swiglu_mlp, rows(width).requires_grad_(grad), rows(width), rows(64), keep_bits=8)
        _refused(llm.swiglu_mlp, rows(64).requires_grad_(grad), rows(64), rows(width), keep_bits=8)


def test_a_configuration_with_heads_that_a_window_cannot_have():
    from aws_ofi_nccl_b200.models.llama import LlamaConfig

    narrow = dict(hidden=256, n_heads=8, n_kv_heads=2)    # heads of 32
    odd = dict(hidden=448, n_heads=7, n_kv_heads=2)       # seven heads of q on two of k and v
    for kw in (narrow, odd, dict(hidden=200, n_heads=3, n_kv_heads=1)):
        LlamaConfig(**kw)
        _refused(LlamaConfig, **kw, window=64, error=ValueError)
        _refused(LlamaConfig, **kw, window=64, sinks=2, error=ValueError)
    for kw in (dict(), dict(hidden=256, n_heads=4, n_kv_heads=2), dict(hidden=384, n_heads=3, n_kv_heads=3)):
        assert LlamaConfig(**kw, window=64).head_dim in (64, 128)


def _config(**kw):
    from aws_ofi_nccl_b200.models.llama import LlamaConfig

    return LlamaConfig(**dict(dict(vocab_size=1024, hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn=512, max_seq=128), **kw))


@pytest.mark.gpu
def test_launches_of_a_step_are_those_that_the_counter_saw():
    """Per layer beside a model without: three kernels of a window's backward pass and one forward, a fourth where its sinks are seen from far away; three each way
    of activations in 8 bits."""
    from aws_ofi_nccl_b200.ops import _lib
    from aws_ofi_nccl_b200.parallel.engine import Trainer

    def launches(seq, **kw):
        trainer = Trainer(_config(max_seq=seq, **kw))
        assert trainer.launches_per_step() == 0
        for _ in range(2):
            ids, labels = (torch.randint(0, 1024, (2, seq)).pin_memory() for _ in range(2))
            before = _lib.launch_count
            trainer.step(ids, labels)
            assert trainer.launches_per_step() == _lib.launch_count - before
        return trainer.launches_per_step()

    plain = launches(128)
    assert launches(1024) == plain
    assert launches(128, window=64, sinks=2) == launches(1024, window=64) == plain + 4 * 2
    assert launches(1024, window=64, sinks=2) == plain + 5 * 2
    assert launches(128, keep_bits=8) == plain + 6 * 2
    assert launches(1024, window=64, sinks=2, keep_bits=8) == plain + 11 * 2


def _asked():
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 64])
def test_a_model_with_8_bits_holds_less_between_its_passes(window):
    """A layer's fused projection keeps 33/32 bytes of an element of its input instead of two, its MLP 33/32 (hidden + 2 F) a token instead of
    2 hidden + 6 F. Nothing else holds these tensors."""
    import aws_ofi_nccl_b200.models.llama as L

    ids, labels = (torch.randint(0, 1024, (4, 512), device="cuda") for _ in range(2))
    tokens, held = ids.numel(), {}
    for bits in (16, 8):
        cfg = _config(max_seq=512, window=window, keep_bits=bits)
        model = L.Llama(cfg, seed=1)
        model.forward_loss(ids, labels).backward()
        before = _asked()
        loss = model.forward_loss(ids, labels)
        held[bits] = _asked() - before
        loss.backward()
        del loss, model
    h, f = cfg.hidden, cfg.ffn
    less = cfg.n_layers * tokens * ((2 * h - h * 33 / 32) + (2 * h + 6 * f - (h + 2 * f) * 33 / 32))
    assert abs(held[16] - held[8] - less) <= 8192


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_a_layer_holds_what_it_keeps(bits):
    """Of its input, beside the output: bytes asked for that live on when the program lets go of it."""
    from aws_ofi_nccl_b200.ops import gemm, llm

    t, n = 2048, 512
    w = torch.randn(256, n, device="cuda").to(BF).requires_grad_(True)
    for call, out_bytes in ((lambda x: gemm.linear(x, w, keep_bits=bits), t * 256 * 2), (lambda x: llm.swiglu(x, keep_bits=bits), t * n)):
        call(torch.ones(t, n, device="cuda", dtype=BF).requires_grad_(True).clone())
        x = torch.randn(t, n, device="cuda").to(BF)
        source = x.requires_grad_(True) * 1   # not a leaf, which its graph would hold
        before = _asked()
        y = call(source)
        del source
        kept = _asked() - before + t * n * 2 - out_bytes
        assert abs(kept - t * n * (2 if bits == 16 else 33 / 32)) <= 4096, kept
        del y
