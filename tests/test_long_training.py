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
