"""RMSNorm with its output in 8 bits, against 64 bits: codes within half a step of e4m3, scales within the rounding of a sum in 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F = 2.0 ** -24   # half a step of fp32, relative


def _check(x, w, res, group, eps=1e-5):
    from aws_ofi_nccl_b200.ops import llm

    q, scale, h = llm.rmsnorm_fp8(x, w, eps, residual=res, group=group)
    H = x.shape[-1]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and q.is_contiguous()
    assert scale.dtype == torch.float32 and scale.shape == (x.shape[:-1] + (H // group,) if group else x.shape[:-1])
    if res is None:
        assert h is x
    else:
        assert torch.equal(h, (x.float() + res.float()).bfloat16()) and h.is_contiguous()
    v = h.double().reshape(-1, H)
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()
    b = y.view(len(y), -1, group or H)
    want = b.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 448
    s = scale.double().view(want.shape)
    # the sum's H roundings halve in the root; the root's, the two products', the factor 1 / 448 and the product with it
    rel = (H / 2 + 8) * F
    assert ((s - want).abs() <= rel * want).all()
    # half a step: 2^-4 of a normal number, 2^-10 of a scale below; the codes were made from products in 32 bits
    got = q.double().view(b.shape) * s
    assert ((got - b).abs() <= (2.0 ** -4 + 2 * rel) * b.abs() + (2.0 ** -10 + 448 * 2 * rel) * s).all()
    return q, scale


# every layout of a row, full, ragged and of one vector; one row, a CTA's rows and one more
@pytest.mark.parametrize("T,H", [(1, 8), (9, 256), (7, 264), (8, 512), (17, 520), (5, 1024), (6, 1032), (300, 2048), (3, 2056), (299, 4096), (4, 4104),
                                 (301, 8192), (2, 8200), (3, 16384), (1, 4096), (11, 768), (5, 776), (9, 1536), (6, 1544), (3, 5120), (4, 5128),
                                 (5, 6144), (2, 6152), (4, 7168), (3, 7176)])
@pytest.mark.parametrize("with_res", [False, True])
def test_row_scales(T, H, with_res):
    g = torch.Generator(device="cuda").manual_seed(T + H)
    x, r = (torch.randn(T, H, device="cuda", generator=g).bfloat16() for _ in range(2))
    _check(x, (1 + 0.3 * torch.randn(H, device="cuda", generator=g)).bfloat16(), r if with_res else None, 0)


@pytest.mark.parametrize("T,H", [(1, 128), (9, 256), (7, 384), (17, 640), (300, 2048), (33, 7168), (5, 8192), (3, 16384), (11, 1152), (5, 768), (3, 896), (5, 1536), (4, 1664), (3, 5120), (2, 5248), (3, 6144), (4, 6272), (2, 7296)])
@pytest.mark.parametrize("with_res", [False, True])
def test_group_scales(T, H, with_res):
    g = torch.Generator(device="cuda").manual_seed(T + H)
    x, r = (torch.randn(T, H, device="cuda", generator=g).bfloat16() for _ in range(2))
    x *= torch.logspace(-3, 2, H, device="cuda").bfloat16()   # groups of very different size
    _check(x, (1 + 0.3 * torch.randn(H, device="cuda", generator=g)).bfloat16(), r if with_res else None, 128)


def test_shapes_strides_and_alignments():
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (1 + 0.1 * torch.randn(256, device="cuda", generator=g)).bfloat16()
    x = torch.randn(2, 5, 256, device="cuda", generator=g).bfloat16()
    _check(x, w, torch.randn(2, 5, 256, device="cuda", generator=g).bfloat16(), 0)
    _check(x, w, None, 128)
    _check(x[0, 0], w, None, 0)
    wide = torch.randn(40, 1000, device="cuda", generator=g).bfloat16()
    for at in (0, 8, 3, 700):   # rows of a wider matrix, on and off a 16-byte boundary
        _check(wide[:, at:at + 256], w, wide[:, 400:656], 0)
        _check(wide[:, at:at + 256], w, None, 128)
    odd = torch.randn(40, 999, device="cuda", generator=g).bfloat16()
    _check(odd[:, 1:257], w, odd[:, :256], 0)
    _check(torch.randn(256, 30, device="cuda", generator=g).bfloat16().t(), w, None, 0)
    _check(wide[:1].expand(6, 1000)[:, :256], w, None, 0)
    _check(x.transpose(0, 1), w, x.transpose(0, 1), 128)
    off = torch.empty(257, device="cuda", dtype=torch.bfloat16)
    off[1:] = w
    _check(x, off[1:], None, 0)


def test_no_rows():
    from aws_ofi_nccl_b200.ops import llm

    x, w = torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    q, s, h = llm.rmsnorm_fp8(x, w, residual=x, group=128)
    assert q.shape == (0, 256) and s.shape == (0, 2) and h.shape == (0, 256)


@pytest.mark.parametrize("group", [0, 128])
def test_zeros_and_what_is_not_finite(group):
    """A row of zeros has the least scale; a row that holds a NaN or an infinity has NaN as every scale that the row's norm enters; others are untouched."""
    from aws_ofi_nccl_b200.ops import llm

    x = torch.randn(6, 512, device="cuda").bfloat16()
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    clean, clean_scale, _ = llm.rmsnorm_fp8(x, w, group=group)
    bad = x.clone()
    bad[1] = 0
    bad[2, 77] = float("nan")
    bad[3, 500] = float("inf")
    bad[4, 3] = -float("inf")
    q, scale, _ = llm.rmsnorm_fp8(bad, w, group=group)
    assert (q[1].float() == 0).all() and torch.allclose(scale[1], torch.full_like(scale[1], 1e-12 / 448), rtol=1e-6, atol=0)
    for row in (0, 5):
        assert torch.equal(q[row].view(torch.uint8), clean[row].view(torch.uint8)) and torch.equal(scale[row], clean_scale[row])
    assert scale[2].isnan().all()   # the sum of squares is a NaN
    assert scale[3].isnan().any() and scale[4].isnan().any()   # an infinity times a root of zero
    w[9] = float("nan")
    q, scale, _ = llm.rmsnorm_fp8(x, w, group=group)
    assert scale.view(6, -1)[:, 0].isnan().all()


def test_extreme_magnitudes():
    """Sums of squares up to the range of 32 bits, weights of both ends, values that a row's largest leaves below e4m3"""
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.ones(1024, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(4, 1024, device="cuda", generator=g)
    for std in (1e-20, 1e-6, 1e6, 1e16):
        _check((x * std).bfloat16(), w, None, 0, eps=0.0 if std > 1 else 1e-5)
    x[:, 5] = 1e4
    _check(x.bfloat16(), w, None, 0)
    _check(x.bfloat16(), (w * 1e-30), None, 128)


def test_feeds_the_fp8_product():
    """Norm and product against the same in 64 bits of the codes' values: what the product adds is its own rounding."""
    from aws_ofi_nccl_b200.ops import gemm, llm

    g = torch.Generator(device="cuda").manual_seed(6)
    x, r = (torch.randn(300, 512, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.randn(512, device="cuda", generator=g)).bfloat16()
    wq, ws = gemm.quantize_rows_fp8((torch.randn(256, 512, device="cuda", generator=g) / 20).bfloat16())
    q, s, _ = llm.rmsnorm_fp8(x, w, residual=r)
    a, b = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    want, mag = a @ b.t(), a.abs() @ b.abs().t()
    got = gemm.gemm_fp8(q, wq, s, ws).double()
    # fp8 products add up exactly to within 32 bits' rounding; e4m3 operands keep 14 bits at the least in the tensor core's sums
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * mag).all()


def test_captured_and_replayed():
    from aws_ofi_nccl_b200.ops import llm

    x, w = torch.randn(64, 1024, device="cuda").bfloat16(), torch.ones(1024, device="cuda", dtype=torch.bfloat16)
    llm.rmsnorm_fp8(x, w, residual=x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s, h = llm.rmsnorm_fp8(x, w, residual=x)
    x.normal_()
    graph.replay()
    for got, want in zip((q, s, h), llm.rmsnorm_fp8(x, w, residual=x)):
        assert torch.equal(got.float(), want.float())
