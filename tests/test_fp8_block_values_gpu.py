"""GPU: residual RMSNorm and block-scaled e4m3 Linear on rows that hold NaN, infinities or overflow."""
import pytest
import torch

from lightx2v_amd import hip

pytestmark = pytest.mark.gpu


def _linear_of(form, r, w):
    """The quantised Linear that takes this form of the norm's output."""
    if form == "group":
        return hip.gemm_fp8_block(r.q, r.scale, *hip.quant_fp8_block128(w))
    return hip.gemm_int8(r.q, r.scale, *hip.quant_int8_rowwise(w, weight_mode=True)) if form == "int8" else hip.gemm_fp8(r.q, r.scale, *hip.quant_fp8_rowwise(w))


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [128, 1024, 1152, 5120, 8192])
@pytest.mark.parametrize("form", ["row", "group", "int8"])
def test_nan_and_infinite_rows_of_the_norm_are_nan_behind_the_linear(cuda, form, dim, stream):
    """One bad element anywhere in x, y or the norm's weight: no Linear behind the norm may return finite values for that row."""
    g = torch.Generator(device=cuda).manual_seed(dim)
    x = torch.randn(9, dim, generator=g, device=cuda).to(stream)
    y = torch.randn(9, dim, generator=g, device=cuda).to(torch.bfloat16)
    w = (torch.randn(136, dim, generator=g, device=cuda) * 0.05).to(torch.bfloat16)
    clean = hip.add_rmsnorm_(x.clone(), y, None, quant=form)
    inf, nan = float("inf"), float("nan")
    x[0, 0], x[1, dim - 1], x[2, dim // 2], y[3, 7], y[4, dim - 8] = nan, inf, -inf, nan, inf
    x[5], y[5, 3] = nan, 1.0
    x[6, 9], y[6, 9] = inf, -inf
    r = hip.add_rmsnorm_(x.clone(), y, None, quant=form)
    out, keep = _linear_of(form, r, w), [7, 8]
    assert bool(out[:7].isnan().all()), out[:7].isnan().all(dim=1).tolist()
    assert torch.equal(out[keep], _linear_of(form, clean, w)[keep]) and bool(out[keep].isfinite().all())
    assert torch.equal(r.q.view(torch.uint8)[keep], clean.q.view(torch.uint8)[keep]) and torch.equal(r.scale[keep], clean.scale[keep])
    for bad in (nan, inf):   # a bad weight of the norm reaches every row
        nw = torch.ones(dim, device=cuda)
        nw[dim - 1] = bad
        r = hip.add_rmsnorm_(x.clone(), y, nw, quant=form)
        assert not bool(_linear_of(form, r, w)[keep].isfinite().any())


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
def test_int8_row_whose_sum_of_squares_overflows_has_a_nan_scale(cuda, stream):
    x = torch.ones(4, 512, device=cuda, dtype=stream)
    x[1, 5], x[2] = 1e30, 3e38
    r = hip.add_rmsnorm_(x.clone(), None, None, quant="int8")
    assert bool(r.scale[1:3].isnan().all()) and bool(r.scale[[0, 3]].isfinite().all()) and bool((r.q[[0, 3]] == 127).all())


@pytest.mark.parametrize("seg,seg2", [(64, 8), (8, 256), (128, 128), (200, 40)])
def test_quant_of_a_source_in_two_regions(cuda, seg, seg2):
    """Column segments of two widths (a sequence-parallel result with its own remainder): groups of 128 columns astride them."""
    rows, n, n2 = 37, 4, 3
    g = torch.Generator(device=cuda).manual_seed(6)
    flat = torch.randn(rows * (n * seg + n2 * seg2) + 16, generator=g, device=cuda).to(torch.bfloat16)
    base2 = rows * n * seg
    first = flat[:base2].view(n, rows, seg)
    second = flat[base2:base2 + rows * n2 * seg2].view(n2, rows, seg2)
    plain = torch.cat([first.permute(1, 0, 2).reshape(rows, -1), second.permute(1, 0, 2).reshape(rows, -1)], dim=1).contiguous()
    ks = hip.KSeg(seg=seg, stride=rows * seg, split=n * seg, seg2=seg2, stride2=rows * seg2, base2=base2, lda2=seg2)
    q, s = hip.quant_fp8_group128(first[0], kseg=ks, dim=plain.shape[1])
    want_q, want_s = hip.quant_fp8_group128(plain)
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s, want_s)
