"""GPU: block-scaled e4m3 Linear (`gemm_fp8_block`), its quantisers and the residual RMSNorm that feeds it, against the 64-bit
formulas of oracle/fp8_block_ref.py.  Tolerances are error bounds of the arithmetic, derived there and beside each check."""
import pytest
import torch

import lightx2v_amd as L
from lightx2v_amd import hip
from oracle import fp8_block_ref as R
from oracle import wan_block_ref as BR
from tests.util import case_inputs, cos, load_golden

pytestmark = pytest.mark.gpu
EPI = {"none": hip.EPI_NONE, "gelu": hip.EPI_GELU_TANH, "residual": hip.EPI_RESIDUAL}


def _rand(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device=gen.device, dtype=torch.float32) * std


def _operands(cuda, M, N, K, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    a = _rand(g, M, K) * torch.exp(_rand(g, 1, K))
    w = _rand(g, N, K, std=0.05) * torch.exp(_rand(g, N, 1))
    (aq, a_s), (wq, w_s) = R.quantise(a, 1), R.quantise(w, 128)
    return aq, a_s.t().contiguous().t(), wq, w_s.contiguous(), g


def _within(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((got.double() - ref).abs() / tol).max()))


# one row, the skinny kernel's last size and the next, part tiles and full ones of every tile kernel, the split along K;
# one block of K, less than one, a short last one; N below a block, across its edge, a short last one
SHAPES = [(1, 8, 16), (1, 64, 128), (1, 5120, 5120), (2, 136, 112), (13, 520, 1456), (16, 256, 4096), (17, 264, 144), (33, 2056, 272), (64, 512, 2048), (65, 128, 1024),
          (200, 384, 640), (257, 5120, 1280), (512, 1536, 8960), (1000, 2056, 1456), (1111, 4096, 384), (4100, 3080, 208), (9000, 1544, 528), (193, 13824, 5120),
          # each tile kernel with one block of K and with two, one tile and several for a workgroup; split along K with a ragged last part
          (70, 136, 16), (900, 1288, 96), (12001, 136, 16), (577, 4104, 144), (20000, 520, 16), (20000, 520, 144), (12001, 1288, 16), (12001, 1288, 144), (20000, 776, 1040),
          (40, 512, 2048), (70, 136, 4112), (70, 8200, 4112), (484, 4096, 8976), (151, 8960, 13840),
          (385, 8200, 16), (385, 8200, 272), (77, 5120, 13840), (262, 4096, 13840), (151, 8960, 16400)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("epi", ["none", "gelu", "residual"])
def test_gemm_matches_64_bit(cuda, M, N, K, epi):
    aq, a_s, wq, w_s, g = _operands(cuda, M, N, K, M + N + K)
    bias = _rand(g, N, std=0.5)
    resid = _rand(g, M, N).to(torch.bfloat16) if epi == "residual" else None
    gate = _rand(g, N) if epi == "residual" else None
    ref, tol = R.linear(aq, a_s, wq, w_s, bias, epi, resid, gate)
    buf = torch.full((M + 1, N + 8), 7.0, dtype=torch.bfloat16, device=cuda)
    out = hip.gemm_fp8_block(aq, a_s, wq, w_s, bias, epilogue=EPI[epi], resid=resid, gate=gate, out=buf[:M, :N])
    assert out.data_ptr() == buf.data_ptr()
    _within(out, ref, tol)
    # the bound of a single element adds up the worst case of K products; over all elements those errors are far below the
    # rounding to bf16, at most 2^-8 of each value and uniform within its step, which alone stays below 2^-8 / sqrt(3) rms
    assert float((out.double() - ref).norm()) <= 2.0 ** -8 * float(ref.norm())
    assert bool((buf[M:] == 7).all()) and bool((buf[:, N:] == 7).all())   # nothing past the result is written
    # again, the result in the residual's place: the same bits
    again = hip.gemm_fp8_block(aq, a_s, wq, w_s, bias, epilogue=EPI[epi], resid=resid, gate=gate, out=resid)
    assert torch.equal(again, out)


def test_gemm_without_bias_or_gate_and_with_other_strides(cuda):
    M, N, K = 300, 264, 400
    aq, a_s, wq, w_s, g = _operands(cuda, M, N, K, 5)
    resid = _rand(g, M, N).to(torch.bfloat16)
    ref, tol = R.linear(aq, a_s, wq, w_s, None, "residual", resid, None)
    out = hip.gemm_fp8_block(aq, a_s, wq, w_s, epilogue=hip.EPI_RESIDUAL, resid=resid)
    _within(out, ref, tol)
    # operands as column / row ranges of wider ones, NaN codes and NaN scales all around them
    wide_a = torch.full((M + 2, K + 64), 0x7f, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    wide_a.view(torch.uint8)[1:M + 1, 16:K + 16] = aq.view(torch.uint8)
    wide_w = torch.full((N + 1, K + 32), 0x7f, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    wide_w.view(torch.uint8)[:N, :K] = wq.view(torch.uint8)
    wide_s = torch.full((5, M + 3), float("nan"), device=cuda)
    wide_s[:4, 2:M + 2] = a_s.t()
    wide_r = torch.full((M, N + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_r[:, 8:N + 8] = resid
    args = (wide_a[1:M + 1, 16:K + 16], wide_s[:4, 2:M + 2].t(), wide_w[:N, :K], w_s)
    assert torch.equal(hip.gemm_fp8_block(*args, epilogue=hip.EPI_RESIDUAL, resid=wide_r[:, 8:N + 8]), out)
    # scales row after row (copied into the kernel's order first), weight scales as a column range
    wide_ws = torch.full((w_s.shape[0], w_s.shape[1] + 3), float("nan"), device=cuda)
    wide_ws[:, 1:1 + w_s.shape[1]] = w_s
    assert torch.equal(hip.gemm_fp8_block(aq, a_s.contiguous(), wq, wide_ws[:, 1:1 + w_s.shape[1]], epilogue=hip.EPI_RESIDUAL, resid=resid), out)


@pytest.mark.parametrize("M,N,K", [(3, 64, 256), (40, 136, 400), (300, 264, 272), (5000, 3080, 144)])
def test_gemm_special_values_stay_in_their_row(cuda, M, N, K):
    """A NaN code or an infinite scale reaches its own row only; scales of zero and the smallest ones are exact."""
    aq, a_s, wq, w_s, _ = _operands(cuda, M, N, K, 9)
    clean = hip.gemm_fp8_block(aq, a_s, wq, w_s)
    aq2, a_s2 = aq.clone(), a_s.clone()
    aq2.view(torch.uint8)[0, K - 1] = 0x7f
    a_s2[1, 0] = float("inf")
    a_s2[2] = 0.0
    got = hip.gemm_fp8_block(aq2, a_s2.t().contiguous().t(), wq, w_s)
    assert bool(got[0].isnan().all()) and not bool(got[1].isfinite().any()) and bool((got[2] == 0).all())
    assert torch.equal(got[3:], clean[3:])
    zero = hip.gemm_fp8_block(torch.zeros_like(aq.view(torch.uint8)).view(torch.float8_e4m3fn), torch.full_like(a_s, 1e-12 / 448), wq, w_s, bias=torch.ones(N, device=cuda))
    assert bool((zero == 1).all())


def test_gemm_of_no_rows(cuda):
    aq, a_s, wq, w_s, _ = _operands(cuda, 4, 64, 256, 3)
    assert hip.gemm_fp8_block(aq[:0], a_s[:0], wq, w_s).shape == (0, 64)


def test_gemm_split_along_k_with_and_without_its_workspace(cuda):
    M, N, K = 40, 256, 8192
    need = hip.gemm_fp8_block_workspace_bytes(M, N, K)
    assert need > 0
    aq, a_s, wq, w_s, _ = _operands(cuda, M, N, K, 11)
    ref, tol = R.linear(aq, a_s, wq, w_s)
    own = hip.gemm_fp8_block(aq, a_s, wq, w_s)
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device=cuda)
    _within(own, ref, tol)
    for _ in range(3):
        assert torch.equal(hip.gemm_fp8_block(aq, a_s, wq, w_s, workspace=ws[:need]), own)
    assert bool((ws[need:] == 0xff).all())
    _within(hip.gemm_fp8_block(aq, a_s, wq, w_s, workspace=ws[:64]), ref, tol)   # too small: not split


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,dim", [(1, 8), (1, 128), (3, 120), (16, 512), (17, 520), (130, 1536), (33, 5120), (5, 13824), (257, 1280), (1000, 136)])
def test_quant_group_bit_exact(cuda, rows, dim, dtype):
    g = torch.Generator(device=cuda).manual_seed(rows + dim)
    x = (_rand(g, rows, dim) * torch.exp(2 * _rand(g, rows, 1))).to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, :dim // 2] = 0
    wide = torch.full((rows, dim + 24), float("nan"), dtype=dtype, device=cuda)
    wide[:, 8:8 + dim] = x
    q_ref, s_ref = R.quantise(x.cpu(), 1)
    for src in (x, wide[:, 8:8 + dim]):
        q, s = hip.quant_fp8_group128(src)
        assert s.shape == s_ref.shape and torch.equal(s.cpu(), s_ref)
        assert torch.equal(q.view(torch.uint8).cpu(), q_ref.view(torch.uint8))
    if dim == 128:   # one group a row: the row-wise quantiser's bytes
        q, s = hip.quant_fp8_rowwise(x)
        assert torch.equal(s.cpu(), s_ref[:, 0]) and torch.equal(q.view(torch.uint8).cpu(), q_ref.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,dim", [(8, 16), (64, 64), (128, 128), (136, 400), (1536, 1536), (2056, 1456)])
def test_quant_block_bit_exact(cuda, rows, dim, dtype):
    g = torch.Generator(device=cuda).manual_seed(rows)
    w = (_rand(g, rows, dim) * torch.exp(2 * _rand(g, rows, 1))).to(dtype)
    w[:, :min(dim, 128)] = 0   # blocks of zeros
    wide = torch.full((rows, dim + 8), float("nan"), dtype=dtype, device=cuda)
    wide[:, :dim] = w
    q_ref, s_ref = R.quantise(w.cpu(), 128)
    for src in (w, wide[:, :dim]):
        q, s = hip.quant_fp8_block128(src)
        assert torch.equal(s.cpu(), s_ref) and torch.equal(q.view(torch.uint8).cpu(), q_ref.view(torch.uint8))


def test_quant_of_nan_and_infinities(cuda):
    x = torch.ones(3, 256, dtype=torch.bfloat16)
    x[0, 5] = float("nan")
    x[1, 7], x[1, 200] = float("inf"), -float("inf")
    q, s = hip.quant_fp8_group128(x.to(cuda))
    q, s = q.float().cpu(), s.cpu()
    assert bool(q[0, 5].isnan()) and int(q.isnan().sum()) == 3 and bool(q[1, 7].isnan()) and bool(q[1, 200].isnan())
    assert torch.equal(s[0], torch.full((2,), 1.0 / 448)) and bool(s[1].isinf().all()) and bool((q[0, 6:] == 448).all()) and bool((q[1, :7] == 0).all())
    f = torch.full((1, 128), 3e38)   # the largest magnitudes of fp32
    q, s = hip.quant_fp8_group128(f.to(cuda))
    assert bool((q.float() == 448).all()) and torch.equal(s.cpu(), R.quantise(f, 1)[1])


def test_quant_of_a_segmented_source(cuda):
    """The receive layout of a sequence-parallel attention: column segments in separate row blocks."""
    rows, seg, n = 37, 64, 6
    g = torch.Generator(device=cuda).manual_seed(4)
    parts = _rand(g, n, rows, seg).to(torch.bfloat16)
    ks = hip.KSeg(seg=seg, stride=rows * seg, split=0, seg2=0, stride2=0, base2=0, lda2=0)
    q, s = hip.quant_fp8_group128(parts[0], kseg=ks, dim=n * seg)
    q2, s2 = hip.quant_fp8_group128(parts.permute(1, 0, 2).reshape(rows, n * seg).contiguous())
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


NORM_REL = 200 * 2.0 ** -24   # a lane adds at most 128 squares in turn and ten partial sums (half of it in the root), a few roundings besides


def _check_norm(x, y, w, eps, form):
    h, v = R.add_rmsnorm(x, y, w, eps)
    x2 = x.clone()
    r = hip.add_rmsnorm_(x2, y, w, eps=eps, quant=form)
    want = x if y is None else (x.float() + y.float()).to(x.dtype)
    assert torch.equal(x2, want)
    if form is None:
        _within(r, v, (2.0 ** -8 + 2 * NORM_REL) * v.abs())
        return r
    s = r.scale.double()
    if form == "group":
        amax, grid = R.blocks(v, 1).abs().amax(dim=(1, 3)), s.repeat_interleave(128, dim=1)[:, :x.shape[1]]
    else:
        amax, grid = v.abs().amax(dim=1), s[:, None]
    _within(r.scale, amax.clamp(min=0 if form == "int8" else 1e-12) / (127 if form == "int8" else 448), (amax + 1e-12) / 127 * 2 * NORM_REL)
    # half a step of the code (e4m3: 2^-4 of the value, or 2^-10 where the code is subnormal; int8: 1/2), in units of the scale
    step = 0.5 * grid if form == "int8" else torch.maximum(2.0 ** -4 * v.abs(), 2.0 ** -10 * grid)
    _within(r.q.double() * grid, v, step * (1 + 4 * NORM_REL) + 4 * NORM_REL * v.abs())
    return r


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", [None, "row", "group", "int8"])
@pytest.mark.parametrize("rows,dim", [(1, 8), (1, 5120), (2, 128), (5, 8192), (512, 4096), (63, 1000), (300, 2056), (2047, 264), (2048, 264), (2100, 512), (3001, 776), (2500, 1536), (2050, 2048),
                                      (2049, 2560), (4000, 4096), (2600, 5120), (2051, 6144), (2222, 8192)])
def test_add_rmsnorm(cuda, rows, dim, form, stream):
    g = torch.Generator(device=cuda).manual_seed(rows + dim)
    x = (_rand(g, rows, dim) * torch.exp(_rand(g, rows, 1))).to(stream)
    y, w = _rand(g, rows, dim).to(torch.bfloat16), 1 + 0.2 * _rand(g, dim)
    if rows > 3:
        x[1], y[1] = 0, 0            # a row of zeros
        y[2] = -x[2].to(torch.bfloat16)   # a sum that cancels (bf16: to zero)
    _check_norm(x, y, w, 1e-6, form)


@pytest.mark.parametrize("form", [None, "row", "group", "int8"])
def test_add_rmsnorm_without_y_or_weight_and_strided(cuda, form):
    g = torch.Generator(device=cuda).manual_seed(8)
    for rows, dim in ((7, 264), (2500, 264)):
        x, y = _rand(g, rows, dim).to(torch.bfloat16), _rand(g, rows, dim).to(torch.bfloat16)
        _check_norm(x, None, None, 1e-5, form)
        wide = torch.full((rows, 3 * dim), 9.0, dtype=torch.bfloat16, device=cuda)
        wide[:, :dim], wide[:, 2 * dim:] = x, y
        ref = hip.add_rmsnorm_(x.clone(), y, None, quant=form)
        got = hip.add_rmsnorm_(wide[:, :dim], wide[:, 2 * dim:], None, quant=form)
        if form is None:
            assert torch.equal(got, ref)
            got = hip.add_rmsnorm_(x.clone(), wide[:, 2 * dim:], None, out=wide[:, 2 * dim:])   # the result in y's place
            assert torch.equal(got, ref)
        else:
            assert torch.equal(got.q.view(torch.uint8), ref.q.view(torch.uint8)) and torch.equal(got.scale, ref.scale)
        assert bool((wide[:, dim:2 * dim] == 9).all())


def test_add_rmsnorm_nan_and_infinity_stay_in_their_row(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    x, y = _rand(g, 6, 512).to(torch.bfloat16), _rand(g, 6, 512).to(torch.bfloat16)
    clean = hip.add_rmsnorm_(x.clone(), y, None)
    x[1, 3], x[2, 4] = float("nan"), float("inf")
    got = hip.add_rmsnorm_(x.clone(), y, None)
    keep = [0, 3, 4, 5]
    assert torch.equal(got[keep], clean[keep]) and bool(got[1].isnan().all()) and bool(got[2, 4].isnan()) and bool((got[2, 5:] == 0).all())
    q = hip.add_rmsnorm_(x.clone(), y, None, quant="group")
    assert bool(q.q[1].float().isnan().all()) and not bool(q.q[keep].float().isnan().any())


def test_chain_of_norm_and_linears(cuda):
    """A pre-norm feed-forward part as it is used: norm -> e4m3 groups -> Linear + GELU -> e4m3 groups -> Linear + residual."""
    rows, dim, ffn = 300, 512, 1456
    g = torch.Generator(device=cuda).manual_seed(21)
    x, y, nw = _rand(g, rows, dim).to(torch.bfloat16), _rand(g, rows, dim).to(torch.bfloat16), 1 + 0.1 * _rand(g, dim)
    w1, w2 = _rand(g, ffn, dim, std=0.05), _rand(g, dim, ffn, std=0.05)
    q1, q2 = hip.quant_fp8_block128(w1), hip.quant_fp8_block128(w2.to(torch.bfloat16))
    h = hip.add_rmsnorm_(x, y, nw, quant="group")
    u = hip.gemm_fp8_block(h.q, h.scale, *q1, epilogue=hip.EPI_GELU_TANH)
    ref, tol = R.linear(h.q, h.scale, *q1, epilogue="gelu")
    _within(u, ref, tol)
    uq = hip.quant_fp8_group128(u)
    before = x.clone()
    hip.gemm_fp8_block(*uq, *q2, epilogue=hip.EPI_RESIDUAL, resid=x, out=x)
    ref, tol = R.linear(*uq, *q2, epilogue="residual", resid=before)
    _within(x, ref, tol)
    # and the whole scheme stays near the unquantised product: two roundings to e4m3 a product (at most 2^-4 of each value,
    # uniform within the step, so 2^-4 / sqrt 3 at the most rms) in quadrature over independent terms, twice in a row
    full = torch.nn.functional.gelu(R.add_rmsnorm(before, None, nw, 1e-6)[1] @ w1.double().t(), approximate="tanh") @ w2.double().t()
    got = (x.double() - before.double())
    assert float((got - full).norm() / full.norm()) <= 2 * 2 ** 0.5 * 2.0 ** -4 / 3 ** 0.5


def test_captured_and_replayed_on_another_stream(cuda):
    """norm -> quantised Linear (split along K) recorded into a graph, replayed with eager work between the replays."""
    rows, dim, n = 40, 4096, 256
    g = torch.Generator(device=cuda).manual_seed(31)
    x0, y = _rand(g, rows, dim).to(torch.bfloat16), _rand(g, rows, dim).to(torch.bfloat16)
    wq = hip.quant_fp8_block128(_rand(g, n, dim, std=0.05))
    x = x0.clone()

    def chain():
        h = hip.add_rmsnorm_(x, y, None, quant="group")
        return hip.gemm_fp8_block(h.q, h.scale, *wq), h.q, h.scale

    assert hip.gemm_fp8_block_workspace_bytes(rows, n, dim) > 0
    refs = []
    for _ in range(4):
        refs.append([t.clone() for t in chain()] + [x.clone()])
    x.copy_(x0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = chain()
    torch.cuda.synchronize()
    x.copy_(x0)
    other = torch.empty(1 << 20, device=cuda)
    for want in refs:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(list(out) + [x], want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        other.normal_()                       # eager work of the program between the replays
        hip.add_rmsnorm_(other.view(1024, 1024), None, None)
        torch.cuda.synchronize()


def test_two_streams_at_once(cuda):
    """Two products that are split along K, on two streams at the same time: each has its own workspace."""
    sets = [_operands(cuda, 40, 512, 8192, s)[:4] for s in (1, 2)]
    want = [hip.gemm_fp8_block(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(hip.gemm_fp8_block(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_past_32_bit_offsets(cuda):
    """Operands of more than 2^31 (and results of more than 2^32) bytes: the last rows are as right as the first."""
    rows, dim, n = 320000, 8192, 136
    g = torch.Generator(device=cuda).manual_seed(41)
    x = torch.empty((rows, dim), dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    y = torch.empty_like(x).normal_(generator=g)
    w = 1 + 0.1 * _rand(g, dim)
    wq, w_s = hip.quant_fp8_block128(_rand(g, n, dim, std=0.05))
    pick = torch.tensor([0, 1, 131071, 131072, 262143, 262144, rows - 2, rows - 1], device=cuda)
    q, s = hip.quant_fp8_group128(x)
    ref_q, ref_s = (t.to(cuda) for t in R.quantise(x[pick].cpu(), 1))   # on the CPU: torch's GPU quotient of a tensor and a number is not the rounded one
    assert torch.equal(q[pick].view(torch.uint8), ref_q.view(torch.uint8)) and torch.equal(s[pick], ref_s)
    ref, tol = R.linear(ref_q, ref_s, wq, w_s)
    _within(hip.gemm_fp8_block(q, s, wq, w_s)[pick], ref, tol)
    wide = q[:260000].view(-1, 2 * dim)[:, :dim]      # rows 16 KiB apart
    ref, tol = R.linear(wide[-3:].contiguous(), s[:260000:2][-3:], wq, w_s)
    _within(hip.gemm_fp8_block(wide, s[:260000:2], wq, w_s)[-3:], ref, tol)
    del q, s, wide
    x0, y0 = x[pick], y[pick]
    h = hip.add_rmsnorm_(x, y, w, quant="group")
    small = hip.add_rmsnorm_(x0, y0, w, quant="group")
    assert torch.equal(x[pick], x0) and torch.equal(h.q[pick].view(torch.uint8), small.q.view(torch.uint8)) and torch.equal(h.scale[pick], small.scale)


# ---- the plugin and the blocks that run on it ----
def _plugin(name, w, b=None, **extra):
    mm = L.MM_WEIGHT_REGISTER[name]("w.weight", None if b is None else "w.bias")
    mm.load({"w.weight": w, **({} if b is None else {"w.bias": b}), **extra})
    return mm


def test_plugin_loads_quantises_and_applies(cuda):
    M, N, K = 77, 328, 400
    g = torch.Generator(device=cuda).manual_seed(51)
    x, w, b = _rand(g, M, K).to(torch.bfloat16), _rand(g, N, K, std=0.05), _rand(g, N, std=0.3)
    resid, gate = _rand(g, M, N).to(torch.bfloat16), _rand(g, N)
    mm = _plugin("hip-fp8-block128", w, b)
    wq, w_s = (t.to(cuda) for t in R.quantise(w.cpu(), 128))
    assert torch.equal(mm.weight_nk.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(mm.weight_scale, w_s)
    aq, a_s = (t.to(cuda) for t in R.quantise(x.cpu(), 1))
    for epi, run in (("none", lambda: mm.apply(x)), ("gelu", lambda: mm.apply_gelu(x)), ("residual", lambda: mm.apply_residual_(x, resid.clone(), gate))):
        _within(run(), *R.linear(aq, a_s, wq, w_s, b, epi, resid, gate))
    out = torch.empty((M, 2 * N), dtype=torch.bfloat16, device=cuda)[:, N:]
    assert mm.apply(x, out=out) is out and torch.equal(out, mm.apply(hip.QuantGroups(*hip.quant_fp8_group128(x))))
    for name in ("w.weight_scale", "w.weight_scale_inv"):     # a pre-quantised checkpoint loads as it is
        pre = _plugin("hip-fp8-block128", wq.cpu(), b.cpu(), **{name: w_s.cpu()})
        pre.to_cuda()
        assert torch.equal(pre.apply(x), out)
    assert sorted(pre.state_dict()) == ["w.bias", "w.weight", "w.weight_scale"]
    # a residual stream in fp32 and a gate per row: the product in bf16, the gated sum as its own pass
    r32 = resid.float()
    assert mm.apply_residual_(x, r32, gate) is r32
    _within(r32, resid.double() + out.double() * gate.double(), 2.0 ** -22 * (resid.double().abs() + (out.double() * gate).abs()))
    with pytest.raises(hip.Lx2vError):
        mm.apply(hip.QuantRows(*hip.quant_fp8_rowwise(x)))


def test_plugin_fused_members_and_segmented_source(cuda):
    g = torch.Generator(device=cuda).manual_seed(52)
    rows, dim = 37, 384
    x = _rand(g, rows, dim).to(torch.bfloat16)
    sizes = (256, 128, 72)
    mods = [_plugin("hip-fp8-block128", _rand(g, n, dim, std=0.05), _rand(g, n) if i != 1 else None) for i, n in enumerate(sizes)]
    alone = [m.apply(x) for m in mods]
    fused = type(mods[0]).fused(mods)
    got = fused.apply(x)
    slices = [got[:, :256], got[:, 256:384], got[:, 384:]]
    aq, a_s = hip.quant_fp8_group128(x)
    for m, a, b in zip(mods, alone, slices):
        assert m.weight_nk.untyped_storage().data_ptr() == fused.weight_nk.untyped_storage().data_ptr()
        assert torch.equal(m.apply(x), a)
        _within(b, *R.linear(aq, a_s, m.weight_nk, m.weight_scale, m.bias))
    with pytest.raises(ValueError):
        type(mods[0]).fused([mods[2], mods[0]])
    parts = x.view(rows, 6, 64).permute(1, 0, 2).contiguous()
    ks = hip.KSeg(seg=64, stride=rows * 64, split=0, seg2=0, stride2=0, base2=0, lda2=0)
    a, b = (torch.ones(rows, 256, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    mods[0].apply_residual_(x, a, None)
    mods[0].apply_residual_(parts[0], b, None, kseg=ks)
    assert torch.equal(a, b)


@pytest.mark.parametrize("scheme,form", [("hip-fp8-block128", "group"), ("hip-fp8", "row"), ("hip-int8", "int8"), ("hip-bf16", None)])
def test_residual_norm_plugin_writes_the_form_its_consumers_take(cuda, scheme, form):
    """x += y, norm, feed-forward, all through the plugins: the norm hands over the 8-bit rows and the Linear takes them as they are."""
    rows, dim, ffn = 130, 512, 1024
    g = torch.Generator(device=cuda).manual_seed(53)
    x, y = _rand(g, rows, dim).to(torch.bfloat16), _rand(g, rows, dim).to(torch.bfloat16)
    rms = L.RMS_WEIGHT_REGISTER["hip"]("n.weight")
    rms.load({"n.weight": 1 + 0.1 * _rand(g, dim)})
    up, down = _plugin(scheme, _rand(g, ffn, dim, std=0.05)), _plugin(scheme, _rand(g, dim, ffn, std=0.05))
    x2 = x.clone()
    h = rms.apply_residual_(x2, y, quant_for=up)
    want = _check_norm(x, y, rms.weight, rms.eps, form)
    assert type(h) is type(want) and torch.equal(x2, (x.float() + y.float()).to(torch.bfloat16))
    mid = up.apply_gelu(h)
    assert torch.equal(mid, up.apply_gelu(want))
    if form is not None:
        own = up.apply_gelu(rms.apply_residual_(x.clone(), y))   # quantised by the Linear instead, after a rounding to bf16
        assert float((own.float() - mid.float()).norm()) <= 2 * 2.0 ** -4 * float(own.float().norm())
        assert isinstance(rms.apply_residual_(x.clone(), y, quant_for=[up, _plugin("hip-bf16", _rand(g, 8, dim))]), torch.Tensor)   # consumers that differ: bf16
    down.apply_residual_(mid, x2)
    assert bool(torch.isfinite(x2.float()).all())


@pytest.mark.parametrize("fused", [False, True])
def test_wan_block_with_block_scaled_linears(cuda, fused):
    """The whole block with every Linear block-scaled (both runners) against the fp32 oracle, at the gates of the row-scaled form."""
    c = case_inputs(load_golden("wan1p3b_g3x6x8"))
    cfg = {"num_layers": 1, "num_heads": c["heads"], "dim": c["dim"], "task": "t2v", "dit_quant_scheme": "hip-fp8-block128", "fused_block": fused}
    W = L.WanTransformerWeights(cfg)
    W.load({k: v.to(cuda) for k, v in {**c["w"], **c["hw"]}.items()})
    W.to_cuda()
    inf = L.WanTransformerInfer(cfg)
    inf.cos_sin = BR.cos_sin_to_real(c["cos_sin"]).contiguous().to(cuda)
    pre = L.WanPreInferModuleOutput(embed=c["embed"].to(cuda), grid_sizes=c["grid"], x=c["x"].to(torch.bfloat16).to(cuda), embed0=c["embed0"].to(cuda),
                                    context=c["context"].to(torch.bfloat16).to(cuda))
    inf.get_scheduler_values = lambda: None
    out = inf.infer_main_blocks(W.blocks, pre)
    ref = BR.block_forward(c["x"], c["embed0"], c["context"], c["w"], c["cos_sin"], c["heads"])
    c_out, c_delta = cos(out, ref), cos(out.float().cpu() - c["x"], ref - c["x"])
    print(f"\nblock-scaled fp8 block: output cosine {c_out:.6f}, delta cosine {c_delta:.6f}")
    assert c_out >= 0.999 and c_delta >= 0.99


def test_hunyuan_double_block_with_block_scaled_linears(cuda):
    from tests.test_hy_gpu import HY_CASES, _build, _io
    from tests.test_hy_oracle import hy_case_inputs

    for name in HY_CASES:
        rec = load_golden(name)
        c = hy_case_inputs(rec)
        W, inf = _build(c, cuda, dit_quant_scheme="hip-fp8-block128")
        img, txt = inf.infer_double_block(W.double_blocks[0], _io(c, cuda))
        for got, key, x0 in ((img, "img_out", c["img"]), (txt, "txt_out", c["txt"])):
            ref = torch.from_numpy(rec[key])
            assert cos(got[0], ref) >= 0.999 and cos(got[0].float().cpu() - x0[0], ref - x0[0]) >= 0.99, (name, key)


@pytest.mark.parametrize("M,N,K", [(3, 64, 256), (300, 264, 272), (40, 512, 2048)])   # skinny, tile, split along K
def test_gelu_of_huge_and_infinite_values(cuda, M, N, K):
    zero = torch.zeros(M, K, device=cuda).to(torch.float8_e4m3fn)
    a_s = torch.ones((K + 127) // 128, M, device=cuda).t()
    w = torch.zeros(N, K, device=cuda).to(torch.float8_e4m3fn)
    w_s = torch.ones((N + 127) // 128, (K + 127) // 128, device=cuda)
    bias = torch.zeros(N, device=cuda)
    bias[:8] = torch.tensor([-1e30, 1e30, -25.0, 25.0, 0.0, float("inf"), float("nan"), -3e-39])
    out = hip.gemm_fp8_block(zero, a_s, w, w_s, bias, epilogue=hip.EPI_GELU_TANH).float()
    big = torch.tensor(1e30).to(torch.bfloat16).float().item()
    for col, want in enumerate((0.0, big, 0.0, 25.0, 0.0, float("inf"))):
        assert bool((out[:, col] == want).all()), (col, out[0, col])
    assert bool(out[:, 6].isnan().all()) and bool((out[:, 7].abs() <= 3e-39).all()) and bool((out[:, 8:] == 0).all())
