"""Block-scaled e4m3 Linear on operands whose sums are exact (oracle/fp8_block_ref.py: whole_operands): a correct product equals the 64-bit
one rounded to bf16 bit for bit, and one lost column of K or one sum held in too few bits does not.  That these operands show such
mistakes is checked on the CPU, with the mistakes made in the oracle."""
import concurrent.futures

import pytest
import torch

from lightx2v_amd import hip
from oracle import fp8_block_ref as R

EPI = {"none": hip.EPI_NONE, "gelu": hip.EPI_GELU_TANH, "residual": hip.EPI_RESIDUAL}


def _whole(M, N, K, seed, device="cpu"):
    q = R.whole_operands(M, N, K, seed, device)
    return q, R.dequantise(q[0], q[1], 1), R.dequantise(q[2], q[3], 128)


@pytest.mark.parametrize("K", [144, 1280, 1456, 8960, 13840, 16400])
def test_whole_operands_show_mistakes(K):
    M, N = 5, 384
    (aq, a_s, wq, w_s), a, w = _whole(M, N, K, K)
    assert bool((a.abs() * 1.0 == a.abs().round()).all()) and set(a.abs().unique().tolist()) == {1.0, 2.0, 3.0} == set(w.unique().tolist())
    v = a @ w.t()
    want = v.to(torch.bfloat16)
    assert float((v.abs() <= 256).double().mean()) >= 0.9        # sqrt(K) is at most 128: two standard deviations
    lines = lambda u: (u != want).sum(dim=1)   # how many results of each row differ
    last = (K - 1) // 16 * 16
    for k in (0, 15, 16, 127, 128, K // 2, last - 1, last, K - 1):   # any one column of K missing: seen in nearly every result
        assert bool((lines((v - a[:, k:k + 1] * w[:, k]).to(torch.bfloat16)) >= 0.8 * N).all()), k
    for k in range(0, K, 16):    # any 16 bytes of one row missing (those astride K / 2 hold both signs and may add up to nothing)
        differ = int(((v[1] - a[1, k:k + 16] @ w[:, k:k + 16].t()).to(torch.bfloat16) != want[1]).sum())
        assert differ == N or (k < K // 2 < k + 16 and differ >= N // 2), (k, differ)
    for b in range(a_s.shape[1] - 1):   # a block taken with its neighbour's scale of the activation, of the weight
        cols = slice(128 * b, 128 * b + 128)
        part = a[:, cols] @ w[:, cols].t()
        other = a_s[:, b + 1:b + 2].double() / a_s[:, b:b + 1].double()
        bad = (v + part * (other - 1)).to(torch.bfloat16)
        assert bool((lines(bad)[other[:, 0] != 1] == N).all())
    if K >= 1280:    # sums that pass through too few bits: halves joined in bf16, the running sum in fp16, in bf16
        halves = [(a[:, s] @ w[:, s].t()).to(torch.bfloat16).double() for s in (slice(0, K // 2), slice(K // 2, K))]
        assert bool((lines((halves[0] + halves[1]).to(torch.bfloat16)) >= N // 8).all())
        for t in (torch.float16, torch.bfloat16):
            acc = torch.zeros_like(v)
            for b in range(0, K, 128):
                acc = (acc + a[:, b:b + 128] @ w[:, b:b + 128].t()).to(t).double()
            assert bool((lines(acc.to(torch.bfloat16)) >= N // 8).all()), t


# both kernels of up to 32 rows, and each tile of the stream kernel: one block of K and less, two, many, a short last one; one tile and
# several for a workgroup; whole and split along K into two to thirteen parts
SHAPES = [(1, 136, 16), (1, 520, 16400), (2, 264, 1040), (13, 520, 13840), (16, 264, 1456), (17, 264, 1040), (32, 520, 16400),          # up to 32 rows
          (33, 264, 144), (70, 136, 16), (200, 1288, 272), (600, 1288, 400), (900, 1288, 96), (385, 8200, 272), (70, 8200, 4112),           # 64 x 128
          (40, 520, 4112), (40, 520, 8208), (300, 520, 13840), (484, 4096, 8976), (151, 8960, 13840),                                       # 64 x 128 in 11, 13, 10 parts, whole
          (577, 4104, 144), (1000, 2056, 1456), (600, 6152, 2064), (2500, 1536, 8960), (133, 4096, 8208), (512, 2560, 16400),               # 128 x 128, in 4 and 3 parts
          (20000, 520, 144), (1500, 4104, 656), (1153, 5128, 1296), (1153, 5128, 4112), (71, 8200, 16400), (262, 4096, 13840),              # 128 x 256, in 7 and 5 parts
          (12001, 1288, 144), (20000, 776, 1040), (133, 8200, 13840), (2179, 1032, 13840)]                                                  # 192 x 256, in 7 and 4 parts


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_whole_products_are_exact(cuda, M, N, K):
    (aq, a_s, wq, w_s), a, w = _whole(M, N, K, M + N + K, cuda)
    v = a @ w.t().contiguous()
    got = hip.gemm_fp8_block(aq, a_s, wq, w_s)
    assert torch.equal(got, v.to(torch.bfloat16)), (got.double() != v.to(torch.bfloat16).double()).nonzero()[:4].tolist()
    # whole biases and residuals, gates that are powers of two: exact in fp32 as well
    g = torch.Generator(device=cuda).manual_seed(1)
    bias = torch.randint(-8, 9, (N,), generator=g, device=cuda).float()
    gate = torch.exp2(torch.randint(-1, 2, (N,), generator=g, device=cuda).float())
    resid = torch.randint(-8, 9, (M, N), generator=g, device=cuda).to(torch.bfloat16)
    got = hip.gemm_fp8_block(aq, a_s, wq, w_s, bias, epilogue=hip.EPI_RESIDUAL, resid=resid, gate=gate)
    assert torch.equal(got, ((v + bias.double()) * gate.double() + resid.double()).to(torch.bfloat16))
    if hip.gemm_fp8_block_workspace_bytes(M, N, K):    # the same product whole, where the plan splits it
        small = torch.empty(16, dtype=torch.uint8, device=cuda)
        assert torch.equal(hip.gemm_fp8_block(aq, a_s, wq, w_s, workspace=small), v.to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("epi", ["none", "gelu", "residual"])
@pytest.mark.parametrize("M,N,K", [(s[0], max(s[1], 1024), s[2]) for s in SHAPES])
def test_error_is_that_of_the_rounding_in_every_row(cuda, M, N, K, epi):
    """Rounding to bf16 moves a value v by at most 2^-8 |v|, uniformly within its step: a step is at most 2^-7 |v| and the mean square of
    the error a twelfth of its square, so the rms error is below 2^-8 / sqrt(3) of the rms value, for all results and, over 1024
    and more, for each row (their mean square strays from its expectation by 0.9 sqrt(3 / 1024) = 5 % for normal values, and the bound is twice the
    expectation: steps are 2^-8 to 2^-7 of the value).  What the product itself loses, 2^-13 of some terms and fp32 sums, is far below."""
    g = torch.Generator(device=cuda).manual_seed(M + N + K)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda)
    (aq, a_s), (wq, w_s) = R.quantise(rand(M, K), 1), R.quantise(rand(N, K) / K ** 0.5, 128)
    bias = rand(N) * 0.1
    resid, gate = (rand(M, N).to(torch.bfloat16), 1 + 0.1 * rand(N)) if epi == "residual" else (None, None)
    got = hip.gemm_fp8_block(aq, a_s.t().contiguous().t(), wq, w_s.contiguous(), bias, epilogue=EPI[epi], resid=resid, gate=gate)
    v = R.dequantise(aq, a_s, 1) @ R.dequantise(wq, w_s, 128).t().contiguous() + bias.double()
    if epi == "gelu":
        v = v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    elif epi == "residual":
        v = v * gate.double() + resid.double()
    err = got.double() - v
    bound = 2.0 ** -8 / 3 ** 0.5
    assert float(err.norm() / v.norm()) <= bound
    rows = err.norm(dim=1) / v.norm(dim=1)
    assert bool((rows <= bound).all()), (int(rows.argmax()), float(rows.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(300, 520, 13840), (512, 2560, 16400), (262, 4096, 13840), (2179, 1032, 13840), (900, 1288, 96), (13, 520, 272)])
def test_largest_row_strides(cuda, M, N, K):
    """Rows as far apart as the entry point takes them: the offsets inside a tile come near 2^30 (operands) and 2^31 bytes (results)."""
    (aq, a_s, wq, w_s), a, w = _whole(M, N, K, 7, cuda)
    far = lambda rows, ld, dtype: torch.empty_strided((rows, ld), (ld, 1), dtype=dtype, device=cuda)
    wide_a, wide_w = (far(r, (1 << 22) - 16, torch.uint8)[:, -K:] for r in (M, N))
    wide_a.copy_(aq.view(torch.uint8))
    wide_w.copy_(wq.view(torch.uint8))
    out, resid = (far(M, (1 << 22) - 8, torch.bfloat16)[:, -N:] for _ in range(2))
    resid.fill_(3.0)
    v = a @ w.t().contiguous()
    for ws in (None, torch.empty(16, dtype=torch.uint8, device=cuda)):    # split along K where the plan says so, and whole
        args = (wide_a.view(torch.float8_e4m3fn), a_s, wide_w.view(torch.float8_e4m3fn), w_s)
        out.fill_(float("nan"))
        assert torch.equal(hip.gemm_fp8_block(*args, out=out, workspace=ws), v.to(torch.bfloat16))
        hip.gemm_fp8_block(*args, epilogue=hip.EPI_RESIDUAL, resid=resid, out=out, workspace=ws)
        assert torch.equal(out, (v + 3).to(torch.bfloat16))


@pytest.mark.gpu
def test_products_from_several_threads_at_once(cuda):
    """Calls of different shapes from eight threads, each on its own stream: plan, workspace and error text are each call's own."""
    shapes = [(13, 264, 1040), (40, 520, 4112), (300, 520, 2064), (900, 1288, 96)] * 2
    sets = [_whole(*s, seed=i, device=cuda) for i, s in enumerate(shapes)]
    want = [(a @ w.t().contiguous()).to(torch.bfloat16) for _, a, w in sets]
    torch.cuda.synchronize()

    def work(i):
        q, same = sets[i][0], True
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(25):
                same &= torch.equal(hip.gemm_fp8_block(*q), want[i])
                with pytest.raises(hip.Lx2vError, match=f"K={16 * i + 8} "):   # refused: the text is this thread's own
                    k = 16 * i + 8
                    hip.gemm_fp8_block(*R.whole_operands(4, 8, k, 0, cuda))
        return same

    with concurrent.futures.ThreadPoolExecutor(8) as pool:
        assert all(pool.map(work, range(8)))
