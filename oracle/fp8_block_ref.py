"""Plain 64-bit / IEEE restatement of the block-scaled e4m3 Linear, its quantisers and the residual RMSNorm, for the tests.

The operand form is the one of the reference's per-block-128 fp8 scheme (lightx2v/common/ops/mm/mm_weight.py): one fp32
scale per row and 128 columns of the activation, one per 128 x 128 block of the weight.  Its kernels live in a wheel that is
absent here: parity unpinned."""
import math

import torch

BLOCK, E4M3_MAX, AMAX_FLOOR = 128, 448.0, 1e-12


def blocks(x, block_rows):
    """[rows, cols] -> [row blocks, block_rows, groups, 128] with zeros past the edges."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return x.reshape(x.shape[0] // block_rows, block_rows, x.shape[1] // BLOCK, BLOCK)


def quantise(x, block_rows):
    """fp32 / bf16 rows -> (e4m3, scale): fp32 arithmetic with one rounding per operation (on the CPU: torch divides a GPU tensor by a
    number as a product with its reciprocal), NaN skipped by the maximum."""
    rows, cols = x.shape
    b = blocks(x.float(), block_rows)
    amax = torch.where(b.isnan(), torch.zeros_like(b), b.abs()).amax(dim=(1, 3))
    scale = amax.clamp(min=AMAX_FLOOR) / E4M3_MAX
    q = b * (1.0 / scale)[:, None, :, None]
    q = torch.where(q.isnan(), q, q.clamp(-E4M3_MAX, E4M3_MAX))
    return q.reshape(b.shape[0] * block_rows, -1)[:rows, :cols].to(torch.float8_e4m3fn).contiguous(), scale


def dequantise(q, scale, block_rows):
    rows, cols = q.shape
    b = blocks(q.double(), block_rows) * scale.double()[:, None, :, None]
    return b.reshape(b.shape[0] * block_rows, -1)[:rows, :cols]


def linear(aq, a_scale, wq, w_scale, bias=None, epilogue="none", resid=None, gate=None):
    """(value, error bound) in 64 bits.  The bound has three parts.
    The fp8 MFMA: within a run of 8 consecutive k of one product it aligns the eight products at the largest exponent sum
    among them and keeps 13 bits below it (measured on the instruction: next to +256 and -256 in its run of 8, 2^(8 - 13) is
    kept and 2^(8 - 14) lost, in every position; outside the run nothing is lost down to 2^-23), so a product loses less than
    2^-13 of the largest |a| |w| of its run, the eight of a run less than 2^-10 of it, and all of them less than 2^-10 sum |a w|.
    A subnormal code has the exponent of the smallest normal one, so it counts as 2^-6 (a zero does not count).
    fp32 accumulation in any order, a step may truncate (2^-23): (K + 4 groups + 8) 2^-23 sum |a w|.
    Both are carried through the epilogue; then half a bf16 step of the result."""
    a, w = dequantise(aq, a_scale, 1), dequantise(wq, w_scale, BLOCK)
    v = a @ w.t().contiguous()
    size = [dequantise(torch.where(q.float() == 0, q.float(), q.float().abs().clamp(min=2.0 ** -6)), s, rows) for q, s, rows in ((aq, a_scale, 1), (wq, w_scale, BLOCK))]
    err = 2.0 ** -10 * (size[0] @ size[1].t().contiguous()) + (aq.shape[1] + 4 * a_scale.shape[1] + 8) * 2.0 ** -23 * (a.abs() @ w.abs().t().contiguous())
    if bias is not None:
        v = v + bias.double()
        err = err + 2.0 ** -23 * v.abs()
    if epilogue == "gelu":
        u = math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)
        # |gelu'| <= 1.13; u to a few 2^-24, exp(-2u) and the quotient to 2^-20 relative, which moves x * sigmoid(2u) by at
        # most 2^-20 (1 + |2u|) sigmoid(2u) |x| in its own scale
        sg = torch.sigmoid(2 * u)
        err = 1.13 * err + 2.0 ** -20 * (1 + 2 * u.abs()) * sg * v.abs()
        v = v * sg
    elif epilogue == "residual":
        if gate is not None:
            v, err = v * gate.double(), err * gate.double().abs()
        err = err + 2.0 ** -22 * v.abs()
        v = v + resid.double()
        err = err + 2.0 ** -23 * v.abs()
    return v, err + 2.0 ** -8 * (v.abs() + err)


def add_rmsnorm(x, y, w, eps):
    """(x + y, normalised row) in 64 bits."""
    h = x.double() + (0 if y is None else y.double())
    v = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    return h, v if w is None else v * w.double()


def whole_operands(M, N, K, seed, device="cpu"):
    """(a8, a_scale, w8, w_scale) whose products and sums are whole numbers that the fp8 MFMA and fp32 hold exactly, so that a correct
    product equals the 64-bit one before its rounding to bf16, whatever the order of its sums.  Dequantised, |a| and |w| are 2, here
    and there 1 or 3; the second half of K has a negative, so that sums grow to 2 K on the way and come back to the order of sqrt(K):
    mostly below 256, where bf16 has steps of at most 1 and every single product (1 to 9) shows.  Scales are powers of two that
    differ from block to block, the codes hold their inverse."""
    g = torch.Generator(device=device).manual_seed(seed)

    def near_two(rows):
        r = torch.randint(0, 16, (rows, K), generator=g, device=device)
        return 2.0 + (r == 0).float() - (r == 1).float()

    def powers(rows):
        return torch.exp2(torch.randint(-3, 4, (rows, (K + BLOCK - 1) // BLOCK), generator=g, device=device).float())

    a, w = near_two(M), near_two(N)
    a[:, K // 2:] *= -1
    a_scale, w_scale = powers(M), powers((N + BLOCK - 1) // BLOCK)
    a = a / a_scale.repeat_interleave(BLOCK, dim=1)[:, :K]
    w = w / w_scale.repeat_interleave(BLOCK, dim=0)[:N].repeat_interleave(BLOCK, dim=1)[:, :K]
    return a.to(torch.float8_e4m3fn), a_scale.t().contiguous().t(), w.to(torch.float8_e4m3fn), w_scale
