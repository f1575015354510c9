"""Refusals of the block-scaled e4m3 Linear, its quantisers and the residual RMSNorm: nothing is launched, no GPU is needed."""
import ctypes
import shutil
import subprocess

import pytest
import torch

from lightx2v_amd import hip
from oracle import fp8_block_ref as R


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096 + 16)
    yield (ctypes.addressof(buf) + 15) & ~15
    del buf


def _gemm(p, **kw):
    a = dict(A=p, lda=128, sa=p, lsa=64, W=p, ldw=128, sw=p, lsw=1, bias=None, C=p, ldc=64, M=8, N=64, K=128, epi=0, resid=None, ldr=0, gate=None, ws=None, wsb=0, st=None)
    a.update(kw)
    return hip.load().lx2v_gemm_fp8_block128(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(A=None), -1, b"null"), (dict(sa=None), -1, b"null"), (dict(sw=None), -1, b"null"), (dict(C=None), -1, b"null"),
    (dict(M=-1), -1, b"bad shape"), (dict(N=0), -1, b"bad shape"), (dict(K=0), -1, b"bad shape"), (dict(M=1 << 31, lsa=1 << 31), -2, b"31 bits"),
    (dict(K=120), -2, b"multiple of 16"), (dict(N=60), -2, b"of 8"), (dict(lda=136), -1, b"multiples of 16"), (dict(ldc=66), -1, b"ldc of 8"),
    (dict(lda=112), -1, b"smaller"), (dict(ldw=112), -1, b"smaller"), (dict(ldc=56), -1, b"smaller"), (dict(lda=1 << 22), -2, b"4 MiB"),
    (dict(lsa=7), -1, b"ld_a_scale"), (dict(K=256, lda=256, ldw=256), -1, b"ld_w_scale"), (dict(lsw=1 << 28), -2, b"too large"), (dict(epi=3), -1, b"unknown epilogue"), (dict(epi=2), -1, b"resid")])
def test_gemm_refuses(p, kw, code, text):
    assert _gemm(p, **kw) == code
    assert text in hip.load().lx2v_last_error(), hip.load().lx2v_last_error()


def test_gemm_refuses_misaligned_tensors(p):
    for name, off in (("A", 8), ("W", 8), ("C", 8), ("bias", 4), ("sa", 2), ("sw", 1)):
        assert _gemm(p, **{name: p + off}) == -1 and b"aligned" in hip.load().lx2v_last_error()
    for kw in (dict(resid=p + 8, ldr=64), dict(resid=p, ldr=60), dict(resid=p, ldr=56), dict(resid=p, ldr=64, gate=p + 4)):
        assert _gemm(p, epi=2, **kw) == -1
    assert _gemm(p, M=0) == 0   # nothing to do
    assert _gemm(p, M=0, A=None, W=None, C=None, sa=None, sw=None) == 0


def test_quantisers_and_norm_refuse(p):
    lib = hip.load()
    assert lib.lx2v_quant_fp8_group128(None, 128, None, p, 128, p, 4, 4, 128, None) == -1
    assert lib.lx2v_quant_fp8_group128(p, 128, None, p, 128, p, 4, 4, 124, None) == -1       # dim % 8
    assert lib.lx2v_quant_fp8_group128(p, 128, None, p, 128, p, 3, 4, 128, None) == -1       # scales overlap
    assert lib.lx2v_quant_fp8_group128(p, 120, None, p, 128, p, 4, 4, 128, None) == -1       # source rows overlap
    assert lib.lx2v_quant_fp8_group128(p + 2, 128, None, p, 128, p, 4, 4, 128, None) == -1
    bad = hip.KSeg(seg=64, stride=64, split=32, seg2=64, stride2=64, base2=0, lda2=64)
    assert lib.lx2v_quant_fp8_group128(p, 128, ctypes.byref(bad), p, 128, p, 4, 4, 128, None) == -1
    assert lib.lx2v_quant_fp8_group128(p, 128, None, p, 128, p, 0, 0, 128, None) == 0
    assert lib.lx2v_quant_fp8_block128(p, 128, p, 128, p, 0, 4, 128, None) == -1              # scale stride
    assert lib.lx2v_quant_fp8_block128(p, 128, p, 128, p, 1, 0, 128, None) == 0
    assert lib.lx2v_add_rmsnorm_bf16(p, 64, p, 64, None, p, 64, 4, 64, 1e-6, None) == -1 and b"out may not be x" in lib.lx2v_last_error()
    assert lib.lx2v_add_rmsnorm_bf16(p, 64, p, 64, None, p + 64, 64, 4, 8200, 1e-6, None) == -2
    assert lib.lx2v_add_rmsnorm_bf16(p, 64, p, 64, None, p + 64, 64, 4, 60, 1e-6, None) == -2
    assert lib.lx2v_add_rmsnorm_f32(p, 64, p, 56, None, p + 64, 64, 4, 64, 1e-6, None) == -1
    assert lib.lx2v_add_rmsnorm_f32(p, 64, p, 64, p + 4, p + 64, 64, 4, 64, 1e-6, None) == -1
    # more workgroups than a launch has
    assert lib.lx2v_add_rmsnorm_bf16(p, 2048, p, 2048, None, p + 64, 2048, 1 << 24, 2048, 1e-6, None) == -2 and b"workgroups" in lib.lx2v_last_error()
    assert lib.lx2v_add_rmsnorm_f32(p, 64, p, 64, None, p + 64, 64, 1 << 26, 64, 1e-6, None) == -2
    assert lib.lx2v_quant_fp8_group128(p, 512, None, p, 512, p, 1 << 29, 1 << 29, 512, None) == -2 and b"workgroups" in lib.lx2v_last_error()
    for form in (-1, 3):
        assert lib.lx2v_add_rmsnorm_quant_bf16(p, 64, p, 64, None, p + 64, 64, p, 4, form, 4, 64, 1e-6, None) == -1 and b"form" in lib.lx2v_last_error()
    assert lib.lx2v_add_rmsnorm_quant_bf16(p, 64, p, 64, None, p + 64, 64, None, 4, 0, 4, 64, 1e-6, None) == -1
    assert lib.lx2v_add_rmsnorm_quant_bf16(p, 64, p, 64, None, p + 64, 64, p, 3, 1, 4, 64, 1e-6, None) == -1   # scales overlap
    assert lib.lx2v_add_rmsnorm_quant_bf16(p, 64, p, 64, None, p + 64, 64, p, 0, 1, 0, 64, 1e-6, None) == 0


def test_python_refuses_cpu_tensors_and_wrong_types():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    q, s = R.quantise(x, 1)
    for call in (lambda: hip.quant_fp8_group128(x), lambda: hip.quant_fp8_block128(x), lambda: hip.add_rmsnorm_(x, x), lambda: hip.gemm_fp8_block(q, s, q, s),
                 lambda: hip.quant_fp8_group128(x.float()), lambda: hip.add_rmsnorm_(x.float(), x), lambda: hip.quant_fp8_block128(x.half())):
        with pytest.raises(hip.Lx2vError):
            call()


def test_oracle_quantisation_is_within_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 400, generator=g) * torch.exp(torch.randn(200, 1, generator=g))
    for rows in (1, 128):
        q, s = R.quantise(x, rows)
        d = R.dequantise(q, s, rows)
        grid = R.dequantise(torch.ones_like(x).to(torch.float8_e4m3fn), s, rows)
        assert bool(((d - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * grid) * (1 + 2.0 ** -20)).all())


def test_plugin_is_registered_and_refuses_what_does_not_fit():
    import lightx2v_amd as L

    cls = L.MM_WEIGHT_REGISTER["hip-fp8-block128"]
    w = torch.zeros(200, 320).to(torch.float8_e4m3fn)
    for name in ("w.weight_scale", "w.weight_scale_inv"):
        mm = cls("w.weight", None)
        mm.load({"w.weight": w, name: torch.ones(2, 3, dtype=torch.float64)})
        assert mm.weight_scale.dtype is torch.float32 and mm._calculate_size() == 200 * 320 + 24
    with pytest.raises(ValueError, match="128 x 128"):    # one scale per output row: another scheme's checkpoint
        cls("w.weight", None).load({"w.weight": w, "w.weight_scale": torch.ones(200, 1)})
    with pytest.raises(KeyError):
        cls("w.weight", None).load({"w.weight": w})
    with pytest.raises(ValueError, match="fused"):
        cls.fused([mm, mm])
    fused = cls.fused([mm])
    assert fused.weight_nk.shape == (200, 320) and fused.weight_scale.shape == (2, 3)
    with pytest.raises(ValueError):
        mm.adopt(w, None)
    with pytest.raises(NotImplementedError):
        mm.load_state_dict({}, 0)
    with pytest.raises(hip.Lx2vError):
        mm.apply(hip.QuantRows(w, torch.ones(200)))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no GPU"):
            cls("w.weight", None).load({"w.weight": torch.zeros(128, 128)})
    assert [L.MM_WEIGHT_REGISTER[n].norm_form for n in ("hip-bf16", "hip-fp8", "hip-int8", "hip-fp8-block128")] == [None, "row", "int8", "group"]
    assert "hip-fp8-block128" in L.WanTransformerWeights({"num_layers": 1, "num_heads": 2, "dim": 256, "task": "t2v", "dit_quant_scheme": "hip-fp8-block128"}).mm_type


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_a_library_of_other_sources_is_refused_by_name(tmp_path, monkeypatch):
    def built(name, skip, version):
        src = tmp_path / f"{name}.c"
        src.write_text("".join(f"int {e}(void) {{ return {version if e == 'lx2v_abi_version' else 0}; }}\n" for e in hip.EXPORTS if e not in skip))
        so = tmp_path / f"{name}.so"
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
        return str(so)

    monkeypatch.setattr(hip, "_lib", None)
    older = built("older", ("lx2v_gemm_fp8_block128", "lx2v_quant_fp8_group128"), hip.ABI_VERSION)
    monkeypatch.setattr(hip, "lib_path", lambda: older)
    with pytest.raises(RuntimeError, match="lacks 2 of .*lx2v_quant_fp8_group128, lx2v_gemm_fp8_block128.* rebuild"):
        hip.load()
    other = built("other", (), hip.ABI_VERSION + 1)
    monkeypatch.setattr(hip, "lib_path", lambda: other)
    with pytest.raises(RuntimeError, match=f"ABI version {hip.ABI_VERSION + 1}, .* needs {hip.ABI_VERSION}"):
        hip.load()
    assert hip._lib is None
    same = built("same", (), hip.ABI_VERSION)
    monkeypatch.setattr(hip, "lib_path", lambda: same)
    assert hip.load() is hip._lib is not None


def test_more_columns_than_32_bits_count_are_refused(p):
    """2^32 + 8 columns would reach the entry points as 8."""
    lib, big, ld = hip.load(), 2 ** 31 - 8, 1 << 31
    assert lib.lx2v_quant_fp8_group128(p, ld, None, p, ld, p, 1, 1, big, None) == -2 and b"columns" in lib.lx2v_last_error()
    assert lib.lx2v_quant_fp8_group128_f32(p, ld, p, ld, p, 1, 1, big, None) == -2 and b"columns" in lib.lx2v_last_error()
    assert lib.lx2v_quant_fp8_block128(p, ld, p, ld, p, ld, 1, big, None) == -2 and b"columns" in lib.lx2v_last_error()
    assert lib.lx2v_quant_fp8_block128_f32(p, ld, p, ld, p, ld, 1, big, None) == -2 and b"columns" in lib.lx2v_last_error()
    wide = torch.empty(1, 2 ** 32 + 8, dtype=torch.bfloat16, device="meta")
    for call in (lambda: hip.quant_fp8_group128(wide), lambda: hip.quant_fp8_block128(wide), lambda: hip.add_rmsnorm_(wide, None)):
        with pytest.raises(hip.Lx2vError, match="columns"):
            call()
