"""MXFP4 format (CPU): scale rule, rounding, atom layout, LoRA packing and the argument checks that need no GPU."""
import pytest
import torch

from granite_switch_b200.models.packing import interleave_gate_up
from granite_switch_b200.ops import gemm_fp4 as F


def _values(x):
    x4, sf = F.quantize_rows_reference(x)
    return F.dequantize_reference(x4, sf)


def test_scale_rule():
    """Smallest power of two with max|x| <= 7 * 2^e; byte 0 for zero and tiny maxima, 255 for what is not finite."""
    amax = torch.tensor([0.0, 6.0, 7.0, 7.03125, 14.0, 3.5, 3.515625, 2.0 ** -133, 2.9e38, float("inf"), float("nan")])
    b = F._scale_bytes(amax).long().tolist()
    assert b[:7] == [0, 127, 127, 128, 128, 126, 127]
    assert b[7] == 0 and b[9] == 255 and b[10] == 255
    assert 2.9e38 <= 7 * 2.0 ** (b[8] - 127) and 2.9e38 > 7 * 2.0 ** (b[8] - 128)
    # the largest bf16 values saturate at 6 * 2^125 rather than round to infinity
    assert F._scale_bytes(torch.tensor(torch.finfo(torch.bfloat16).max)) == 252


def test_rounding_to_e2m1():
    """Every border goes to the even code; above 6 saturates; signs are kept."""
    row = torch.zeros(1, 32)
    vals = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26, -5.5, 6.5, 0.2, -0.1, 4.9, 5.1, -7.0]
    row[0, : len(vals)] = torch.tensor(vals)
    want = [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.5, -6.0, 6.0, 0.0, -0.0, 4.0, 6.0, -6.0]
    assert _values(row)[0, : len(vals)].tolist() == want
    x4, _ = F.quantize_rows_reference(row)
    codes = torch.stack((x4 & 15, x4 >> 4), 2).view(-1)[: len(vals)].tolist()
    assert codes[12] == 8 and codes[0] == 7 and codes[15] == 15 and codes[8] == 9


@pytest.mark.parametrize("m,k", [(1, 32), (5, 64), (130, 288), (256, 256)])
def test_error_is_half_a_step(m, k):
    """e2m1 keeps one mantissa bit: off by at most a quarter of the value's power of two, at least by 0.25 * 2^e."""
    torch.manual_seed(m + k)
    x = torch.randn(m, k) * 10.0 ** torch.randint(-6, 7, (m, 1)).float()
    v = _values(x.bfloat16()).view(m, k // 32, 32)
    b = x.bfloat16().double().view(m, k // 32, 32)
    scale = F._pow2(F._scale_bytes(b.abs().amax(2, keepdim=True)).long() - 127)
    y = (b / scale).abs()
    half = torch.where(y < 2, 0.25, torch.where(y < 4, 0.5, 1.0))
    assert ((v - b).abs() <= half * scale).all()


def test_atom_layout():
    """Byte 16 (r % 32) + 4 (r // 32) + j holds row r's scale of sub-block j; K tiles are even and padded with 0."""
    m, k = 200, 160
    x = torch.ones(m, k)
    e = torch.randint(-20, 20, (m, k // 32))
    x = torch.ldexp(x.view(m, k // 32, 32), e.unsqueeze(2)).view(m, k) * 4
    _, sf = F.quantize_rows_reference(x)
    assert sf.shape == (2, 2, 512)
    for r in (0, 1, 31, 32, 127, 128, 199):
        t, rr = divmod(r, 128)
        for b in range(8):
            got = int(sf[t, b // 4, 16 * (rr % 32) + 4 * (rr // 32) + b % 4])
            assert got == (int(e[r, b]) + 127 if b < 5 else 0)
    assert torch.equal(F.scale_bytes_from_atoms(sf, m, k).long(), e + 127)


def test_not_finite_blocks_are_nan():
    x = torch.randn(3, 96)
    x[0, 5], x[1, 40], x[2, 95] = float("inf"), float("nan"), -float("inf")
    v = _values(x)
    for r, b in ((0, 0), (1, 1), (2, 2)):
        assert v[r, 32 * b: 32 * b + 32].isnan().all()
    assert int(v.isnan().sum()) == 96


def test_swiglu_lora_packing():
    """The doubled expand weights give each row its own half's delta."""
    torch.manual_seed(0)
    i, cols, m = 128, 64, 7
    gate, up = torch.randn(i, cols), torch.randn(i, cols)
    s = torch.randn(m, 2 * cols)
    lb2 = F.swiglu_lora_b(interleave_gate_up(torch.cat([gate, up]), F.SWIGLU_TILE))
    acc = (s @ lb2.t()).view(m, i // 64, 2, 64)
    assert torch.allclose(acc[:, :, 0].reshape(m, i), s[:, :cols] @ gate.t(), atol=1e-4)
    assert torch.allclose(acc[:, :, 1].reshape(m, i), s[:, cols:] @ up.t(), atol=1e-4)


def test_product_reference_with_slices():
    torch.manual_seed(1)
    m, n, k, cols = 4, 256, 64, 32
    x, w = torch.randn(m, k), torch.randn(n, k)
    s, lb = torch.randn(m, 2 * cols), torch.randn(n, cols)
    acc = F.mxfp4_product_reference(*F.quantize_rows_reference(x), *F.quantize_rows_reference(w), s=s, lb=lb,
                                    rank=32, num_adapters=1, slice_bounds=[0, 128, n])
    want = _values(x) @ _values(w).t()
    want[:, :128] += s[:, :cols].double() @ lb[:128].double().t()
    want[:, 128:] += s[:, cols:].double() @ lb[128:].double().t()
    assert torch.allclose(acc, want, rtol=1e-12, atol=1e-12)


def test_cpu_tensors_are_refused():
    """The ops are CUDA ops; a CPU tensor is refused before anything is launched."""
    pytest.importorskip("granite_switch_b200._C")
    x = torch.randn(4, 64).bfloat16()
    with pytest.raises(RuntimeError, match="CUDA"):
        F.quantize_rows_mxfp4(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.rmsnorm_mxfp4(x, torch.ones(64).bfloat16(), 1e-5)


def _packed(n, k, slices, swiglu=0, lora=True):
    from granite_switch_b200.models.packing import pack_linear

    g = torch.Generator().manual_seed(n + k)
    la = [torch.randn(2, 1, 8, k, generator=g) for _ in slices] if lora else None
    lb = [torch.randn(2, 1, s, 8, generator=g) for s in slices] if lora else None
    return pack_linear(torch.randn(n, k, generator=g), la, lb, slices, 2, "cpu", swiglu_tile=swiglu)


def test_quantise_linear():
    """A packed projection in 4 bits: codes of its weight, LoRA kept in bf16, gate/up expand weights doubled."""
    from granite_switch_b200.models.packing import quantise_linear

    pl = _packed(384, 96, [256, 128])
    w, lb = pl.w.clone(), pl.lb.clone()
    quantise_linear(pl)
    assert pl.w is None and torch.equal(pl.lb, lb)
    x4, sf = F.quantize_rows_reference(w)
    assert torch.equal(pl.w4, x4) and torch.equal(pl.sfw, sf)
    gu = _packed(256, 64, [128, 128], swiglu=F.SWIGLU_TILE)
    lb = gu.lb.clone()
    quantise_linear(gu)
    assert torch.equal(gu.lb, F.swiglu_lora_b(lb))


@pytest.mark.parametrize("kw,what", [(dict(n=64, k=48, slices=[64], lora=False), "multiple of 32"),
                                     (dict(n=20, k=64, slices=[20], lora=False), "N of 8"),
                                     (dict(n=128, k=64, slices=[64, 64]), "multiples of 128"),
                                     (dict(n=256, k=64, slices=[128, 128], swiglu=256), "interleaved")])
def test_projections_that_are_refused(kw, what):
    from granite_switch_b200.models.packing import quantise_linear

    with pytest.raises(ValueError, match=what):
        quantise_linear(_packed(**kw))


def test_engine_refuses_what_it_cannot_run():
    from granite_switch_b200.composer.synthetic import base_config
    from granite_switch_b200.config import GraniteSwitchConfig
    from granite_switch_b200.engine import LLM, EngineConfig

    cfg = GraniteSwitchConfig(**base_config("micro"), num_adapters=0)
    with pytest.raises(ValueError, match="weight_dtype"):
        LLM(cfg, device="cpu", engine_config=EngineConfig(weight_dtype="fp4"))
    with pytest.raises(ValueError, match="CUDA"):
        LLM(cfg, device="cpu", engine_config=EngineConfig(weight_dtype="mxfp4"))
