"""MXFP4 quantisers and products against their fp64 statements (GPU).

Tolerances. Quantisation is exact arithmetic up to the comparison with a border, so bytes are equal.
A product sums K exact terms in fp32: each of the K / 64 accumulations and each sum inside one may lose a
few units of 2^-24 of the terms' absolute sum, taken as (K / 32 + 16) 2^-23 of it; the output adds bf16's half
step, 2^-8 of the value. SwiGLU's fp32 exponential and division add 2^-19 of the value.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA")
    from granite_switch_b200 import _native

    _native.native()  # fail loudly if the extension is missing
    yield
    _native.check_errors(torch.device("cuda", torch.cuda.current_device()))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(m, k, seed, spread=6):
    """bf16 values whose blocks of 32 span several decades, so that a misplaced scale shows."""
    g = _gen(seed)
    x = torch.randn(m, k, device="cuda", generator=g)
    e = torch.randint(-spread, spread + 1, (m, k // 32, 1), device="cuda", generator=g).float()
    return (x.view(m, k // 32, 32) * 2.0 ** e).view(m, k).to(torch.bfloat16)


def _acc_tol(x4, sfx, w4, sfw, extra=0.0):
    from granite_switch_b200.ops import gemm_fp4 as F

    k = 2 * x4.shape[1]
    mass = F.dequantize_reference(x4, sfx).abs() @ F.dequantize_reference(w4, sfw).abs().t() + extra
    return (k / 32 + 16) * 2.0 ** -23 * mass


def _check(out, ref, tol):
    out = out.double()
    bad = ~((out - ref).abs() <= tol + ref.abs() * 2.0 ** -8 + 2.0 ** -133)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off; first {bad.nonzero()[0].tolist()}: " \
                          f"{out[bad][0].item()} vs {ref[bad][0].item()}"


def _check_codes(x4, sf, ref, tol):
    """Codes stand for `ref` to within half a step of their own scale, and the scale is the smallest allowed
    (or its neighbour where the block's largest value lies within `tol` of the border)."""
    from granite_switch_b200.ops import gemm_fp4 as F

    m, k = ref.shape
    v = F.dequantize_reference(x4, sf).view(m, k // 32, 32)
    byte = F.scale_bytes_from_atoms(sf, m, k)
    b, t = ref.view(m, k // 32, 32), tol.view(m, k // 32, 32)
    lo, hi = F._scale_bytes((b.abs() - t).clamp(min=0).amax(2)), F._scale_bytes((b.abs() + t).amax(2))
    assert ((byte >= lo) & (byte <= hi)).all()
    scale = F._pow2(byte.long().unsqueeze(2) - 127)
    y = b.abs() / scale
    half = torch.where(y < 2, 0.25, torch.where(y < 4, 0.5, 1.0))
    # past a binade's border by the tolerance, the step above may already hold
    half = torch.maximum(half, torch.where((y < 2) & (y + t / scale >= 2), 0.5, half))
    half = torch.maximum(half, torch.where((y < 4) & (y + t / scale >= 4), 1.0, half))
    bad = ~((v - b).abs() <= half * scale + t)
    assert not bad.any(), f"{int(bad.sum())} values off by more than half a step"
    pad = F.scale_bytes_from_atoms(sf, m, sf.shape[1] * 128)[:, k // 32:]
    assert not pad.any(), "scales past K must be 0"


# ------------------------------------------------------------------------------------------- quantisers
@pytest.mark.parametrize("m", [1, 3, 128, 257])
@pytest.mark.parametrize("k", [32, 96, 256, 2080, 4096])
def test_quantize_matches_reference(m, k):
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(m, k, seed=m * 7 + k)
    x4, sf = F.quantize_rows_mxfp4(x)
    r4, rsf = F.quantize_rows_reference(x)
    assert torch.equal(x4, r4)
    kt = sf.shape[1] * 128
    assert torch.equal(F.scale_bytes_from_atoms(sf, m, kt), F.scale_bytes_from_atoms(rsf, m, kt))
    assert torch.equal(F.dequantize_mxfp4(x4, sf).double(), F.dequantize_reference(r4, rsf))


@pytest.mark.parametrize("m,k", [(700, 8736), (1003, 4640), (1800, 4640), (2000, 4608), (2500, 4128), (4100, 2080)])
def test_quantize_many_rows(m, k):
    """Sizes at which a warp takes two or four units of a row, with rows that end inside a warp's units."""
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(m, k, seed=m + k)
    x4, sf = F.quantize_rows_mxfp4(x)
    r4, rsf = F.quantize_rows_reference(x)
    assert torch.equal(x4, r4)
    kt = sf.shape[1] * 128
    assert torch.equal(F.scale_bytes_from_atoms(sf, m, kt), F.scale_bytes_from_atoms(rsf, m, kt))
    out = torch.full((m + 1, k), 5.0, dtype=torch.bfloat16, device="cuda")
    F.dequantize_mxfp4(x4, sf, out[:m])
    assert torch.equal(out[:m].double(), F.dequantize_reference(r4, rsf)) and (out[m:] == 5.0).all()


def test_quantize_edges_and_strides():
    """Zeros, subnormals, the largest bf16, borders, infinities and NaN; rows wider than their K; a caller's buffers
    with rows behind the last one left alone."""
    from granite_switch_b200.ops import gemm_fp4 as F

    wide = torch.zeros(9, 512, device="cuda", dtype=torch.bfloat16)
    wide[:, 256:] = 77.0  # neighbours that are not part of the rows
    x = wide[:, :160]
    x[1, :32] = torch.tensor(2.0 ** -133)
    x[2] = torch.finfo(torch.bfloat16).max
    x[3, :8] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[4, 33] = float("inf")
    x[5, 2] = float("nan")
    x[6, 64:96] = -0.0
    x[7] = torch.randn(160, device="cuda", generator=_gen(1)).to(torch.bfloat16) * 2.0 ** -126
    x[8, 159] = -float("inf")
    codes = torch.full((12, 96), 0xAB, dtype=torch.uint8, device="cuda")
    x4, sf = F.quantize_rows_mxfp4(x, x4=codes[:9, :80])
    r4, rsf = F.quantize_rows_reference(x)
    assert torch.equal(x4, r4)
    assert torch.equal(F.scale_bytes_from_atoms(sf, 9, 256), F.scale_bytes_from_atoms(rsf, 9, 256))
    assert (codes[9:] == 0xAB).all() and (codes[:, 80:] == 0xAB).all()
    back = F.dequantize_mxfp4(x4, sf)
    assert back[4, 32:64].isnan().all() and back[5, :32].isnan().all() and back[8, 128:].isnan().all()
    assert torch.equal(torch.nan_to_num(back.double()), torch.nan_to_num(F.dequantize_reference(r4, rsf)))
    assert (back[2].double() == 6 * 2.0 ** 125).all()


@pytest.mark.parametrize("m,h", [(1, 32), (5, 256), (33, 2080), (130, 4096), (3, 16384), (1300, 2048), (1301, 4096),
                                 (1200, 2080), (1190, 96)])
@pytest.mark.parametrize("with_out", [False, True])
def test_rmsnorm_quantised(m, h, with_out):
    from granite_switch_b200.ops import elementwise as E
    from granite_switch_b200.ops import gemm_fp4 as F

    g = _gen(h)
    x = (torch.randn(m, h, device="cuda", generator=g) * 3).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(h, device="cuda", generator=g)).to(torch.bfloat16)
    out = torch.empty(m, h, dtype=torch.bfloat16, device="cuda") if with_out else None
    x4, sf = F.rmsnorm_mxfp4(x, w, 1e-5, out=out)
    xd = x.double()
    ref = xd * torch.rsqrt(xd.square().mean(1, keepdim=True) + 1e-5) * w.double()
    # sum of H squares in fp32, the root and one product: (log2 H + 6) units of 2^-24
    _check_codes(x4, sf, ref, ref.abs() * (h.bit_length() + 6) * 2.0 ** -23)
    if with_out:
        assert torch.equal(out, E.rmsnorm(x, w, 1e-5))


def test_quantize_past_32_bits():
    """Offsets of the last rows pass 2^31 elements."""
    from granite_switch_b200.ops import gemm_fp4 as F

    m, k = 66000, 32768
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    tail = _rows(3, k, seed=3)
    x[-3:] = tail
    x4, sf = F.quantize_rows_mxfp4(x)
    r4, rsf = F.quantize_rows_reference(tail)
    assert torch.equal(x4[-3:], r4)
    assert torch.equal(F.dequantize_mxfp4(x4, sf)[-3:].double(), F.dequantize_reference(r4, rsf))
    assert not x4[:-3].any()


# ------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("m", [1, 2, 3, 4, 16, 77, 128, 200, 300, 600])
@pytest.mark.parametrize("n,k", [(256, 256), (8, 32), (264, 1056), (1024, 4096), (4096, 288), (12808, 96)])
def test_gemm_store(m, n, k):
    from granite_switch_b200.ops import gemm_fp4 as F

    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=1)), F.quantize_rows_mxfp4(_rows(n, k, seed=2, spread=3))
    out = F.mxfp4_gemm(*a, *b, scale=0.5)
    _check(out, 0.5 * F.mxfp4_product_reference(*a, *b), 0.5 * _acc_tol(*a, *b))


@pytest.fixture
def pair_always():
    from granite_switch_b200._native import native

    old = native().mxfp4_pair_min_m(0)
    yield
    native().mxfp4_pair_min_m(old)


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 264, 4096), (129, 136, 288), (260, 1032, 2080), (384, 384, 256)])
@pytest.mark.parametrize("residual", [False, True])
def test_pair_kernel_at_its_edges(pair_always, m, n, k, residual):
    """The CTA-pair kernel on sizes that the rule gives to the split kernel: partial tiles in every direction."""
    from granite_switch_b200.ops import gemm_fp4 as F

    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=31)), F.quantize_rows_mxfp4(_rows(n, k, seed=32, spread=2))
    ref, tol = F.mxfp4_product_reference(*a, *b), _acc_tol(*a, *b)
    if residual:
        h = torch.randn(m, n, device="cuda", generator=_gen(33)).to(torch.bfloat16)
        ref, tol = h.double() + 0.5 * ref, 0.5 * tol + h.double().abs() * 2.0 ** -23
        _check(F.mxfp4_gemm(*a, *b, h, epi=F.EPI_RESADD, scale=0.5, residual=h), ref, tol)
    else:
        _check(F.mxfp4_gemm(*a, *b), ref, tol)


@pytest.mark.parametrize("m", [3, 200, 1400])
@pytest.mark.parametrize("na,rank", [(64, 32), (3, 96)])
def test_gemm_lora_limits(m, na, rank):
    """As many adapters as a mask has bits, a rank of three blocks, mask bits past the last adapter, K over several
    cluster parts."""
    from granite_switch_b200.ops import gemm_fp4 as F

    n, k = 1024, 2048
    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=34)), F.quantize_rows_mxfp4(_rows(n, k, seed=35, spread=2))
    s, dirty, lb, mask = _lora_inputs(m, n, 2, na, rank, seed=36)
    if na < 64:
        mask = mask | (5 << na)
    kw = dict(lb=lb, rank=rank, num_adapters=na, slice_bounds=[0, 640, n])
    ref = F.mxfp4_product_reference(*a, *b, s=s, **kw)
    tol = _acc_tol(*a, *b, extra=(s.double().abs().sum(1, keepdim=True) * lb.double().abs().max()))
    _check(F.mxfp4_gemm(*a, *b, s=dirty, tile_mask=mask, **kw), ref, tol)


def test_two_streams_at_once():
    """Calls of every kernel on two streams that overlap give what they give alone."""
    from granite_switch_b200.ops import gemm_fp4 as F

    b = F.quantize_rows_mxfp4(_rows(4096, 2048, seed=37, spread=1))
    xs = [_rows(m, 2048, seed=m, spread=1) for m in (7, 100, 700, 2000)]
    want = [F.mxfp4_linear(x, *b) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] += [F.mxfp4_linear(x, *b) for x in (xs if i else xs[::-1])]
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for j, y in enumerate(outs):
            assert torch.equal(y, (want if i else want[::-1])[j % 4])


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (222, 1024, 2080), (2048, 2304, 512), (1300, 4096, 1024)])
def test_gemm_residual_in_place(m, n, k):
    """The residual may be the output; rows of a wider, taller buffer are left as they were."""
    from granite_switch_b200.ops import gemm_fp4 as F

    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=3)), F.quantize_rows_mxfp4(_rows(n, k, seed=4, spread=2))
    buf = torch.randn(m + 5, n + 64, device="cuda", generator=_gen(5)).to(torch.bfloat16)
    keep = buf.clone()
    h = buf[:m, :n]
    ref = h.double() + 0.22 * F.mxfp4_product_reference(*a, *b)
    F.mxfp4_gemm(*a, *b, h, epi=F.EPI_RESADD, scale=0.22, residual=h)
    _check(h, ref, 0.22 * _acc_tol(*a, *b) + keep[:m, :n].abs().double() * 2.0 ** -23)
    assert torch.equal(buf[m:], keep[m:]) and torch.equal(buf[:, n:], keep[:, n:])


def _lora_inputs(m, n, slices, na, rank, seed, absent=2):
    """Masked shrink output as the shrink leaves it: zero for other adapters of a 128-row tile, old values (NaN
    here) in the columns of adapters that no row of the tile uses."""
    g = _gen(seed)
    ra = torch.randint(0, na + 1, (m,), device="cuda", generator=g)
    ra[ra == absent] = 0
    if m > 128:
        ra[128:] = torch.where(ra[128:] == 1, 0, ra[128:])  # adapter 1 only in the first tile
    cols = slices * na * rank
    col = (torch.arange(cols, device="cuda") // rank) % na + 1
    s = torch.randn(m, cols, device="cuda", generator=g) * (col == ra[:, None])
    tiles = (m + 127) // 128
    mask = torch.zeros(tiles, dtype=torch.int64)
    dirty = s.clone()
    for t in range(tiles):
        here = set(ra[t * 128:(t + 1) * 128].tolist()) - {0}
        bits = sum(1 << (a - 1) for a in here)
        mask[t] = bits - (1 << 64 if bits >> 63 else 0)
        gone = torch.tensor([int(c) not in here for c in col.tolist()], device="cuda")
        dirty[t * 128:(t + 1) * 128, gone] = float("nan")
    lb = (torch.randn(n, na * rank, device="cuda", generator=g) * 0.5).to(torch.bfloat16)
    return s.to(torch.bfloat16), dirty.to(torch.bfloat16), lb, mask.cuda()


@pytest.mark.parametrize("m", [1, 3, 5, 130, 300, 1100])
@pytest.mark.parametrize("bounds", [[0, 640], [0, 1024, 1280, 1536], [0, 384, 512, 2176]])
def test_gemm_lora_slices(m, bounds):
    from granite_switch_b200.ops import gemm_fp4 as F

    k, na, rank, n = 512, 5, 64, bounds[-1]
    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=6)), F.quantize_rows_mxfp4(_rows(n, k, seed=7, spread=2))
    s, dirty, lb, mask = _lora_inputs(m, n, len(bounds) - 1, na, rank, seed=8)
    kw = dict(lb=lb, rank=rank, num_adapters=na, slice_bounds=bounds)
    ref = F.mxfp4_product_reference(*a, *b, s=s, **kw)
    tol = _acc_tol(*a, *b, extra=(s.double().abs().sum(1, keepdim=True) * lb.double().abs().max()))
    _check(F.mxfp4_gemm(*a, *b, s=dirty, tile_mask=mask, **kw), ref, tol)
    _check(F.mxfp4_gemm(*a, *b, s=s, **kw), ref, tol)  # without a mask every adapter is expanded


@pytest.mark.parametrize("m", [1, 3, 16, 17, 64, 300])
@pytest.mark.parametrize("n,k", [(256, 32), (264, 288), (4096, 2080), (1024, 12800)])
def test_linear_is_quantise_then_gemm(m, n, k):
    """Bit for bit, whether the rows are quantised in a kernel of their own or on the way; strided rows."""
    from granite_switch_b200.ops import gemm_fp4 as F

    wide = torch.full((m, k + 64), 3.0, device="cuda", dtype=torch.bfloat16)
    wide[:, :k] = _rows(m, k, seed=m)
    x = wide[:, :k]
    b = F.quantize_rows_mxfp4(_rows(n, k, seed=2, spread=2))
    s, dirty, lb, mask = _lora_inputs(m, n // 128 * 128 or n, 1, 3, 32, seed=4)
    want = F.mxfp4_gemm(*F.quantize_rows_mxfp4(x), *b)
    assert torch.equal(F.mxfp4_linear(x, *b), want)
    if n % 128 == 0:
        kw = dict(s=dirty, lb=lb, rank=32, num_adapters=3, tile_mask=mask, residual=want, epi=F.EPI_RESADD, scale=0.5)
        assert torch.equal(F.mxfp4_linear(x, *b, **kw), F.mxfp4_gemm(*F.quantize_rows_mxfp4(x), *b, **kw))


@pytest.mark.parametrize("m,i,h", [(1, 64, 64), (2, 1600, 288), (4, 320, 512), (17, 192, 512), (130, 1600, 256), (300, 512, 1056), (1300, 4096, 512)])
@pytest.mark.parametrize("lora", [False, True])
def test_gemm_swiglu(m, i, h, lora):
    from granite_switch_b200.models.packing import interleave_gate_up
    from granite_switch_b200.ops import gemm_fp4 as F

    a = F.quantize_rows_mxfp4(_rows(m, h, seed=9, spread=1))
    w = interleave_gate_up(_rows(2 * i, h, seed=10, spread=1) * h ** -0.5, F.SWIGLU_TILE)
    b = F.quantize_rows_mxfp4(w)
    kw, kd, extra = {}, {}, 0.0
    if lora:
        s, dirty, lb, mask = _lora_inputs(m, 2 * i, 2, 3, 32, seed=11)
        lb2 = F.swiglu_lora_b(lb)
        kw = dict(lb=lb2, rank=32, num_adapters=3)
        kd = dict(s=dirty, tile_mask=mask)
        extra = s.double().abs().sum(1, keepdim=True) * lb.double().abs().max()
        acc = F.mxfp4_product_reference(*a, *b, s=s, **kw)
    else:
        acc = F.mxfp4_product_reference(*a, *b)
    act = torch.full((m + 2, i), 5.0, dtype=torch.bfloat16, device="cuda")
    a4, sf = F.mxfp4_gemm_swiglu(*a, *b, act=act[:m], **kw, **kd)
    ref = F.swiglu_reference(acc)
    t = _acc_tol(*a, *b, extra=extra).view(m, -1, 2, 64)
    v = acc.view(m, -1, 2, 64)
    # |silu'| <= 1.1
    tol = (1.1 * v[:, :, 1].abs() * t[:, :, 0] + v[:, :, 0].abs() * t[:, :, 1] + t[:, :, 0] * t[:, :, 1]).reshape(m, i)
    tol = tol + ref.abs() * 2.0 ** -19
    _check(act[:m], ref, tol)
    assert (act[m:] == 5.0).all()
    _check_codes(a4, sf, ref, tol)
    b4, bsf = F.mxfp4_gemm_swiglu(*a, *b, **kw, **kd)
    assert torch.equal(a4, b4) and torch.equal(F.scale_bytes_from_atoms(sf, m, i), F.scale_bytes_from_atoms(bsf, m, i))


@pytest.mark.parametrize("m", [2, 190, 1025])
def test_mlp_block(m):
    """Norm, gate/up, SwiGLU and down projection as a decoder runs them, each stage against fp64 on its own input."""
    from granite_switch_b200.models.packing import interleave_gate_up
    from granite_switch_b200.ops import gemm_fp4 as F

    h, i = 512, 1088
    g = _gen(12)
    x = torch.randn(m, h, device="cuda", generator=g).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(h, device="cuda", generator=g)).to(torch.bfloat16)
    gu = torch.randn(2 * i, h, device="cuda", generator=g).to(torch.bfloat16) * h ** -0.5
    down = torch.randn(h, i, device="cuda", generator=g).to(torch.bfloat16) * i ** -0.5
    gu4, dn4 = F.quantize_rows_mxfp4(interleave_gate_up(gu, F.SWIGLU_TILE)), F.quantize_rows_mxfp4(down)
    xq = F.rmsnorm_mxfp4(x, w, 1e-5)
    aq = F.mxfp4_gemm_swiglu(*xq, *gu4)
    out = F.mxfp4_gemm(*aq, *dn4, epi=F.EPI_RESADD, scale=0.22, residual=x)
    ref = x.double() + 0.22 * F.mxfp4_product_reference(*aq, *dn4)
    _check(out, ref, 0.22 * _acc_tol(*aq, *dn4) + x.double().abs() * 2.0 ** -23)
    # against the whole block in fp64 from the same 4-bit weights: only rounding borders differ
    full = F.swiglu_reference(F.mxfp4_product_reference(*xq, *gu4))
    full = F.dequantize_reference(*F.quantize_rows_reference(full)) @ F.dequantize_reference(*dn4).t()
    assert ((out.double() - x.double() - 0.22 * full).norm() / (0.22 * full).norm()).item() < 2.0 ** -6


def test_broadcast_rows_and_in_place_norm():
    """One row for all as input; the norm's bf16 rows over its own input."""
    from granite_switch_b200.ops import elementwise as E
    from granite_switch_b200.ops import gemm_fp4 as F

    row = _rows(1, 512, seed=41)
    w = torch.ones(512, device="cuda").bfloat16()
    b = F.quantize_rows_mxfp4(_rows(256, 512, seed=42, spread=1))
    for m in (3, 300):
        assert torch.equal(F.mxfp4_linear(row.expand(m, 512), *b), F.mxfp4_linear(row.repeat(m, 1), *b))
        x = torch.randn(m, 512, device="cuda", generator=_gen(43)).to(torch.bfloat16)
        want, ref = E.rmsnorm(x, w, 1e-5), F.rmsnorm_mxfp4(x, w, 1e-5)
        x4, sf = F.rmsnorm_mxfp4(x, w, 1e-5, out=x)
        assert torch.equal(x, want) and torch.equal(x4, ref[0])
        assert torch.equal(F.scale_bytes_from_atoms(sf, m, 512), F.scale_bytes_from_atoms(ref[1], m, 512))


def test_nan_and_empty():
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(20, 512, seed=13)
    x[3, 100] = float("inf")
    b = F.quantize_rows_mxfp4(_rows(256, 512, seed=14, spread=1))
    out = F.mxfp4_linear(x, *b)
    assert out[3].isnan().all()
    rest = torch.arange(20, device="cuda") != 3
    assert out[rest].isfinite().all()
    few = F.mxfp4_linear(x[2:5], *b)
    assert few[1].isnan().all() and few[::2].isfinite().all()
    none = torch.empty(0, 512, dtype=torch.bfloat16, device="cuda")
    assert F.mxfp4_linear(none, *b).shape == (0, 256)
    a4, _ = F.mxfp4_gemm_swiglu(*F.rmsnorm_mxfp4(none, torch.ones(512, device="cuda").bfloat16(), 1e-5), *b)
    assert a4.shape == (0, 64)


def _check_swiglu_not_finite(m):
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(m, 256, seed=51, spread=1)
    b = F.quantize_rows_mxfp4(_rows(384, 256, seed=52, spread=1))
    clean = F.mxfp4_gemm_swiglu(*F.quantize_rows_mxfp4(x), *b)
    x[2, 7] = float("nan")
    x[m - 1, 200] = float("-inf")
    act = torch.empty(m, 192, dtype=torch.bfloat16, device="cuda")
    a4, sf = F.mxfp4_gemm_swiglu(*F.quantize_rows_mxfp4(x), *b, act=act)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[2] = bad[m - 1] = True
    got, want = (F.scale_bytes_from_atoms(t, m, 192) for t in (sf, clean[1]))
    assert (a4[bad] == 0).all() and (got[bad] == 255).all() and act[bad].isnan().all()
    assert torch.equal(a4[~bad], clean[0][~bad]) and torch.equal(got[~bad], want[~bad]) and act[~bad].isfinite().all()


@pytest.mark.parametrize("m", [5, 200])
def test_swiglu_rows_that_are_not_finite(m):
    """A NaN or infinity in a row makes its blocks' scales NaN and their codes 0, and leaves the other rows alone."""
    _check_swiglu_not_finite(m)


@pytest.mark.parametrize("m", [5, 300])
def test_pair_swiglu_rows_that_are_not_finite(pair_always, m):
    _check_swiglu_not_finite(m)


def test_output_past_32_bits():
    from granite_switch_b200.ops import gemm_fp4 as F

    m, n, k = 264000, 8192, 64
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-2:] = _rows(2, k, seed=15, spread=1)
    b = F.quantize_rows_mxfp4(_rows(n, k, seed=16, spread=1))
    out = F.mxfp4_linear(x, *b)
    a = F.quantize_rows_mxfp4(x[-2:])
    _check(out[-2:], F.mxfp4_product_reference(*a, *b), _acc_tol(*a, *b))
    assert not out[-300:-2].any()


def test_streams_and_graphs():
    """A call on another stream, and a captured pass replayed on new inputs, give the eager result bit for bit."""
    from granite_switch_b200.ops import gemm_fp4 as F

    m, n, k = 48, 1024, 2048
    xs = [_rows(m, k, seed=s, spread=1) for s in (17, 18)]
    b = F.quantize_rows_mxfp4(_rows(n, k, seed=19, spread=1))
    want = [F.mxfp4_linear(x, *b) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.mxfp4_linear(xs[0], *b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.mxfp4_linear(x, *b)
    for src, ref in zip(xs[::-1], want[::-1]):
        x.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_programmatic_launch_matches():
    """Weights quantised just before, and kernels of either launch kind around: results are the same. (The MXFP4
    kernels are always programmatic dependents; set_pdl makes the others so too.)"""
    from granite_switch_b200._native import native
    from granite_switch_b200.ops import elementwise as E
    from granite_switch_b200.ops import gemm_fp4 as F

    x, w = _rows(64, 2048, seed=20, spread=1), _rows(2048, 2048, seed=21, spread=1)
    want = F.mxfp4_linear(x, *F.quantize_rows_mxfp4(w))
    old = native().set_pdl(True)
    try:
        for _ in range(20):
            for on in (False, True):
                native().set_pdl(on)
                y = E.rmsnorm(x, torch.ones(2048, device="cuda").bfloat16(), 0.0)
                assert torch.equal(F.mxfp4_linear(x, *F.quantize_rows_mxfp4(w)), want)
                z = F.mxfp4_linear(y, *F.quantize_rows_mxfp4(w * 2))
                E.residual_axpy(z, z, 1.0)
                assert torch.equal(z, 2 * F.mxfp4_linear(y.clone(), *F.quantize_rows_mxfp4(w * 2)))
    finally:
        native().set_pdl(old)


def test_refusals():
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(16, 256, seed=22)
    a, b = F.quantize_rows_mxfp4(x), F.quantize_rows_mxfp4(_rows(256, 256, seed=23))
    out = torch.empty(16, 256, dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: F.quantize_rows_mxfp4(x.float()),
        lambda: F.quantize_rows_mxfp4(x[:, 1:33]),                                  # not 16-byte aligned
        lambda: F.quantize_rows_mxfp4(x.t()),
        lambda: F.quantize_rows_mxfp4(x[:, :48]),
        lambda: F.mxfp4_linear(x[:, :128], *b),
        lambda: F.quantize_rows_mxfp4(x, sf=a[1][:, :1]),
        lambda: F.quantize_rows_mxfp4(x, x4=a[0][:8]),
        lambda: F.rmsnorm_mxfp4(x, torch.ones(128, device="cuda").bfloat16(), 1e-5),
        lambda: F.rmsnorm_mxfp4(x, torch.ones(256, device="cuda"), 1e-5),
        lambda: F.dequantize_mxfp4(*a, out=torch.empty(16, 128, dtype=torch.bfloat16, device="cuda")),
        lambda: F.dequantize_mxfp4(*a, out=out[:1].expand(16, 256)),                # one row for all
        lambda: F.quantize_rows_mxfp4(x, x4=a[0][:1].expand(16, 128)),
        lambda: F.mxfp4_gemm(*a, *b, out=out[:1].expand(16, 256)),
        lambda: F.mxfp4_gemm(a[0][:, :64], a[1], *b),                               # K differs
        lambda: F.mxfp4_gemm(*a, b[0], a[1]),                                       # too few scales
        lambda: F.mxfp4_gemm(*a, b[0][:252], b[1]),                                 # N not a multiple of 8
        lambda: F.mxfp4_gemm(*a, *b, out=out.float()),
        lambda: F.mxfp4_gemm(*a, *b, out=out[:8]),
        lambda: F.mxfp4_gemm(*a, *b, epi=F.EPI_RESADD),
        lambda: F.mxfp4_gemm(*a, *b, epi=2),
        lambda: F.mxfp4_gemm(*a, *b, s=out),
        lambda: F.mxfp4_gemm(*a, *b, s=out, lb=b[0].bfloat16(), rank=16, num_adapters=2),
        lambda: F.mxfp4_gemm(*a, *b, s=out, lb=b[0].bfloat16(), rank=32, num_adapters=65),
        lambda: F.mxfp4_gemm(*a, *b, s=out, lb=b[0].bfloat16(), rank=32, num_adapters=2, slice_bounds=[0, 100, 256]),
        lambda: F.mxfp4_gemm(*a, *b, s=out, lb=b[0].bfloat16(), rank=32, num_adapters=16),  # s too narrow
        lambda: F.mxfp4_gemm(*a, *b, s=out, lb=b[0].bfloat16(), rank=32, num_adapters=2,
                             tile_mask=torch.zeros(1, dtype=torch.int32, device="cuda")),
        lambda: F.mxfp4_gemm_swiglu(*a, b[0][:192], torch.empty(2, 2, 512, dtype=torch.uint8, device="cuda")),
        lambda: F.mxfp4_gemm(a[0].cpu(), a[1], *b),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")


@pytest.mark.parametrize("between", [False, True])
@pytest.mark.parametrize("source", ["dequantise", "product", "norm", "swiglu"])
def test_outputs_as_weights_of_the_next_product(source, between):
    """Rows that an MXFP4 kernel has just written are the weights of a decode-sized bf16 product, once directly and
    once with a quantiser launched in between, under programmatic launch, eagerly and replayed from a graph: the
    product of the new rows, as in plain stream order. (Three sets of rows go through one buffer.)"""
    from granite_switch_b200._native import native
    from granite_switch_b200.ops import gemm as G
    from granite_switch_b200.ops import gemm_fp4 as F

    n = k = 4096
    x = _rows(16, k, seed=61, spread=1)
    rows = [_rows(n, k if source in ("dequantise", "norm") else 512, seed=62 + i, spread=1) for i in range(3)]
    codes = [F.quantize_rows_mxfp4(r) for r in rows]
    b = F.quantize_rows_mxfp4(_rows(k if source == "product" else 2 * k, 512, seed=66, spread=1))
    ones = torch.ones(k, device="cuda").bfloat16()
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    write = dict(dequantise=lambda i: F.dequantize_mxfp4(*codes[i], out=w),
                 product=lambda i: F.mxfp4_gemm(*codes[i], *b, w),
                 norm=lambda i: F.rmsnorm_mxfp4(rows[i], ones, 1e-5, out=w),
                 swiglu=lambda i: F.mxfp4_gemm_swiglu(*codes[i], *b, act=w))[source]
    assert native().gemm_decode_plan(16, n, k, G.EPI_STORE, 0)[0] > 0  # the kernel that can read weights early

    def chain():
        outs = []
        for i in range(3):
            write(i)
            if between:
                F.quantize_rows_mxfp4(x)
            outs.append(G.switched_gemm(x, w))
        return outs

    old = native().set_pdl(False)
    try:
        want = chain()
        torch.cuda.synchronize()
        native().set_pdl(True)
        eager = [chain() for _ in range(5)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = chain()
        replayed = []
        for _ in range(5):
            for t in captured:
                t.zero_()
            graph.replay()
            replayed.append([t.clone() for t in captured])
        torch.cuda.synchronize()
        del graph
    finally:
        native().set_pdl(old)
    for got in eager + replayed:
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("m", [16, 222])
def test_constant_weights_match(m):
    """``w_constant`` changes when a decode-sized product starts reading, not its bits."""
    from granite_switch_b200._native import native
    from granite_switch_b200.ops import elementwise as E
    from granite_switch_b200.ops import gemm as G

    h, w = _rows(m, 4096, seed=67, spread=1), _rows(4096, 4096, seed=68, spread=1)
    gu = _rows(2048, 4096, seed=69, spread=1)
    ones = torch.ones(4096, device="cuda").bfloat16()

    def chain(constant):
        x = E.rmsnorm(h, ones, 1e-5)
        y = G.switched_gemm(x, w, epi=G.EPI_RESADD, residual=h, scale=0.5, w_constant=constant)
        return y, G.switched_gemm(E.rmsnorm(y, ones, 1e-5), gu, epi=G.EPI_SWIGLU, bn=128, w_constant=constant)

    old = native().set_pdl(False)
    try:
        want = chain(False)
        torch.cuda.synchronize()
        native().set_pdl(True)
        got = [chain(c) for c in (False, True) * 5]
        torch.cuda.synchronize()
    finally:
        native().set_pdl(old)
    for pair in got:
        assert all(torch.equal(a, c) for a, c in zip(pair, want))


def _programmatic_edges(graph):
    """(programmatic dependencies, all dependencies) of a captured graph."""
    import ctypes

    rt = ctypes.CDLL("libcudart.so.12")
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert rt.cudaGraphGetEdges_v2(raw, None, None, None, ctypes.byref(n)) == 0
    src, dst = (ctypes.c_void_p * n.value)(), (ctypes.c_void_p * n.value)()
    data = (ctypes.c_uint8 * (8 * n.value))()  # per edge: from port, to port, type, five reserved bytes
    assert rt.cudaGraphGetEdges_v2(raw, src, dst, data, ctypes.byref(n)) == 0
    return sum(data[8 * i + 2] == 1 for i in range(n.value)), n.value


def test_programmatic_launch_can_be_turned_off():
    """The MXFP4 kernels start as programmatic dependents as the extension is loaded and with set_pdl(1), and in
    plain stream order with set_pdl(0); their results are the same."""
    from granite_switch_b200._native import native
    from granite_switch_b200.ops import gemm_fp4 as F

    x = _rows(64, 1024, seed=71, spread=1)
    w = torch.ones(1024, device="cuda").bfloat16()
    b = F.quantize_rows_mxfp4(_rows(1024, 1024, seed=72, spread=1))
    outs = []
    for mode in (-1, 0, 1):
        old = native().set_pdl(mode)
        try:
            graph = torch.cuda.CUDAGraph(keep_graph=True)
            with torch.cuda.graph(graph):
                y = F.dequantize_mxfp4(*F.quantize_rows_mxfp4(F.mxfp4_linear(x, *b)))
                y = F.mxfp4_gemm(*F.rmsnorm_mxfp4(y, w, 1e-5), *b)
        finally:
            assert native().set_pdl(old) == mode
        few, every = _programmatic_edges(graph)
        assert every >= 5 and few == (0 if mode == 0 else every)
        graph.instantiate()
        graph.replay()
        outs.append(y.clone())
        torch.cuda.synchronize()
        del graph
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("m,n,k", [(3, 4096, 4096), (16, 512, 2048), (128, 2048, 12800)])
@pytest.mark.parametrize("part", [0, 1])
def test_a_part_that_gives_up_writes_nothing(m, n, k, part):
    """When one K part of a tile's cluster reports a wait that ran out, no CTA of the cluster stores sums that lack
    it: the output, a residual's in place, SwiGLU's codes and scales stay as they were. The error word says so, and
    the next call is right."""
    from granite_switch_b200 import _native
    from granite_switch_b200.ops import gemm_fp4 as F

    nat, dev = _native.native(), torch.device("cuda", torch.cuda.current_device())
    pair, _, ks, _ = nat.mxfp4_gemm_plan(m, n, k)
    assert not pair and ks > part  # every tile has that part
    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=73)), F.quantize_rows_mxfp4(_rows(n, k, seed=74, spread=2))
    h = torch.randn(m, n, device="cuda", generator=_gen(75)).to(torch.bfloat16)
    want = F.mxfp4_gemm(*a, *b, epi=F.EPI_RESADD, scale=0.5, residual=h)
    keep = h.clone()
    a4 = torch.full((m, n // 4), 0xAB, dtype=torch.uint8, device="cuda")
    sf = torch.full(((m + 127) // 128, (n // 2 + 255) // 256 * 2, 512), 0xCD, dtype=torch.uint8, device="cuda")
    act = torch.full((m, n // 2), 5.0, dtype=torch.bfloat16, device="cuda")
    assert _native.read_errors(dev) == 0
    old = nat.mxfp4_split_give_up(part)
    try:
        F.mxfp4_gemm(*a, *b, h, epi=F.EPI_RESADD, scale=0.5, residual=h)
        assert _native.read_errors(dev) == _native.ERR_GEMM_WAIT
        F.mxfp4_gemm_swiglu(*a, *b, a4, sf, act)
        assert _native.read_errors(dev) == _native.ERR_GEMM_WAIT
    finally:
        nat.mxfp4_split_give_up(old)
    assert torch.equal(h, keep) and (a4 == 0xAB).all() and (sf == 0xCD).all() and (act == 5.0).all()
    F.mxfp4_gemm(*a, *b, h, epi=F.EPI_RESADD, scale=0.5, residual=h)
    assert torch.equal(h, want) and _native.read_errors(dev) == 0


def test_too_many_rows_are_named():
    from granite_switch_b200.ops import gemm_fp4 as F

    few = F.quantize_rows_mxfp4(_rows(8, 32, seed=76))
    many = (torch.zeros(1 << 24, 16, dtype=torch.uint8, device="cuda"),
            torch.zeros(1 << 17, 2, 512, dtype=torch.uint8, device="cuda"))
    out = torch.empty(8, 8, dtype=torch.bfloat16, device="cuda")
    for a, b in ((many, few), (few, many)):
        with pytest.raises(RuntimeError, match="2\\^24 - 1 rows"):
            F.mxfp4_gemm(*a, *b, out)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        F.mxfp4_gemm(*few, few[0][:7], few[1], out)


def test_overlapping_outputs_are_refused():
    """An output that shares memory with what the call reads (or with another output) is refused, unless it is the
    residual, the norm's rows or the linear's rows themselves; columns and rows of one buffer beside them are not."""
    from granite_switch_b200.ops import elementwise as E
    from granite_switch_b200.ops import gemm_fp4 as F

    m, k = 200, 256
    bytes_ = torch.zeros(1 << 21, dtype=torch.uint8, device="cuda")

    def at(offset, shape, dtype=torch.uint8):
        n = shape[0] * shape[1] * torch.empty(0, dtype=dtype).element_size()
        return bytes_[offset:offset + n].view(dtype).view(shape)

    def atoms(offset, rows, cols):
        tiles, kt = (rows + 127) // 128, (cols + 255) // 256 * 2
        return bytes_[offset:offset + tiles * kt * 512].view(tiles, kt, 512)

    x = at(0, (m, k), torch.bfloat16)  # 102,400 bytes
    x.copy_(_rows(m, k, seed=81, spread=1))
    w = torch.ones(k, device="cuda").bfloat16()
    a, b = F.quantize_rows_mxfp4(x), F.quantize_rows_mxfp4(_rows(k, k, seed=82, spread=1))
    here = at(200704, (m, k // 2)), atoms(262144, m, k)  # codes and scales in the buffer
    here[0].copy_(a[0])
    here[1].copy_(a[1])
    h = at(400384, (m + 8, k), torch.bfloat16)
    s, lb = at(600064, (m, 32), torch.bfloat16), at(700416, (k, 32), torch.bfloat16)
    lora = dict(s=s, lb=lb, rank=32, num_adapters=1)
    bad = [
        lambda: F.quantize_rows_mxfp4(x, x4=at(1024, (m, k // 2))),
        lambda: F.quantize_rows_mxfp4(x, sf=atoms(102384, m, k)),
        lambda: F.quantize_rows_mxfp4(x, x4=at(200704, (m, k // 2)), sf=atoms(200704, m, k)),
        lambda: F.dequantize_mxfp4(*here, out=at(200704 - 4096, (m, k), torch.bfloat16)),
        lambda: F.dequantize_mxfp4(*here, out=at(262144 - 4096, (m, k), torch.bfloat16)),
        lambda: F.rmsnorm_mxfp4(x, w, 1e-5, out=at(512, (m, k), torch.bfloat16)),          # a row further down
        lambda: F.rmsnorm_mxfp4(x, w, 1e-5, x4=at(0, (m, k // 2))),
        lambda: F.rmsnorm_mxfp4(x, w, 1e-5, *here, out=at(200704, (m, k), torch.bfloat16)),
        lambda: F.rmsnorm_mxfp4(x, at(400384, (1, k), torch.bfloat16)[0], 1e-5, out=h[:m]),
        lambda: F.mxfp4_gemm(*here, *b, at(200704, (m, k), torch.bfloat16)),
        lambda: F.mxfp4_gemm(*a, *b, h[:m], epi=F.EPI_RESADD, residual=h[8:]),
        lambda: F.mxfp4_gemm(*a, *b, at(600064, (m, k), torch.bfloat16), **lora),
        lambda: F.mxfp4_gemm(*a, *b, at(700416, (m, k), torch.bfloat16), **lora),
        lambda: F.mxfp4_gemm(*a, here[0], here[1], at(200704, (m, m), torch.bfloat16)),      # the weight
        lambda: F.mxfp4_linear(x, *here, at(262144, (m, m), torch.bfloat16)),                # its scales
        lambda: F.mxfp4_gemm_swiglu(*here, *b, a4=at(200704, (m, k // 4))),
        lambda: F.mxfp4_gemm_swiglu(*here, *b, sf=atoms(262144, m, k // 2)),
        lambda: F.mxfp4_gemm_swiglu(*here, *b, act=at(200704, (m, k // 2), torch.bfloat16)),
        lambda: F.mxfp4_gemm_swiglu(*a, *b, a4=at(400384, (m, k // 4)), act=at(400384, (m, k // 2), torch.bfloat16)),
    ]
    keep = bytes_.clone()
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
            pytest.fail(f"call {i} was accepted")
    assert torch.equal(bytes_, keep)
    # columns of one buffer, rows behind one another, and the operand itself
    want = F.mxfp4_gemm(*a, *b)
    wide = torch.empty(m, 3 * k, dtype=torch.bfloat16, device="cuda")
    wide[:, :k] = x
    F.mxfp4_linear(wide[:, :k], *b, wide[:, k:2 * k])
    F.mxfp4_gemm(*a, *b, wide[:, 2 * k:], epi=F.EPI_RESADD, residual=wide[:, k:2 * k], scale=0.0)
    assert torch.equal(wide[:, :k], x) and torch.equal(wide[:, k:2 * k], want) and torch.equal(wide[:, 2 * k:], want)
    F.mxfp4_linear(wide[:, :k], *b, wide[:, :k])
    assert torch.equal(wide[:, :k], want)
    y = torch.cat((x, x))
    F.rmsnorm_mxfp4(y[:m], w, 1e-5, out=y[m:])
    assert torch.equal(y[m:], E.rmsnorm(x, w, 1e-5)) and torch.equal(y[:m], x)
    one = torch.empty(3 * k, dtype=torch.bfloat16, device="cuda").view(1, -1)
    one[:, k:2 * k] = x[:1]
    F.rmsnorm_mxfp4(one[:, k:2 * k], w, 1e-5, out=one[:, 2 * k:])
    assert torch.equal(one[:, 2 * k:], E.rmsnorm(x[:1], w, 1e-5))


# ------------------------------------------------------------- the CTA-pair kernel at sizes of the split kernel's
def _is_pair(m, n, k):
    from granite_switch_b200._native import native

    return native().mxfp4_gemm_plan(m, n, k)[0] == 1


@pytest.mark.parametrize("m", [3, 200, 1400])
@pytest.mark.parametrize("na,rank", [(64, 32), (3, 96)])
def test_pair_lora_limits(pair_always, m, na, rank):
    assert _is_pair(m, 1024, 2048)
    test_gemm_lora_limits(m, na, rank)


@pytest.mark.parametrize("m", [1, 3, 5, 130, 300, 1100])
@pytest.mark.parametrize("bounds", [[0, 640], [0, 1024, 1280, 1536], [0, 384, 512, 2176], [0, 128, 256, 384, 640]])
def test_pair_lora_slices(pair_always, m, bounds):
    """Bounds at odd multiples of 128 cut a 256-row weight tile in two slices of S."""
    assert _is_pair(m, bounds[-1], 512)
    test_gemm_lora_slices(m, bounds)


def _check_lora_residual(m, bounds, na, rank, k=1056):
    from granite_switch_b200.ops import gemm_fp4 as F

    n = bounds[-1]
    a, b = F.quantize_rows_mxfp4(_rows(m, k, seed=91)), F.quantize_rows_mxfp4(_rows(n, k, seed=92, spread=2))
    s, dirty, lb, mask = _lora_inputs(m, n, len(bounds) - 1, na, rank, seed=93)
    kw = dict(lb=lb, rank=rank, num_adapters=na, slice_bounds=bounds)
    h = torch.randn(m, n, device="cuda", generator=_gen(94)).to(torch.bfloat16)
    ref = h.double() + 0.5 * F.mxfp4_product_reference(*a, *b, s=s, **kw)
    tol = _acc_tol(*a, *b, extra=(s.double().abs().sum(1, keepdim=True) * lb.double().abs().max()))
    tol = 0.5 * tol + h.double().abs() * 2.0 ** -23
    _check(F.mxfp4_gemm(*a, *b, h, epi=F.EPI_RESADD, scale=0.5, residual=h, s=dirty, tile_mask=mask, **kw), ref, tol)


@pytest.mark.parametrize("m", [2, 129, 700])
@pytest.mark.parametrize("bounds,na,rank", [([0, 384, 1160], 2, 32), ([0, 896], 5, 96), ([0, 128, 264], 3, 64)])
def test_lora_with_residual(m, bounds, na, rank):
    _check_lora_residual(m, bounds, na, rank)


@pytest.mark.parametrize("m", [2, 129, 700])
@pytest.mark.parametrize("bounds,na,rank", [([0, 384, 1160], 2, 32), ([0, 896], 5, 96), ([0, 128, 264], 3, 64)])
def test_pair_lora_with_residual(pair_always, m, bounds, na, rank):
    assert _is_pair(m, bounds[-1], 1056)
    _check_lora_residual(m, bounds, na, rank)


def test_lora_products_of_the_rule_reach_the_pair_kernel():
    """A size that the rule itself gives to the pair kernel, with three slices, one of them cutting a tile."""
    assert _is_pair(2100, 1664, 1056)
    _check_lora_residual(2100, [0, 1152, 1408, 1664], 4, 32)


@pytest.mark.parametrize("m,i,h", [(1, 64, 64), (17, 192, 512), (4, 320, 512), (130, 1088, 256), (300, 512, 1056),
                                   (257, 192, 2080)])
@pytest.mark.parametrize("lora", [False, True])
def test_pair_swiglu(pair_always, m, i, h, lora):
    assert _is_pair(m, 2 * i, h)
    test_gemm_swiglu(m, i, h, lora)


@pytest.mark.parametrize("m", [2, 190, 1025])
def test_pair_mlp_block(pair_always, m):
    test_mlp_block(m)


def _check_swiglu_padding(m, i):
    from granite_switch_b200.ops import gemm_fp4 as F

    a = F.quantize_rows_mxfp4(_rows(m, 256, seed=95, spread=1))
    b = F.quantize_rows_mxfp4(_rows(2 * i, 256, seed=96, spread=1))
    a4 = torch.full((m + 3, i // 2), 0xAB, dtype=torch.uint8, device="cuda")
    sf = torch.full(((m + 127) // 128, (i + 255) // 256 * 2, 512), 0xFF, dtype=torch.uint8, device="cuda")
    F.mxfp4_gemm_swiglu(*a, *b, a4[:m], sf)
    byte = F.scale_bytes_from_atoms(sf, m, sf.shape[1] * 128)
    assert not byte[:, i // 32:].any() and (byte[:, :i // 32] < 255).all()
    rest = F.scale_bytes_from_atoms(sf, sf.shape[0] * 128, sf.shape[1] * 128)[m:]
    assert (rest == 0xFF).all() and (a4[m:] == 0xAB).all()  # rows behind the last one stay as they were


@pytest.mark.parametrize("m", [1, 100, 300])
@pytest.mark.parametrize("i", [64, 192, 320, 1088])
def test_swiglu_clears_the_scales_past_its_rows(m, i):
    _check_swiglu_padding(m, i)


@pytest.mark.parametrize("m", [1, 100, 300])
@pytest.mark.parametrize("i", [64, 192, 320, 1088])
def test_pair_swiglu_clears_the_scales_past_its_rows(pair_always, m, i):
    assert _is_pair(m, 2 * i, 256)
    _check_swiglu_padding(m, i)


@pytest.mark.parametrize("m,h", [(1000, 4128), (1003, 6144), (1000, 8192), (1001, 8224), (999, 12800), (900, 16384),
                                 (1500, 4224), (1500, 8256)])
@pytest.mark.parametrize("with_out", [False, True])
def test_rmsnorm_quantised_wide_rows(m, h, with_out):
    """Widths of every instantiation above 4096 columns, with more rows than CTAs: rings and sums are used again."""
    test_rmsnorm_quantised(m, h, with_out)


@pytest.mark.parametrize("h", [2048, 4096, 8192, 12800])
def test_rmsnorm_scales_of_old_buffers(h):
    """A caller's buffers: scales past the row's end are cleared, rows behind the last one stay as they were."""
    from granite_switch_b200.ops import gemm_fp4 as F

    m, h = 700, h - 96
    x = _rows(m, h, seed=97, spread=1)
    w = torch.ones(h, device="cuda").bfloat16()
    x4 = torch.full((m + 2, h // 2), 0xAB, dtype=torch.uint8, device="cuda")
    sf = torch.full(((m + 127) // 128, (h + 255) // 256 * 2, 512), 0xFF, dtype=torch.uint8, device="cuda")
    F.rmsnorm_mxfp4(x, w, 1e-5, x4[:m], sf)
    f4, fsf = F.rmsnorm_mxfp4(x, w, 1e-5)
    byte = F.scale_bytes_from_atoms(sf, sf.shape[0] * 128, sf.shape[1] * 128)
    assert torch.equal(x4[:m], f4) and (x4[m:] == 0xAB).all() and (byte[m:] == 0xFF).all()
    assert torch.equal(byte[:m, :h // 32], F.scale_bytes_from_atoms(fsf, m, h)) and not byte[:m, h // 32:].any()


def _check_strided_operands(m):
    """Codes, shrink output and expand weights that are columns of wider buffers, weights that are rows of a larger one,
    an output among other columns: as of contiguous copies, bit for bit, and nothing beside the output written."""
    from granite_switch_b200.ops import gemm_fp4 as F

    n, k, na, rank = 384, 1056, 3, 32
    a = F.quantize_rows_mxfp4(_rows(m, k, seed=101, spread=1))
    big = F.quantize_rows_mxfp4(_rows(n + 128, k, seed=102, spread=1))
    b = big[0][128:], big[1][1:]
    s, dirty, lb, mask = _lora_inputs(m, n, 2, na, rank, seed=103)
    kw = dict(tile_mask=mask, rank=rank, num_adapters=na, slice_bounds=[0, 128, n])

    def inside(t, fill):
        wide = torch.full((t.shape[0] + 2, t.shape[1] + 64), fill, dtype=t.dtype, device="cuda")
        wide[1:-1, 32:-32] = t
        return wide[1:-1, 32:-32]

    want = F.mxfp4_gemm(*a, b[0].clone(), b[1].clone(), s=dirty, lb=lb, **kw)
    out = torch.full((m + 2, n + 64), 5.0, dtype=torch.bfloat16, device="cuda")
    got = F.mxfp4_gemm(inside(a[0], 0xAB), a[1], inside(b[0], 0xCD), b[1], out[1:-1, 32:-32],
                       s=inside(dirty, float("nan")), lb=inside(lb, float("nan")), **kw)
    assert torch.equal(got, want)
    out[1:-1, 32:-32] = 5.0
    assert (out == 5.0).all()


@pytest.mark.parametrize("m", [1, 7, 200, 700])
def test_strided_operands(m):
    _check_strided_operands(m)


@pytest.mark.parametrize("m", [1, 7, 200, 700])
def test_pair_strided_operands(pair_always, m):
    _check_strided_operands(m)


def test_graphs_replayed_in_turn():
    """Two captured graphs and eager calls between them, each with a workspace of its own."""
    from granite_switch_b200.ops import gemm_fp4 as F

    b = F.quantize_rows_mxfp4(_rows(1024, 2080, seed=104, spread=1))
    xs = [_rows(m, 2080, seed=105 + m, spread=1) for m in (9, 600)]
    want = [F.mxfp4_linear(x, *b) for x in xs]
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(F.mxfp4_linear(F.dequantize_mxfp4(*F.quantize_rows_mxfp4(x)), *b))
    back = [F.mxfp4_linear(F.dequantize_mxfp4(*F.quantize_rows_mxfp4(x)), *b) for x in xs]
    for _ in range(4):
        for i in (0, 1):
            graphs[i].replay()
            assert torch.equal(F.mxfp4_linear(xs[1 - i], *b), want[1 - i])
            assert torch.equal(outs[i], back[i])
