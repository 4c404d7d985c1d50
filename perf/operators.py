"""The microscaled 4-bit (MXFP4) operators of :mod:`granite_switch_b200.ops.gemm_fp4` as measured cases.

A value is held as e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times a power of two shared by the 32 neighbours of a
block along K. The scale 2^e is the smallest power of two with max|x| <= 7 * 2^e, and a value rounds to the nearest
e2m1, ties to the even code; what is above 6 becomes 6, off by at most half of the last step.

Kinds of case:

* ``quant``        bf16 rows -> 4 bits -> the bf16 values they stand for
* ``linear``       bf16 rows times 4-bit weights, with the switched LoRA of several adapters or a scaled residual
* ``norm_linear``  RMSNorm and quantisation in one step, then the product
* ``mlp``          a decoder's whole MLP block: norm, gate/up product with SwiGLU, down product, scaled residual
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
RANK = 32


def listed():
    return [
        # one decode batch's rows, and the widest projection's input of a long prefill step
        dict(name="quant decode 16 rows", kind="quant", m=16, k=4096),
        dict(name="quant prefill 8192 rows", kind="quant", m=8192, k=12800),
        # rows of a shape no tile divides (a shard of an odd width)
        dict(name="quant ragged 1003 rows", kind="quant", m=1003, k=2080),
        # a single stream decoding: output projection into the residual
        dict(name="linear decode 1 row", kind="linear", m=1, n=4096, k=4096, adapters=0, residual=True),
        # a decode batch of twelve adapters' requests at the qkv projection
        dict(name="linear decode 128 lora", kind="linear", m=128, n=6144, k=4096, adapters=12, residual=False),
        # decode rows plus two short follow-up chunks at the down projection
        dict(name="linear mixed 222 rows", kind="linear", m=222, n=4096, k=12800, adapters=0, residual=True),
        # prefill chunks of many conversations, every adapter present
        dict(name="linear prefill 4096 lora", kind="linear", m=4096, n=6144, k=4096, adapters=12, residual=False),
        # the largest prefill step's down projection
        dict(name="linear prefill 8192", kind="linear", m=8192, n=4096, k=12800, adapters=0, residual=True),
        # the norm before the attention block: a small batch, and a ragged prefill chunk
        dict(name="norm linear 32 rows", kind="norm_linear", m=32, n=6144, k=4096),
        dict(name="norm linear 1537 rows", kind="norm_linear", m=1537, n=2048, k=2048),
        # whole MLP blocks: a decode batch, and a prefill step with LoRA on gate and up
        dict(name="mlp decode 64 rows", kind="mlp", m=64, h=4096, i=12800, adapters=0),
        dict(name="mlp prefill 2048 lora", kind="mlp", m=2048, h=2048, i=8192, adapters=4),
    ]


def _log(rng, lo, hi, step):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "norm_linear", "mlp"])
    if kind == "quant":
        return dict(kind=kind, m=_log(rng, 1, 8192, 1), k=_log(rng, 64, 12800, 32))
    if kind == "linear":
        adapters = rng.choice([0, 0, 1, 5, 12])
        m = _log(rng, 1, 8192, 1)
        k = _log(rng, 256, 12800, 32)
        n = _log(rng, 512, 6144, 128) if adapters else _log(rng, 256, 8192, 8)
        while m * n * k > 8192 * 4096 * 12800:
            m = max(1, m // 2)
        return dict(kind=kind, m=m, n=n, k=k, adapters=adapters, residual=rng.random() < 0.5)
    if kind == "norm_linear":
        return dict(kind=kind, m=_log(rng, 1, 4096, 1), n=_log(rng, 256, 6144, 8), k=_log(rng, 256, 8192, 32))
    return dict(kind=kind, m=_log(rng, 1, 2048, 1), h=_log(rng, 256, 4096, 64), i=_log(rng, 256, 12800, 64),
                adapters=rng.choice([0, 0, 3]))


# ---------------------------------------------------------------------------------------------- the 4-bit format

def _pow2(e, like):
    """Exact 2^e of whole numbers, in `like`'s type."""
    return ((e.long() + 1023) << 52).view(torch.float64).to(like.dtype)


def _blocks(v):
    """Values ``[rows, K]`` -> (e2m1 values, exponents): ``[rows, K / 32, 32]`` and ``[rows, K / 32, 1]``."""
    b = v.reshape(v.shape[0], -1, 32)
    mant, ex = torch.frexp(b.abs().amax(2, keepdim=True))
    e = torch.where(mant <= 0.875, ex - 3, ex - 2).clamp(min=-127)
    y = b * _pow2(-e, b)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    q = ((a / step).round() * step).clamp(max=6.0)
    return torch.copysign(q, y), e


def _rounded(v):
    """The values that 4 bits keep of ``[rows, K]``."""
    q, e = _blocks(v)
    return (q * _pow2(e, q)).reshape(v.shape)


def _pack(v):
    """``[rows, K]`` -> (two codes a byte, the lower K in the low nibble; scale bytes in 512-byte atoms of 128 rows
    x 4 blocks: row r's four bytes at 16 (r % 32) + 4 (r // 32), K padded to 256)."""
    q, e = _blocks(v)
    rows, k = v.shape
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).reshape(rows, k)
    tiles, kb = -(-rows // 128), -(-k // 256) * 2
    byte = torch.zeros(tiles * 128, kb * 4, dtype=torch.uint8, device=v.device)
    byte[:rows, :k // 32] = (e.squeeze(2) + 127).to(torch.uint8)
    atoms = byte.view(tiles, 4, 32, kb, 4).permute(0, 3, 2, 1, 4).reshape(tiles, kb, 512)
    return code[:, 0::2] | (code[:, 1::2] << 4), atoms.contiguous()


def _unpack(w4, sf):
    """fp32 ``[rows, K]`` of packed codes and scale atoms."""
    rows, k = w4.shape[0], w4.shape[1] * 2
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=w4.device)
    v = table[torch.stack((w4 & 15, w4 >> 4), dim=2).reshape(rows, k).int()]
    tiles, kb = sf.shape[0], sf.shape[1]
    byte = sf.view(tiles, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * 128, kb * 4)[:rows, :k // 32]
    return (v.view(rows, k // 32, 32) * _pow2(byte.int() - 127, v).unsqueeze(2)).view(rows, k)


# ---------------------------------------------------------------------------------------------- inputs

def _slices(n):
    """A query-sized slice and two smaller ones, as a fused qkv projection has them."""
    a, b = n // 3 * 2 // 128 * 128, n // 6 // 128 * 128
    return [0, a, a + b, n] if a and b else [0, n]


def _lora(m, n, adapters, slices, g):
    """Per-row adapters in runs (requests), the masked shrink output, its expand weights and the 128-row bit masks.
    Columns of adapters that no row of a 128-row tile uses are never written by the shrink: they hold old values."""
    runs = torch.randint(0, adapters + 1, (-(-m // 16),), generator=g, device=DEV)
    row_adapter = runs.repeat_interleave(16)[:m].contiguous()
    cols = adapters * RANK
    s = torch.randn(m, slices * cols, generator=g, device=DEV)
    col = (torch.arange(slices * cols, device=DEV) // RANK) % adapters + 1
    tiles = -(-m // 128)
    padded = torch.zeros(tiles * 128, dtype=torch.long, device=DEV)
    padded[:m] = row_adapter
    present = (padded.view(tiles, 128, 1) == torch.arange(1, adapters + 1, device=DEV)).any(1)
    mask = (present.long() << torch.arange(adapters, device=DEV)).sum(1)
    here = present.repeat_interleave(128, 0)[:m][:, col - 1]
    keep = col == row_adapter[:, None]
    s = torch.where(here & ~keep, torch.zeros_like(s), s).to(torch.bfloat16)
    lb = (torch.randn(n, cols, generator=g, device=DEV) * 0.02).to(torch.bfloat16)
    return dict(s=s, lb=lb, mask=mask, row_adapter=row_adapter)


def _rows(m, k, g):
    """Hidden states: unit normals with a few channels that run an order of magnitude larger."""
    x = torch.randn(m, k, generator=g, device=DEV)
    big = torch.rand(k, generator=g, device=DEV) < 0.01
    return torch.where(big, x * 12, x).to(torch.bfloat16)


def _weight(n, k, g):
    return _pack((torch.randn(n, k, generator=g, device=DEV) * 0.02).to(torch.bfloat16).float())


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    st = dict(case=c)
    if c["kind"] == "mlp":
        h, i, m = c["h"], c["i"], c["m"]
        st["x"] = _rows(m, h, g)
        st["norm"] = (1 + 0.1 * torch.randn(h, generator=g, device=DEV)).to(torch.bfloat16)
        # gate and up rows alternate in runs of 64
        st["gu"], st["gu_sf"] = _weight(2 * i, h, g)
        st["down"], st["down_sf"] = _weight(h, i, g)
        st["scale"] = 0.22
        if c["adapters"]:
            st.update(_lora(m, 2 * i, c["adapters"], 2, g))
            # an expand row uses its own half of the columns: the gate's, then the up's
            lb = st["lb"].view(i // 64, 2, 64, -1)
            full = torch.zeros(i // 64, 2, 64, 2, lb.shape[3], dtype=lb.dtype, device=DEV)
            full[:, 0, :, 0], full[:, 1, :, 1] = lb[:, 0], lb[:, 1]
            st["lb"] = full.view(2 * i, -1)
        return st
    st["x"] = _rows(c["m"], c["k"], g)
    if c["kind"] == "quant":
        return st
    st["w4"], st["sf"] = _weight(c["n"], c["k"], g)
    st["scale"] = 1.0
    if c["kind"] == "norm_linear":
        st["norm"] = (1 + 0.1 * torch.randn(c["k"], generator=g, device=DEV)).to(torch.bfloat16)
        return st
    if c["residual"]:
        st["residual"] = torch.randn(c["m"], c["n"], generator=g, device=DEV).to(torch.bfloat16)
        st["scale"] = 0.22
    if c["adapters"]:
        st["bounds"] = _slices(c["n"])
        st.update(_lora(c["m"], c["n"], c["adapters"], len(st["bounds"]) - 1, g))
    return st


# ---------------------------------------------------------------------------------------------- one pass

def _own_run(st):
    from granite_switch_b200.ops import gemm_fp4 as F

    c, x = st["case"], st["x"]
    lora = {}
    if c.get("adapters"):
        lora = dict(s=st["s"], lb=st["lb"], tile_mask=st["mask"], rank=RANK, num_adapters=c["adapters"])
    if c["kind"] == "quant":
        return F.dequantize_mxfp4(*F.quantize_rows_mxfp4(x))
    if c["kind"] == "linear":
        if lora:
            lora["slice_bounds"] = st["bounds"]
        epi = F.EPI_RESADD if c["residual"] else F.EPI_STORE
        return F.mxfp4_linear(x, st["w4"], st["sf"], epi=epi, scale=st["scale"], residual=st.get("residual"), **lora)
    x4, sf = F.rmsnorm_mxfp4(x, st["norm"], EPS)
    if c["kind"] == "norm_linear":
        return F.mxfp4_gemm(x4, sf, st["w4"], st["sf"])
    a4, asf = F.mxfp4_gemm_swiglu(x4, sf, st["gu"], st["gu_sf"], **lora)
    return F.mxfp4_gemm(a4, asf, st["down"], st["down_sf"], epi=F.EPI_RESADD, scale=st["scale"], residual=x)


def _plain_norm(x, w):
    v = x.double()
    return v * (v.square().mean(1, keepdim=True) + EPS).rsqrt() * w.double()


def _plain_s(st):
    """The shrink output with every column but the row's own adapter's taken as zero."""
    cols = st["s"].shape[1]
    col = (torch.arange(cols, device=DEV) // RANK) % st["case"]["adapters"] + 1
    return torch.where(col == st["row_adapter"][:, None], st["s"].float(), 0.0)


def _plain_run(st):
    c, x = st["case"], st["x"]
    if c["kind"] == "quant":
        return _rounded(x.float()).to(torch.bfloat16)
    if c["kind"] == "mlp":
        acc = _rounded(_plain_norm(x, st["norm"])).float() @ _unpack(st["gu"], st["gu_sf"]).t()
        if c["adapters"]:
            acc += _plain_s(st) @ st["lb"].float().t()
        acc = acc.view(c["m"], -1, 2, 64)
        gate, up = acc[:, :, 0], acc[:, :, 1]
        act = (gate / (1 + torch.exp(-gate)) * up).reshape(c["m"], -1)
        y = _rounded(act) @ _unpack(st["down"], st["down_sf"]).t()
        return (x.float() + y * st["scale"]).to(torch.bfloat16)
    v = _rounded(_plain_norm(x, st["norm"])).float() if c["kind"] == "norm_linear" else _rounded(x.float())
    acc = v @ _unpack(st["w4"], st["sf"]).t()
    if c.get("adapters"):
        s, cols = _plain_s(st), st["lb"].shape[1]
        b = st["bounds"]
        delta = [s[:, q * cols:(q + 1) * cols] @ st["lb"][b[q]:b[q + 1]].float().t() for q in range(len(b) - 1)]
        acc += torch.cat(delta, 1)
    acc *= st["scale"]
    if c.get("residual"):
        acc += st["residual"].float()
    return acc.to(torch.bfloat16)


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ---------------------------------------------------------------------------------------------- work and 64 bits

def _w_bytes(n, k):
    return n * k / 2 + n * k / 32


def work(case):
    c, m = case, case["m"]
    if c["kind"] == "quant":
        return {"bytes": 4.0 * m * c["k"], "flops": 0.0}
    if c["kind"] == "mlp":
        h, i, a = c["h"], c["i"], c["adapters"]
        b = 4.0 * m * h + 2 * h + _w_bytes(2 * i, h) + _w_bytes(h, i)
        b += a and 2.0 * (m * 2 * a * RANK + 2 * i * a * RANK)
        return {"bytes": b, "flops": 6.0 * m * h * i + (a and 2.0 * m * 2 * i * RANK)}
    n, k, a = c["n"], c["k"], c.get("adapters", 0)
    b = 2.0 * m * (k + n) + _w_bytes(n, k) + (2.0 * m * n if c.get("residual") else 0)
    slices = len(_slices(n)) - 1 if a else 0
    b += a and 2.0 * (m * slices * a * RANK + n * a * RANK)
    return {"bytes": b, "flops": 2.0 * m * n * k + (a and 2.0 * m * n * RANK)}


_TABLE = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64)  # by scale byte


def _exact_values(v):
    """float64 ``[rows, K]`` -> what 4 bits keep, by counting the rounding borders that each value is above."""
    b = v.reshape(v.shape[0], v.shape[1] // 32, 32)
    top = b.abs().amax(2)
    # the exponent field of a positive double; 7 = 1.75 * 2^2
    field, frac = top.view(torch.int64) >> 52, top.view(torch.int64) & ((1 << 52) - 1)
    e = torch.where(top > 0, field - 1023 - 2 + (frac > 3 << 50).long(), -127).clamp(min=-127)
    power = _TABLE.to(v.device)[e + 127].unsqueeze(2)
    y = b / power
    a, out = y.abs(), torch.zeros_like(b)
    # (border, step up, whether the border itself goes up: to the even code)
    for at, up, tie in ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False), (1.75, 0.5, True), (2.5, 1.0, False),
                        (3.5, 1.0, True), (5.0, 2.0, False)):
        out += up * ((a >= at) if tie else (a > at)).double()
    return (out * y.sign() * power).reshape(v.shape)


def _exact_weight(w4, sf):
    n, k = w4.shape[0], 2 * w4.shape[1]
    mag = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=w4.device) / 2
    out = torch.empty(n, k, dtype=torch.float64, device=w4.device)
    for half in (0, 1):
        code = (w4.long() >> (4 * half)) & 15
        out[:, half::2] = mag[code & 7] * (1 - 2 * (code >> 3)).double()
    r = torch.arange(n, device=w4.device)[:, None]
    blk = torch.arange(k // 32, device=w4.device)[None]
    byte = sf[r // 128, blk // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + blk % 4]
    return out * _TABLE.to(w4.device)[byte.long()].repeat_interleave(32, dim=1)


def _exact_delta(st, bounds):
    """Row by row of adapters: ``s`` of the row's own adapter against that adapter's expand columns."""
    c = st["case"]
    s, lb, cols = st["s"].double(), st["lb"].double(), c["adapters"] * RANK
    out = torch.zeros(c["m"], lb.shape[0], dtype=torch.float64, device=s.device)
    for a in range(c["adapters"]):
        rows = (st["row_adapter"] == a + 1).nonzero().squeeze(1)
        for q, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
            left = s[rows, q * cols + a * RANK:q * cols + (a + 1) * RANK]
            out[rows, lo:hi] = left @ lb[lo:hi, a * RANK:(a + 1) * RANK].t()
    return out


def exact(case, seed):
    st, c = prepare(case, seed), case
    x = st["x"].double()
    if "norm" in st:
        x = x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * st["norm"].double()
    v = _exact_values(x)
    if c["kind"] == "quant":
        return v
    if c["kind"] == "mlp":
        gu = v @ _exact_weight(st["gu"], st["gu_sf"]).t()
        half = torch.arange(2 * c["i"], device=x.device) // 64 % 2
        if c["adapters"]:
            lb, cols = st["lb"], c["adapters"] * RANK
            for q in (0, 1):
                sub = dict(st, s=st["s"][:, q * cols:(q + 1) * cols], lb=lb[:, q * cols:(q + 1) * cols])
                gu += _exact_delta(sub, [0, 2 * c["i"]])
        gate, up = gu[:, half == 0], gu[:, half == 1]
        act = _exact_values(gate * torch.sigmoid(gate) * up)
        return st["x"].double() + st["scale"] * (act @ _exact_weight(st["down"], st["down_sf"]).t())
    y = v @ _exact_weight(st["w4"], st["sf"]).t()
    if c.get("adapters"):
        y += _exact_delta(st, st["bounds"])
    y = y * st["scale"]
    return y + st["residual"].double() if c.get("residual") else y
