"""Linear layers in microscaled 4-bit floating point (MXFP4) with the bf16 switched-LoRA
expand fused: quantisers, products and their fp64 oracles.

32 neighbours along K share a scale ``2^e`` (a byte ``e + 127``), the smallest power of two
with ``max|x| <= 7 * 2^e``; each value is the e2m1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
sign) nearest to ``x / 2^e``, ties to the even code, and what is above 6 becomes 6 (off by at
most 1, half of the last step). e is at most 125, so finite values stay finite in bf16 (what is
above ``7 * 2^125`` saturates). A block that is not finite gets the byte 255 and stands for
NaN. K is a multiple of 32.

An ``[M, K]`` matrix is held as codes ``[M, K / 2]`` (two a byte, the lower K in the low
nibble) and scale atoms ``[ceil(M / 128), 2 ceil(K / 256), 512]``: byte
``16 (r % 32) + 4 (r // 32) + j`` of an atom is row ``r``'s scale for the 32 values at
``32 j`` of the atom's 128; bytes of blocks past K are 0, bytes of rows past M in the last atom
are not written (compare scales through :func:`scale_bytes_from_atoms`). Activations and weights
have the same format, so :func:`quantize_rows_mxfp4` serves both. Where a call allocates both,
codes and scales are views of one storage: keeping or saving either keeps both (``clone`` parts
them).

Products are summed in fp32 by the tensor core and rounded once, in the epilogue. An output
that shares memory with an operand is refused, but for the few that may be an operand itself
(the residual, the norm's ``x``, the linear's ``x``).
"""
from __future__ import annotations

import torch

from .._native import err_buffer, native

EPI_STORE = 0
EPI_RESADD = 1
BLOCK = 32
SWIGLU_TILE = 128  # gate/up rows of a packed weight alternate in runs of 64
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize_rows_mxfp4(x: torch.Tensor, x4: torch.Tensor | None = None, sf: torch.Tensor | None = None):
    """``x [M, K]`` bf16 -> (codes ``[M, K / 2]``, scale atoms), on the GPU."""
    return native().quantize_mxfp4(x, x4, sf)


def dequantize_mxfp4(x4: torch.Tensor, sf: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The bf16 values ``[M, K]`` that codes and scale atoms stand for (exact), on the GPU."""
    return native().dequantize_mxfp4(x4, sf, out)


def rmsnorm_mxfp4(x: torch.Tensor, w: torch.Tensor, eps: float, x4: torch.Tensor | None = None,
                  sf: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """RMSNorm of ``x [M, H]`` bf16 and its quantisation in one pass: ``x w / sqrt(mean(x^2) + eps)``
    in fp32, rounded once, to 4 bits. ``out [M, H]`` also receives the bf16 rows that
    :func:`ops.elementwise.rmsnorm` writes (the LoRA shrink reads them). H is at most 16384."""
    return native().rmsnorm_mxfp4(x, w, eps, x4, sf, out)


def mxfp4_gemm(x4, sfx, w4, sfw, out=None, *, epi: int = EPI_STORE, scale: float = 1.0, residual=None, s=None,
               lb=None, tile_mask=None, rank: int = 0, num_adapters: int = 0, slice_bounds=None):
    """``out [M, N]`` bf16 ``= (x4 @ w4.T + S @ LB.T) * scale``, plus ``residual`` with
    ``EPI_RESADD`` (``out`` may be the residual itself). N is a multiple of 8.

    The LoRA operands follow :func:`ops.gemm.switched_gemm` (bf16, ``rank`` a multiple of 32,
    ``s`` the masked shrink output, ``tile_mask`` the adapters present per 128 rows); slice
    bounds are multiples of 128.
    """
    return native().mxfp4_gemm(x4, sfx, w4, sfw, out, epi, scale, residual, s, lb, tile_mask, rank, num_adapters,
                               slice_bounds, err_buffer(x4.device))


def mxfp4_linear(x, w4, sfw, out=None, *, epi: int = EPI_STORE, scale: float = 1.0, residual=None, s=None, lb=None,
                 tile_mask=None, rank: int = 0, num_adapters: int = 0, slice_bounds=None):
    """:func:`mxfp4_gemm` of bf16 rows ``x [M, K]``, quantised into a workspace of the call."""
    return native().mxfp4_linear(x, w4, sfw, out, epi, scale, residual, s, lb, tile_mask, rank, num_adapters,
                                 slice_bounds, err_buffer(x.device))


def mxfp4_gemm_swiglu(x4, sfx, w4, sfw, a4=None, sf=None, act=None, *, s=None, lb=None, tile_mask=None,
                      rank: int = 0, num_adapters: int = 0):
    """``silu(gate) * up`` of the gate/up product ``[M, 2 I]``, quantised in the epilogue:
    (codes ``[M, I / 2]``, scale atoms); ``act [M, I]`` also receives it as bf16. The rows of
    ``w4`` alternate in runs of 64 (``models.packing.interleave_gate_up(w, SWIGLU_TILE)``), I is
    a multiple of 64. With LoRA ``s`` holds the gate's columns, then the up's, and ``lb`` is
    :func:`swiglu_lora_b` of the interleaved expand weights."""
    return native().mxfp4_gemm_swiglu(x4, sfx, w4, sfw, a4, sf, act, s, lb, tile_mask, rank, num_adapters,
                                      err_buffer(x4.device))


def swiglu_lora_b(lb: torch.Tensor) -> torch.Tensor:
    """Interleaved expand weights ``[2 I, cols]`` -> ``[2 I, 2 cols]``: gate rows in the first half of
    the columns and up rows in the second, zero elsewhere (load time; both halves then run
    through one accumulator tile)."""
    n, cols = lb.shape
    v = lb.reshape(n // SWIGLU_TILE, 2, SWIGLU_TILE // 2, cols)
    out = torch.zeros(*v.shape[:3], 2, cols, dtype=lb.dtype, device=lb.device)
    out[:, 0, :, 0] = v[:, 0]
    out[:, 1, :, 1] = v[:, 1]
    return out.reshape(n, 2 * cols)


# ---------------------------------------------------------------- oracles (any device)
def _pow2(e: torch.Tensor) -> torch.Tensor:
    """Exact fp64 ``2^e`` of whole numbers (``torch.ldexp`` may be off by an ulp on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scale_bytes(amax: torch.Tensor) -> torch.Tensor:
    mant, ex = torch.frexp(amax.double())
    e = torch.where(mant <= 0.875, ex - 3, ex - 2).clamp(-127, 125)
    byte = torch.where(amax > 0, e + 127, torch.zeros_like(e))
    return torch.where(torch.isfinite(amax), byte, torch.full_like(byte, 255)).to(torch.uint8)


def quantize_rows_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """PyTorch statement of :func:`quantize_rows_mxfp4` for rows of any type (same bytes)."""
    m, k = x.shape
    b = x.double().view(m, k // BLOCK, BLOCK)
    byte = _scale_bytes(b.abs().amax(2))
    y = b * _pow2(127 - byte.long().unsqueeze(2))
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = ((a / step).round() * step).clamp(max=6.0)
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4))
    nan = (byte == 255).unsqueeze(2)
    code = torch.where(nan, 0.0, code).to(torch.uint8) | ((torch.signbit(y) & ~nan).to(torch.uint8) << 3)
    code = code.view(m, k)
    tiles, kt = (m + 127) // 128, (k + 255) // 256 * 2
    full = torch.zeros(tiles * 128, kt * 4, dtype=torch.uint8, device=x.device)
    full[:m, : k // BLOCK] = byte
    sf = full.view(tiles, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(tiles, kt, 512)
    return code[:, 0::2] | (code[:, 1::2] << 4), sf.contiguous()


def scale_bytes_from_atoms(sf: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """Scale bytes ``[rows, K / 32]`` of atoms."""
    tiles, kt = sf.shape[0], sf.shape[1]
    return sf.view(tiles, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * 128, kt * 4)[:rows, : k // BLOCK]


def dequantize_reference(x4: torch.Tensor, sf: torch.Tensor) -> torch.Tensor:
    """fp64 values of codes and scale atoms."""
    m, k = x4.shape[0], x4.shape[1] * 2
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=x4.device)
    v = table[torch.stack((x4 & 15, x4 >> 4), dim=2).view(m, k).long()]
    byte = scale_bytes_from_atoms(sf, m, k)
    scale = torch.where(byte == 255, float("nan"), _pow2(byte.long() - 127))
    return (v.view(m, k // BLOCK, BLOCK) * scale.unsqueeze(2)).view(m, k)


def mxfp4_product_reference(x4, sfx, w4, sfw, *, s=None, lb=None, rank: int = 0, num_adapters: int = 0,
                            slice_bounds=None) -> torch.Tensor:
    """fp64 accumulator ``[M, N]`` of :func:`mxfp4_gemm` before its epilogue (``s`` zero outside each
    row's own adapter). For SwiGLU pass the doubled ``lb`` and leave ``slice_bounds`` out."""
    acc = dequantize_reference(x4, sfx) @ dequantize_reference(w4, sfw).t()
    if s is not None and lb is not None and num_adapters > 0:
        n, cols = w4.shape[0], lb.shape[1]
        bounds = slice_bounds or [0, n]
        for i in range(len(bounds) - 1):
            rows = slice(bounds[i], bounds[i + 1])
            acc[:, rows] += s[:, i * cols:(i + 1) * cols].double() @ lb[rows].double().t()
    return acc


def swiglu_reference(acc: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` of an interleaved gate/up accumulator."""
    v = acc.view(acc.shape[0], -1, 2, SWIGLU_TILE // 2)
    return (torch.nn.functional.silu(v[:, :, 0]) * v[:, :, 1]).reshape(acc.shape[0], -1)


__all__ = ["quantize_rows_mxfp4", "dequantize_mxfp4", "rmsnorm_mxfp4", "mxfp4_gemm", "mxfp4_linear",
           "mxfp4_gemm_swiglu", "swiglu_lora_b", "quantize_rows_reference", "dequantize_reference",
           "scale_bytes_from_atoms", "mxfp4_product_reference", "swiglu_reference", "EPI_STORE", "EPI_RESADD", "SWIGLU_TILE"]
