"""o_proj for decode: ``y[tokens, hidden] = x[tokens, K] @ w[hidden, K]^T``.

CUDA tensors run the tcgen05 / TMEM kernel (``csrc/oproj_gemm.cu``); CPU tensors use a plain
matmul.  In the reference this is vLLM's cuBLAS linear layer.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _ext
from ..utils import env as _env


def oproj(x: torch.Tensor, w, *, splits: int = 0, library: Optional[bool] = None) -> torch.Tensor:
    """``x [tokens, K]`` bf16, ``w [hidden, K]`` bf16 (``nn.Linear`` weight layout) -> bf16 ``[tokens, hidden]``.

    ``splits``: 0 lets the library pick (stream-K over all SMs when the plain grid would leave
    some idle), -1 forces the stream-K kernel, ``n >= 1`` forces the plain kernel with ``n`` K splits.

    The hand-written kernel is built for decode: few tokens, bound by streaming W once (swap-AB, one 128-row slab
    of W per CTA, every CTA reads all of x); above 16 tokens it splits K finely and sums the partials in a second
    kernel.  Every slab's CTA re-reads x, so with many tokens cuBLAS is faster (measured on B200 inside CUDA graphs,
    hidden 8192, K = 8192 / 4096 / 2048 / 1024, packed weights under programmatic launch against cuBLAS: 8 tokens
    25.0 / 14.6 / 9.3 / 5.6 us against 23.8 / 13.4 / 7.8 / 5.6, 32 tokens 27.7 / 17.5 / 12.7 / 6.9 against
    25.6 / 14.4 / 8.2 / 5.8, 128 tokens 35.8 / 22.8 / 16.7 / 11.0 against 25.7 / 14.1 / 8.6 / 6.3; launches that do not
    overlap take about 3 us more).  So with ``splits=0`` and a plain weight matrix calls of 32 tokens or more go to
    ``torch.nn.functional.linear``; ``library=False`` (or ``HELIX_A2A_OPROJ_LIBRARY=0``) keeps the hand-written
    kernel for every size.  Packed weights always use the hand-written kernel (the plain matrix is not kept).

    ``w`` may also be an :class:`Int4OprojWeight` (``splits`` and ``library`` have no meaning then): bf16 or fp16 ``x`` like its
    scales, a quarter of the bytes.  That pays up to some 100 tokens: a launch has at most 128, each reads and unpacks all weights, and with 8192 x 8192
    1024 tokens take 212 us where 16-bit weights take 90.  A group's products are added up in fp32 before its scale, so bf16 values beyond 10^35 overflow.
    """
    if isinstance(w, Int4OprojWeight):
        if not x.is_cuda:
            return (x.float() @ unpack_weight_int4(w).t()).to(x.dtype)
        if x.dtype != w.dtype:
            raise RuntimeError(f"x is {x.dtype}, the weight's scales are {w.dtype}")
        return _ext.ops().oproj_int4(x, w.packed, w.hidden, w.K, w.group, w.zeros)
    if isinstance(w, PackedOprojWeight):
        if not x.is_cuda:
            return (x.float() @ unpack_weight(w).float().t()).to(x.dtype)
        return _ext.ops().oproj_packed(x, w.packed, w.hidden, w.K, max(splits, 0))
    if not x.is_cuda:
        return (x.float() @ w.float().t()).to(x.dtype)
    if splits == 0 and library is not False and library_gemm_pays(x.shape[0], w.shape[1]):
        return torch.nn.functional.linear(x, w)
    return _ext.ops().oproj(x, w, splits)


def library_gemm_pays(tokens: int, K: int) -> bool:
    """The measured crossover between the decode kernel and cuBLAS (see :func:`oproj`)."""
    del K          # the crossover does not depend on it: 32 tokens at K = 1024 ... 8192
    return tokens >= 32 and _env.oproj_library()


class PackedOprojWeight:
    """A ``[hidden, K]`` bf16 weight re-laid for the o_proj kernel: per 128-row slab, ``K / 64`` atoms
    (padded with zeros to a multiple of 4) of ``128 rows x 128 bytes``, each atom stored exactly as the
    tensor core reads it from shared memory (16-byte chunk ``c`` of row ``r`` sits at chunk ``c ^ (r & 7)``).
    One pipeline stage of the kernel is then a single contiguous bulk copy instead of several strided
    tensor copies that open a DRAM page for 128 bytes at a time.  Weights are static, so this is done once."""

    def __init__(self, packed: torch.Tensor, hidden: int, K: int):
        self.packed, self.hidden, self.K = packed, hidden, K

    @property
    def shape(self):
        return (self.hidden, self.K)


def packed_atoms(K: int) -> int:
    return ((K + 63) // 64 + 3) // 4 * 4


def prepack_weight(w: torch.Tensor) -> PackedOprojWeight:
    """``w [hidden, K]`` bf16 (any row stride, e.g. a CP rank's column slice of W_o) -> ``PackedOprojWeight``."""
    hidden, K = w.shape
    if hidden % 128 or K % 64 or w.dtype != torch.bfloat16:
        raise ValueError("prepack_weight needs a bfloat16 [hidden % 128 == 0, K % 64 == 0] matrix")
    na = packed_atoms(K)
    wp = torch.zeros(hidden, na * 64, dtype=w.dtype, device=w.device)
    wp[:, :K] = w
    # [slab, row, atom, chunk, 8 elements] -> [slab, atom, row, chunk', 8] with chunk' = chunk ^ (row & 7)
    t = wp.view(hidden // 128, 128, na, 8, 8).permute(0, 2, 1, 3, 4).contiguous()
    r = torch.arange(128, device=w.device).view(1, 1, 128, 1, 1)
    c = torch.arange(8, device=w.device).view(1, 1, 1, 8, 1)
    src_chunk = (c ^ (r & 7)).expand(t.shape[0], na, 128, 8, 8)      # position c' holds source chunk c' ^ (r & 7)
    t = torch.gather(t, 3, src_chunk.contiguous())
    return PackedOprojWeight(t.contiguous().view(torch.uint8).reshape(-1), hidden, K)


def unpack_weight(pw: PackedOprojWeight) -> torch.Tensor:
    """Inverse of ``prepack_weight`` (tests, debugging)."""
    na = packed_atoms(pw.K)
    t = pw.packed.view(torch.bfloat16).view(pw.hidden // 128, na, 128, 8, 8)
    r = torch.arange(128, device=t.device).view(1, 1, 128, 1, 1)
    c = torch.arange(8, device=t.device).view(1, 1, 1, 8, 1)
    t = torch.gather(t, 3, (c ^ (r & 7)).expand_as(t).contiguous())   # the swizzle is its own inverse
    return t.permute(0, 2, 1, 3, 4).reshape(pw.hidden, na * 64)[:, :pw.K].contiguous()


class Int4OprojWeight:
    """A ``[hidden, K]`` weight in 4 bits with one scale (and zero point) per row and ``group`` columns: ``(q - z) * s`` with ``q`` and
    ``z`` in 0 .. 15, ``z = 8`` where there are no zero points.  Laid out for the kernel (``csrc/oproj_int4.h``): a record per 128 rows
    (those behind ``hidden`` are zeros) and 128 columns, its nibbles in the order in which they become matrix operands, then its scales and
    zero points.  Made by :func:`quantize_weight_int4` from a matrix or by :func:`pack_weight_int4` from a checkpoint's arrays, once, at
    load time."""

    def __init__(self, packed: torch.Tensor, hidden: int, K: int, group: int, dtype: torch.dtype, zeros: bool):
        self.packed, self.hidden, self.K, self.group, self.dtype, self.zeros = packed, hidden, K, group, dtype, zeros

    @property
    def shape(self):
        return (self.hidden, self.K)

    def records(self):
        """Views of the packed bytes, 128 columns at a time: nibbles ``[slabs, 8 tiles, blocks of 32 columns, 16 rows, 16 bytes]``, scales
        ``[slabs, groups, 8 tiles, 8, 2]`` and zero points of that shape (or ``None``)."""
        slabs, at = -(-self.hidden // 128), 0
        rows = self.packed.view(slabs, -1)
        for k in range(0, self.K, 128):
            k1 = min(k + 128, self.K)
            blocks, groups = (k1 - k) // 32, (k1 - k) // self.group
            q, at = rows[:, at:at + blocks * 2048].unflatten(1, (8, blocks, 16, 16)), at + blocks * 2048
            s, at = rows[:, at:at + groups * 256].view(self.dtype).unflatten(1, (groups, 8, 8, 2)), at + groups * 256
            z = None
            if self.zeros:
                z, at = rows[:, at:at + groups * 128].unflatten(1, (groups, 8, 8, 2)), at + groups * 128
            yield slice(k, k1), q, s, z


def pack_weight_int4(qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> Int4OprojWeight:
    """``qweight [hidden, K / 2]`` uint8 (column ``2 i`` in the low half of byte ``i``), ``scales [hidden, K / group]`` bf16 or fp16 and
    ``zeros`` uint8 of the same shape (values 0 .. 15; ``None``: 8 everywhere) -> :class:`Int4OprojWeight`.  ``group`` is 32, 64 or 128."""
    hidden, K = qweight.shape[0], 2 * qweight.shape[1]
    group = K // max(scales.shape[-1], 1)
    if qweight.dtype != torch.uint8 or scales.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("pack_weight_int4 needs uint8 nibbles and bfloat16 or float16 scales")
    if group not in (32, 64, 128) or scales.shape != (hidden, K // group) or K % 64 or K % group or not hidden or not K:
        raise ValueError("pack_weight_int4 needs K % 64 == 0 and scales [hidden, K / group], group 32, 64 or 128")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("zeros must be uint8 of the scales' shape")
    if zeros is not None and int(zeros.max()) > 15:
        raise ValueError("zeros must be 0 .. 15")
    slabs = -(-hidden // 128)

    def in_slabs(t):
        t = torch.nn.functional.pad(t, (0, 0, 0, slabs * 128 - hidden)) if hidden % 128 else t
        return t.view(slabs, 128, -1)

    q = torch.stack([qweight & 15, qweight >> 4], -1).view(hidden, K)
    # slab, tile, row, block of 32, word, pair, column of the pair -> slab, tile, block, row, word, nibble = pair + 4 * column
    q = in_slabs(q).view(slabs, 8, 16, K // 32, 4, 4, 2).permute(0, 1, 3, 2, 4, 6, 5).reshape(slabs, 8, K // 32, 16, 16, 2)
    q = q[..., 0] | (q[..., 1] << 4)
    # slab, tile, upper or lower eight rows, row, group -> slab, group, tile, row, half
    s, z = (None if t is None else in_slabs(t).view(slabs, 8, 2, 8, K // group).permute(0, 4, 1, 3, 2) for t in (scales, zeros))
    packed = torch.empty(slabs * (K * 64 + K // group * (256 if zeros is None else 384)), dtype=torch.uint8, device=qweight.device)
    w = Int4OprojWeight(packed, hidden, K, group, scales.dtype, zeros is not None)
    for cols, to_q, to_s, to_z in w.records():
        to_q.copy_(q[:, :, cols.start // 32:cols.stop // 32])
        to_s.copy_(s[:, cols.start // group:cols.stop // group])
        if z is not None:
            to_z.copy_(z[:, cols.start // group:cols.stop // group])
    return w


def quantize_weight_int4(w: torch.Tensor, group: int = 128, *, zero_points: bool = False) -> Int4OprojWeight:
    """Round a bf16 or fp16 ``[hidden, K]`` matrix to 4 bits, to the nearest: with zero points a group's range from its least to its
    largest value (and zero), without them -7 .. 7 times its largest magnitude / 7.  The scales have the matrix's type."""
    if w.dtype not in (torch.bfloat16, torch.float16) or w.dim() != 2 or group not in (32, 64, 128) or w.shape[1] % group or w.shape[1] % 64 \
            or not w.numel():
        raise ValueError("quantize_weight_int4 needs a bfloat16 or float16 [hidden, K % 64 == 0 and % group == 0] matrix")
    hidden, K = w.shape
    v = w.float().view(hidden, K // group, group)
    least = 2.0 ** -24                                   # a group of zeros has to have a scale, too
    if zero_points:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scales = ((hi - lo) / 15).clamp(min=least).to(w.dtype)
        zeros = (-lo / scales.float()).round().clamp(0, 15)
    else:
        scales = (v.abs().amax(-1) / 7).clamp(min=least).to(w.dtype)
        zeros = torch.full_like(scales, 8, dtype=torch.float32)
    q = (v / scales.float().unsqueeze(-1) + zeros.unsqueeze(-1)).round().clamp(0, 15).to(torch.uint8).view(hidden, K)
    return pack_weight_int4(q[:, 0::2] | (q[:, 1::2] << 4), scales, zeros.to(torch.uint8) if zero_points else None)


def unpack_weight_int4(w: Int4OprojWeight) -> torch.Tensor:
    """The fp32 ``[hidden, K]`` matrix that a packed 4-bit weight stands for (oracles, debugging)."""
    slabs = -(-w.hidden // 128)
    out = torch.empty(slabs * 128, w.K, device=w.packed.device)
    for cols, q, s, z in w.records():
        q = torch.stack([q & 15, q >> 4], -1).view(slabs, 8, -1, 16, 4, 2, 4).permute(0, 1, 3, 2, 4, 6, 5).reshape(slabs * 128, -1, w.group)

        def rows(t):
            return t.permute(0, 2, 4, 3, 1).reshape(slabs * 128, -1, 1).float()

        out[:, cols] = ((q.float() - (8.0 if z is None else rows(z))) * rows(s)).flatten(1)
    return out[:w.hidden]


def check_compute_status(like: torch.Tensor) -> None:
    """Raise if an attention / GEMM kernel gave up on a bounded wait since the last check."""
    ops = _ext.ops
    code = int(ops().read_error_flag(like))
    if code != 0:
        ops().clear_error_flag(like)
        raise RuntimeError(f"helix compute kernel reported status {code} (a bounded wait ran out)")
