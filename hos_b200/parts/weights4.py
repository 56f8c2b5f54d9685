"""A matrix held in 4 bits: codes 0..15, a scale (bfloat16) and, if it has them, a zero code per `group` neighbouring weights of a
row; W[n, k] = (code - zero) * scale, zero 8 where there are none.  Products with it go through `linear.matmul` like those with any
other matrix, with rows in bfloat16 or in 32 bits.  Up to 32 rows, and for rows in 32 bits, no weight is rounded; for more bfloat16 rows a
weight is rounded once to 11 bits, also where the result is asked for in 32 bits (csrc/weights4_tc.cu).

`from_codes` takes what a quantised checkpoint holds, `from_matrix` rounds a matrix.  Both lay the codes out once, as the
operand registers of the tensor cores want them (csrc/fourbit.cuh)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import ops
from ..errors import KernelError, SpecError

ROWS, COLS = 16, 64             # of a block of codes
# Up to so many rows the codes are multiplied as they are, above the weights are formed in half precision (us a product, that kernel's / the
# tcgen05 one's: 2304 x 9216, 32 rows 12.8 / 19.3, 33 rows, one more tile of 32, 22.1 / 19.6; 9216 x 2304 gated, 16 rows 13.6 / 17.5, 32 rows
# 21.1 / 18.5, 33 rows 35.9 / 19.1).  Gated products of many weights would gain from 17 rows on (14336 x 3584, 24 rows 41.4 / 32.2), but
# up to 32 rows, where most steps of a few sequences lie, no weight is rounded.
FEW_ROWS = 32
MOST_TC_K = 1 << 21
LARGEST_SCALE = 2048.0          # a feature's largest scale in half precision lies between it and twice it


def _in_half(records: torch.Tensor, n: int, blocks: int, zeros: bool):
    """What the products of many rows take: the records with scales in half precision, a feature's times the power of two that brings its
    largest between 2^11 and 2^12 (a weight is at most 15 of it, 61,440), and 1024 + zero codes; and the powers that undo it, float32
    [blocks * n]."""
    r = records.float()                                          # [blocks * tiles, groups, 8, 1 or 2, 2]
    tiles = r.shape[0] // blocks
    scale = r[:, :, :, 0].nan_to_num(0.0, 0.0, 0.0).abs().amax(1)   # [blocks * tiles, 8, 2]: of the rows g and g + 8
    power = torch.exp2(torch.floor(torch.log2(scale.double().clamp(min=2.0 ** -126))).clamp(-126, 127)).float()
    power = torch.where(scale > 0, power, 1.0) / LARGEST_SCALE
    r[:, :, :, 0] /= power[:, None]
    if zeros:
        r[:, :, :, 1] += 1024.0 - 128.0
    powers = power.permute(0, 2, 1).reshape(blocks, tiles * ROWS)[:, :n].contiguous()
    return r.to(torch.float16).contiguous(), powers.view(-1)


def _check_on_gpu(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The kernels keep the tensors' addresses: all of them have to be one GPU's."""
    there = {t.device for t in tensors if t is not None}
    if len(there) != 1 or next(iter(there)).type != "cuda":
        raise SpecError(f"{what} must be on the GPU, all on the same, found {sorted(map(str, there))}")


def _check_group(group: int) -> None:
    if group != 32 and (group < 64 or group % 64):
        raise SpecError(f"groups of {group} weights: 32 or a multiple of 64 is wanted")


class Weight4:
    def __init__(self, codes: torch.Tensor, records: torch.Tensor, n: int, k: int, group: int, blocks: int, zeros: bool):
        _check_on_gpu("a matrix in 4 bits", codes, records)
        self.codes, self.records = codes, records
        self.records16, self.powers = _in_half(records, n, blocks, zeros)
        self.n, self.k, self.group, self.blocks, self.zeros = n, k, group, blocks, zeros
        self._matrix = ops.Matrix4(codes.data_ptr(), records.data_ptr(), self.records16.data_ptr(), self.powers.data_ptr(), n, k, group, int(zeros), int(blocks == 2))
        self._address = ctypes.addressof(self._matrix)
        self._forms = COLS <= k <= MOST_TC_K and codes.numel() < 1 << 32      # what the kernel that forms weights takes

    @property
    def shape(self):
        return torch.Size((self.blocks * self.n, self.k))

    def nbytes(self) -> int:
        return self.codes.numel() + 2 * (self.records.numel() + self.records16.numel()) + 4 * self.powers.numel()

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], group: int, blocks: int = 1) -> "Weight4":
        """On the GPU, codes: uint8 [rows, k], 0..15; scales: [rows, ceil(k / group)], kept in
        bfloat16 (scales in another type are rounded to it, by up to 2^-8 of themselves); zeros: uint8 like the scales, or None.
        `blocks`: the rows are that many matrices one after another (2: gate and up of a gated feed-forward)."""
        _check_group(group)
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise SpecError(f"codes must be uint8 [rows, k], found {codes.dtype} {tuple(codes.shape)}")
        _check_on_gpu("codes, scales and zero codes", codes, scales, zeros)
        rows, k = codes.shape
        want = (rows, -(-k // group))
        if k == 0 or rows == 0 or blocks < 1 or rows % blocks:
            raise SpecError(f"{rows} x {k} codes are not {blocks} matrices")
        if tuple(scales.shape) != want or not scales.is_floating_point():
            raise SpecError(f"scales must be floating-point numbers {want}, found {scales.dtype} {tuple(scales.shape)}")
        if zeros is not None and (tuple(zeros.shape) != want or zeros.dtype != torch.uint8):
            raise SpecError(f"zero codes must be uint8 {want}, found {zeros.dtype} {tuple(zeros.shape)}")
        if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
            raise SpecError("codes and zero codes must be 0..15")
        n = rows // blocks
        tiles, k_blocks = -(-n // ROWS), -(-k // COLS)
        groups = -(-k_blocks * COLS // group)
        padded = codes.new_zeros((blocks, tiles * ROWS, k_blocks * COLS))
        padded[:, :n, :k] = codes.reshape(blocks, n, k)
        # a row 8 hi + g, a number 32 w + 8 t + 2 r + h of a block: byte (g, t, hi, w, h, r / 2), nibble r % 2
        p = padded.view(blocks * tiles, 2, 8, k_blocks, 2, 4, 4, 2).permute(0, 3, 2, 5, 1, 4, 7, 6)
        packed = (p[..., 0::2] | (p[..., 1::2] << 4)).contiguous().view(blocks * tiles, k_blocks, 512)

        def records(t):                                      # [blocks * tiles, groups, 8, 2]: rows g and g + 8 side by side
            r = t.new_zeros((blocks, tiles * ROWS, groups), dtype=torch.bfloat16)
            r[:, :n, :want[1]] = t.reshape(blocks, n, want[1]).to(torch.bfloat16)
            return r.view(blocks * tiles, 2, 8, groups).permute(0, 3, 2, 1)
        parts = [records(scales)]
        if zeros is not None:
            parts.append(records(zeros.to(torch.int32) + 128))
        return cls(packed, torch.stack(parts, dim=3).contiguous(), n, k, group, blocks, zeros is not None)

    @classmethod
    def from_matrix(cls, w: torch.Tensor, group: int = 64, zeros: bool = False, blocks: int = 1) -> "Weight4":
        """The matrix [rows, k] rounded: scale (max - min) / 15 and the zero code nearest to 0's place (`zeros`), or largest
        magnitude / 7, per group; the scale is rounded to bfloat16 before the codes are taken."""
        _check_group(group)
        if w.dim() != 2 or not w.is_floating_point():
            raise SpecError(f"a matrix is wanted, found {w.dtype} {tuple(w.shape)}")
        _check_on_gpu("a matrix to be held in 4 bits", w)
        rows, k = w.shape
        g = torch.nn.functional.pad(w.float(), (0, -k % group)).reshape(rows, -1, group)
        if not bool(torch.isfinite(g).all()):
            raise SpecError("a matrix with infinities or NaN cannot be held in 4 bits")
        if zeros:
            lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
            s = ((hi - lo) / 15).to(torch.bfloat16)
            z = torch.round(-lo / torch.where(s > 0, s.float(), 1.0)).clamp(0, 15)
        else:
            s = (g.abs().amax(-1) / 7).to(torch.bfloat16)
            z = torch.full_like(s, 8.0, dtype=torch.float32)
        inner = g / torch.where(s > 0, s.float(), 1.0)[..., None] + z[..., None]
        codes = torch.round(inner).clamp_(0, 15).to(torch.uint8).view(rows, -1)[:, :k].contiguous()
        return cls.from_codes(codes, s, z.to(torch.uint8) if zeros else None, group, blocks)

    def first_rows(self, n: int) -> Optional["Weight4"]:
        """The first n rows (a view), or None where n cuts a block."""
        if self.blocks != 1 or n % ROWS or n > self.n:
            return None
        return Weight4(self.codes[:n // ROWS], self.records[:n // ROWS], n, self.k, self.group, 1, self.zeros)

    def product(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None, epilogue: int = ops.EPI_NONE, cap: float = 0.0, act: int = 0,
                out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x . W^T as `linear.matmul` describes it; epilogues: none, gated."""
        gated = epilogue == ops.EPI_GATED
        if epilogue not in (ops.EPI_NONE, ops.EPI_GATED) or bias is not None:
            raise KernelError("products with 4-bit weights have no epilogue but the gated one")
        if self.blocks != (2 if gated else 1):
            raise KernelError(f"a {'gated' if gated else 'plain'} product is asked of {self.blocks} matrices")
        ops._check_rows(x, "left operand")
        if x.shape[1] != self.k:
            raise KernelError(f"product with 4-bit weights: rows of {x.shape[1]} numbers, weights of {self.k}")
        if out is None:
            out = x.new_empty((x.shape[0], self.n), dtype=out_dtype or x.dtype)
        else:
            ops._check_rows(out, "product")
            if tuple(out.shape) != (x.shape[0], self.n):
                raise KernelError(f"product with 4-bit weights: the output is {tuple(out.shape)}, not {(x.shape[0], self.n)}")
        if x.shape[0] > FEW_ROWS and self._forms and x.dtype == torch.bfloat16:
            ops.product4_tc(x, self._address, self.k, out, act, cap)
        else:
            ops.product4(x, self._address, out, act, cap)
        return out
