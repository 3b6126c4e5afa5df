"""Models served in microscaling formats: matrices in 4 bits, rows in 8, and the operators that take and leave them.

A group of 32 neighbours along a row shares a power of two, kept as one byte s: 2^(s - 127), 255 for a group that is no number. A matrix
holds e2m1 numbers (`Mxfp4Matrix`, a little over a quarter of bfloat16's bytes), rows of activations e4m3 numbers (`Mxfp8Rows`). The
group's byte follows from its largest magnitude m 2^x, 1 <= m < 2: s - 127 = x - emax + (m > 1.75), emax = 2 and 8; numbers are rounded to
nearest, ties to even. A group that holds an infinity or a NaN is NaN throughout. The reference serves 4-bit weights in formats of its own
(src/core/quant.cpp, groups of 32 with a 16-bit scale); these are the ones that gfx950's instructions convert and multiply.

    w = Mxfp4Matrix.quantize(weight)                 # once, at load
    gemm_mx(x, w, bias, out=y)                       # x bfloat16, float32 or Mxfp8Rows
    rows = Mxfp8Rows.empty(n, width)
    norm_mx(rows, stream, norm_weight, eps, add=y, stream=stream)
    gemm_mx(rows, w, bias, residual=stream)

As everywhere in this package, operands are checked on the host, launches go to torch's current stream, and nothing runs without the GPU.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ..errors import KernelError
from . import lib as _lib
from . import ops
from .ops import ACTIVATION_EPILOGUE, EPI_QKV_PAGED, EPI_RESIDUAL, F32, GLU_ACTIVATIONS, _dev, _epilogue, _f32vec, _ptr, _rows, _stream, dtype_code

GROUP = 32
CHUNK = 128  # k of a block of a matrix; rows of codes are padded to whole chunks
STRIP = 16  # matrix rows of a block
BLOCK_BYTES = 1088  # 16 x 128 numbers of 4 bits and their 64 scales
NORM_MAX_WIDTH = 65536
CLAMPED_GLU = 2
_ROWS_BF16, _ROWS_F32, _ROWS_MX = 0, 1, 2


def _round_up(n: int, m: int) -> int:
    return -(-n // m) * m


# torch's types of what the formats hold; a tensor of another 8-bit type stands for other numbers than its bytes would be taken for
_E4M3, _E2M1, _E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _bytes(t: torch.Tensor, what: str, kind: torch.dtype) -> torch.Tensor:
    """The bytes of a tensor of uint8 or of `kind`, rows contiguous."""
    _dev(t, what)
    if t.dtype not in (torch.uint8, kind):
        raise KernelError(f"{what} must be uint8 or {str(kind).replace('torch.', '')}, not {t.dtype}")
    t = t if t.dtype == torch.uint8 else t.view(torch.uint8)
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise KernelError(f"{what} must be 2-D with contiguous rows, got shape {tuple(t.shape)} strides {t.stride()}")
    return t


class Mxfp4Matrix:
    """A matrix [out, in] in 4 bits, in the order in which the products read it: `blocks`, uint8 [strips of 16 rows, chunks of 128 k, 1,088
    bytes] (csrc/mx.h). Made once, by `quantize` or `pack`; `dense` gives its values."""

    replayable = True  # (layers that hold it may run from a recorded list: it is its tensor and its sizes)

    eight_bit_rows = False  # a model served with 8-bit rows sets it on its matrices: products by them take `Mxfp8Rows`

    def __init__(self, blocks: torch.Tensor, rows: int, width: int):
        if rows < 1 or width < 1:
            raise KernelError(f"a matrix of {rows} x {width}")
        shape = (-(-rows // STRIP), -(-width // CHUNK), BLOCK_BYTES)
        _dev(blocks, "blocks")
        if blocks.dtype != torch.uint8 or tuple(blocks.shape) != shape or not blocks.is_contiguous() or blocks.data_ptr() % 16:
            raise KernelError(f"a 4-bit matrix of {rows} x {width} needs contiguous uint8 blocks {shape} on a 16-byte boundary, got {tuple(blocks.shape)} {blocks.dtype}")
        self.blocks, self.rows, self.width, self.index = blocks, rows, width, blocks.get_device()

    @property
    def shape(self):
        return (self.rows, self.width)

    @property
    def device(self):
        return self.blocks.device

    def bytes(self) -> int:
        return self.blocks.numel()

    @classmethod
    def _empty(cls, rows: int, width: int, device) -> "Mxfp4Matrix":
        if rows < 1 or width < 1:
            raise KernelError(f"a matrix of {rows} x {width}")
        return cls(torch.empty((-(-rows // STRIP), -(-width // CHUNK), BLOCK_BYTES), dtype=torch.uint8, device=device), rows, width)

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Mxfp4Matrix":
        """The matrix w [out, in] (float32 or bfloat16) rounded to 4 bits."""
        _dev(w, "w")
        ldw = _rows(w, "w")
        code = dtype_code(w.dtype)
        out = cls._empty(w.shape[0], w.shape[1], w.device)
        with torch.cuda.device(w.device):
            _lib.call("liyab_mx_quantize", out.blocks.data_ptr(), w.data_ptr(), code, ldw, out.rows, out.width, _stream())
        return out

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, width: int) -> "Mxfp4Matrix":
        """From plain rows: codes uint8 (or float4_e2m1fn_x2) [out, ceil(width / 2)], two numbers a byte, the first in the low half (or whole groups, [out, 16 ceil(width / 32)],
        where what lies behind the width does not count), and scales [out, ceil(width / 32)], uint8 or float8_e8m0fnu."""
        codes, scales = _bytes(codes, "codes", _E2M1), _bytes(scales, "scales", _E8M0)
        if width < 1 or codes.shape[1] not in (-(-width // 2), -(-width // GROUP) * (GROUP // 2)) or tuple(scales.shape) != (codes.shape[0], -(-width // GROUP)) or scales.device != codes.device:
            raise KernelError(f"a 4-bit matrix of width {width} needs codes [out, {-(-width // 2)}] or [out, {-(-width // GROUP) * (GROUP // 2)}] and scales [out, {-(-width // GROUP)}], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        out = cls._empty(codes.shape[0], width, codes.device)
        with torch.cuda.device(codes.device):
            _lib.call("liyab_mx_pack", out.blocks.data_ptr(), codes.data_ptr(), _rows(codes, "codes"), scales.data_ptr(), _rows(scales, "scales"), out.rows, width, _stream())
        return out

    def dense(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [out, in]; bfloat16 holds them as exactly as float32 does (a number of 2^128, which only a matrix
        with values above 2.9e38 has, is infinite in both)."""
        w = torch.empty((self.rows, self.width), dtype=dtype, device=self.blocks.device)
        with torch.cuda.device(self.blocks.device):
            _lib.call("liyab_mx_dense", w.data_ptr(), dtype_code(dtype), self.width, self.blocks.data_ptr(), self.rows, self.width, _stream())
        return w


class Mxfp8Rows:
    """Rows [n, width] in 8 bits: `codes` uint8 [n, width rounded up to 128] (e4m3, zeros behind the width) and `scales` uint8 [n, a byte a
    group of 32, padded to 16]. `empty` and `pack` make the tensors; a workspace's may be given. The operators that write rows write all of a last chunk of 128:
    who fills them otherwise leaves zeros behind the width in both (a byte of 255 there would make products of the row no numbers)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, width: int):
        self.codes, self.scales, self.n, self.width = codes, scales, codes.shape[0], width
        if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or tuple(scales.shape) != (self.n, self.scale_width(width))
                or width < 1 or codes.shape[1] != _round_up(width, CHUNK) or not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device):
            raise KernelError(f"rows of {width} values in 8 bits need contiguous uint8 codes [n, {_round_up(max(width, 1), CHUNK)}] and scales "
                              f"[n, {self.scale_width(max(width, 1))}], got {tuple(codes.shape)} {codes.dtype} and {tuple(scales.shape)} {scales.dtype}")
        _dev(codes, "codes")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise KernelError("codes and scales must start on 16-byte boundaries")
        self.index = codes.get_device()

    @staticmethod
    def scale_width(width: int) -> int:
        return _round_up(-(-width // GROUP), 16)

    @property
    def shape(self):
        return (self.n, self.width)

    @property
    def device(self):
        return self.codes.device

    @classmethod
    def shapes(cls, n: int, width: int):
        """The shapes of the codes and the scales of n rows."""
        return (n, _round_up(width, CHUNK)), (n, cls.scale_width(width))

    @classmethod
    def empty(cls, n: int, width: int, device="cuda") -> "Mxfp8Rows":
        codes, scales = cls.shapes(n, width)
        return cls(torch.empty(codes, dtype=torch.uint8, device=device), torch.empty(scales, dtype=torch.uint8, device=device), width)

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Mxfp8Rows":
        """From plain rows: codes [n, width] (float8_e4m3fn, or their bytes) and scales [n, ceil(width / 32)] (float8_e8m0fnu, or their bytes)."""
        codes, scales = _bytes(codes, "codes", _E4M3), _bytes(scales, "scales", _E8M0)
        n, width = codes.shape
        if width < 1 or tuple(scales.shape) != (n, -(-width // GROUP)) or scales.device != codes.device:
            raise KernelError(f"rows [{n}, {width}] need scales [{n}, {-(-width // GROUP)}], got {tuple(scales.shape)}")
        out = cls(torch.zeros((n, _round_up(width, CHUNK)), dtype=torch.uint8, device=codes.device),
                  torch.zeros((n, cls.scale_width(width)), dtype=torch.uint8, device=codes.device), width)
        out.codes[:, :width] = codes
        out.scales[:, : scales.shape[1]] = scales
        return out


def _check_out(out: Mxfp8Rows, n: int, d: int, what: str) -> None:
    if not isinstance(out, Mxfp8Rows):
        raise KernelError(f"{what}: the result goes to Mxfp8Rows, not to {type(out).__name__}")
    if out.n != n or out.width != d:
        raise KernelError(f"{what}: the rows have places for [{out.n}, {out.width}], not [{n}, {d}]")


def _stride(t: torch.Tensor, what: str) -> int:
    """`ops._rows`, asking the usual rows less (0.4 us a tensor of a call's 8)."""
    if t.is_cuda and t.dim() == 2:
        ld, step = t.stride()
        if step == 1 and ld >= t.shape[1]:
            return ld
    return _rows(t, what)


def _stream_on(index: int) -> int:
    """The stream that launches go to (`ops._stream`; asked for without the objects that torch makes around it, 2 us of a call)."""
    return ops._pinned_stream if ops._pinned_stream is not None else torch._C._cuda_getCurrentRawStream(index)


def _refuse_devices(what: str, index: int, *tensors) -> None:
    """Every operand lies on the device that launches go to; `_on` has found one that does not."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise KernelError(f"{what}: operands on {t.device} and cuda:{index}")
    raise KernelError(f"{what}: operands on cuda:{index}, the current device is cuda:{torch.cuda.current_device()}")


def _on(what: str, index: int, *tensors) -> int:
    if index != torch._C._cuda_getDevice():
        _refuse_devices(what, index)
    for t in tensors:
        if t is not None and t.get_device() != index:
            _refuse_devices(what, index, t)
    return _stream_on(index)


def rows_mx(out: Mxfp8Rows, x: torch.Tensor) -> None:
    """out = x [n, d] (float32 or bfloat16, rows contiguous) in 8 bits."""
    ldx = _stride(x, "x")
    _check_out(out, x.shape[0], x.shape[1], "rows_mx")
    stream = _on("rows_mx", out.index, x)
    if out.n == 0:
        return
    _lib.call("liyab_mx_rows", out.codes.data_ptr(), out.codes.shape[1], out.scales.data_ptr(), out.scales.shape[1], x.data_ptr(), dtype_code(x.dtype), ldx,
              out.n, out.width, stream)


def glu_mx(out: Mxfp8Rows, gu: torch.Tensor, activation: str, clamp=None) -> None:
    """out = act(G) * U in 8 bits; gu float32 [n, 2 * d] = [G | U]; act "silu" or "gelu_tanh", or "clamped" with clamp = (limit, slope, shift): g *
    sigmoid(slope * g) * (u + shift), g = min(G, limit), u = clamp(U, -limit, limit) (`ops.glu`, `ops.glu_clamped`). Computed in 64 bits, `clamp`'s numbers too, as `norm_mx`."""
    ld = _stride(gu, "gu")
    n, d2 = gu.shape
    if gu.dtype != torch.float32 or d2 % 2:
        raise KernelError(f"glu_mx: needs float32 [n, 2 * d], got {tuple(gu.shape)} {gu.dtype}")
    _check_out(out, n, d2 // 2, "glu_mx")
    stream = _on("glu_mx", out.index, gu)
    if (activation == "clamped") != (clamp is not None) or (clamp is None and activation not in GLU_ACTIVATIONS):
        raise KernelError(f"glu_mx: activation '{activation}' with clamp {clamp}")
    limit, slope, shift = clamp or (1.0, 1.0, 0.0)
    if not limit > 0:
        raise KernelError(f"glu_mx: a limit of {limit}")
    if n == 0:
        return
    act = CLAMPED_GLU if clamp is not None else GLU_ACTIVATIONS[activation]
    _lib.call("liyab_mx_glu", out.codes.data_ptr(), out.codes.shape[1], out.scales.data_ptr(), out.scales.shape[1], gu.data_ptr(), ld, n, d2 // 2, act,
              float(limit), float(slope), float(shift), stream)


def _shifted(t: torch.Tensor, other: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory other than value by value."""
    a, b = t.data_ptr(), other.data_ptr()
    if a == b and t.dtype == other.dtype:
        return False
    return a < b + other.numel() * other.element_size() and b < a + t.numel() * t.element_size()


def norm_mx(out: Mxfp8Rows, x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, *, bias: Optional[torch.Tensor] = None, centred: bool = False,
            add: Optional[torch.Tensor] = None, stream: Optional[torch.Tensor] = None) -> None:
    """With t = x + add: out = t / sqrt(mean(t^2) + eps) * weight (+ bias) in 8 bits; `centred`: a layer norm, (t - mean(t)) / sqrt(var(t) + eps) * weight
    + bias. x float32 [n, d], d up to 65,536; `add` [n, d] float32 or bfloat16 (a sublayer's result); `stream` float32 [n, d] gets t (it may be
    x itself, or `add`, but lie across neither). Computed in 64 bits, eps too: values next to a border of the 8-bit numbers land on its right side."""
    _dev(x, "x")
    if x.dtype != torch.float32 or x.dim() != 2 or not x.is_contiguous():
        raise KernelError(f"norm_mx: x must be contiguous float32 [n, d], got {tuple(x.shape)} {x.dtype}")
    n, d = x.shape
    if d > NORM_MAX_WIDTH:
        raise KernelError(f"norm_mx: rows of {d} values (up to {NORM_MAX_WIDTH})")
    _check_out(out, n, d, "norm_mx")
    _f32vec(weight, "norm weight", d)
    _f32vec(bias, "norm bias", d)
    code = F32
    if add is not None:
        code = dtype_code(add.dtype)
        if add.shape != x.shape or not add.is_contiguous():
            raise KernelError(f"norm_mx: what is added must be contiguous [{n}, {d}], got {tuple(add.shape)}")
    if stream is not None and (stream.dtype != torch.float32 or stream.shape != x.shape or not stream.is_contiguous()):
        raise KernelError(f"norm_mx: the stream must be contiguous float32 [{n}, {d}], got {tuple(stream.shape)} {stream.dtype}")
    to = _on("norm_mx", out.index, x, weight, bias, add, stream)
    if stream is not None and (_shifted(stream, x) or (add is not None and _shifted(stream, add))):
        raise KernelError("norm_mx: the stream lies across what the norm reads")
    if n == 0:
        return
    _lib.call("liyab_mx_norm", out.codes.data_ptr(), out.codes.shape[1], out.scales.data_ptr(), out.scales.shape[1], x.data_ptr(), _ptr(add), code, _ptr(stream),
              _ptr(weight), _ptr(bias), float(eps), 1 if centred else 0, n, d, to)


def gemm_mx(a, w: Mxfp4Matrix, bias: Optional[torch.Tensor], *, out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
            activation: str = "none", kv=None, shape: int = 0) -> None:
    """out = act(a . w^T + bias), or residual += a . w^T + bias, or the paged query, key and value product (`kv` as `ops.gemm` takes it): one of the three. a [M, K]: bfloat16 or
    float32 with contiguous rows, or `Mxfp8Rows`; out [M, N] bfloat16 or float32, residual float32. Products are exact in 32 bits
    and their sums are 32-bit, whatever the rows' kind and number. A row has the same bits whatever the other rows if it is float32, or under `ops.batch_invariant`. `shape`: the workgroups' (csrc/mx_product.hip; 0: chosen from the sizes), for bfloat16 and 8-bit rows."""
    if not isinstance(w, Mxfp4Matrix):
        raise KernelError(f"gemm_mx: the matrix is a Mxfp4Matrix, not {type(w).__name__}")
    if residual is not None and (out is not None or kv is not None):
        raise KernelError("gemm_mx: the result is added to a residual or goes to out, not both")
    if activation != "none" and (residual is not None or kv is not None):
        raise KernelError(f"gemm_mx: activation '{activation}' is for results that go to out")
    if activation not in ACTIVATION_EPILOGUE:
        raise KernelError(f"gemm_mx: activation '{activation}' is not known")
    index, K, N = w.index, w.width, w.rows
    if isinstance(a, Mxfp8Rows):
        kind, operand, M, dtype = _ROWS_MX, a.codes, a.n, torch.bfloat16
        if a.width != K:
            raise KernelError(f"gemm_mx: rows of {a.width} values, a matrix of width {K}")
        lda, scales, lds = operand.shape[1], a.scales.data_ptr(), a.scales.shape[1]
    else:
        lda, operand, scales, lds, dtype = _stride(a, "a"), a, None, 0, a.dtype
        M, width = a.shape
        if width != K or (dtype is not torch.bfloat16 and dtype is not torch.float32):
            raise KernelError(f"gemm_mx: a {tuple(a.shape)} {dtype} does not fit a matrix of {N} x {K}")
        kind, per = (_ROWS_BF16, 8) if dtype is torch.bfloat16 else (_ROWS_F32, 4)
        if shape and kind == _ROWS_F32:
            raise KernelError(f"gemm_mx: float32 rows have one shape of workgroups, not shape {shape}")
    stream = _on("gemm_mx", index, operand, bias, out, residual, *(kv[:3] if kv is not None else ()))
    if kv is not None:
        e = _epilogue(_Like(M, dtype), w, bias, out, None, EPI_QKV_PAGED, kv)
    else:
        _f32vec(bias, "bias", N)
        if residual is not None:
            if residual.dtype is not torch.float32 or residual.shape != (M, N):
                raise KernelError("gemm_mx: needs a float32 residual [M, N]")
            e = _lib.EpiParams(EPI_RESIDUAL, F32, _ptr(bias), None, 0, residual.data_ptr(), _stride(residual, "residual"))
        else:
            if out is None or out.shape != (M, N):
                raise KernelError("gemm_mx: out must be [M, N]")
            e = _lib.EpiParams(ACTIVATION_EPILOGUE[activation], dtype_code(out.dtype), _ptr(bias), out.data_ptr(), _stride(out, "out"))
        e.exact = 1 if kind == _ROWS_F32 else 0
    if M == 0:
        return
    ptr = operand.data_ptr()
    if kind != _ROWS_MX and (K % per or lda % per or ptr % 16):
        # rows that are no whole pieces of 16 bytes, or lie between them: a copy that is, in memory that only this call has (a list of launches
        # that is run again would find somebody else's there)
        _lib.not_recordable()
        K = lda = _round_up(K, per)
        own = torch.empty((M, K), dtype=dtype, device=a.device)
        _lib.call("liyab_mx_align", own.data_ptr(), K, ptr, _rows(a, "a"), a.element_size(), M, w.width, stream)
        ptr = own.data_ptr()
    _lib.call("liyab_mx_product", ptr, lda, scales, lds, kind, w.blocks.data_ptr(), M, N, K, shape or (-1 if ops._invariant else 0), ctypes.byref(e), stream)


class _Like:
    """What the epilogue's checks read of rows in 8 bits."""

    def __init__(self, n: int, dtype: torch.dtype):
        self.shape, self.dtype = (n, 0), dtype
