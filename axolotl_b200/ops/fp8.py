"""8-bit blocks: E4M3 activations with a power-of-two scale for each row and 128 columns, frozen E4M3 weights with an fp32 scale for
each 128 x 128 block (the layout of block-FP8 checkpoints), and the linear layers on them.

A row's block is held as ``q s`` with ``s = 2^ceil(log2(max |x| / 448))`` (1 for a block of zeros, never below 2^-126) and ``q`` the
nearest E4M3 number to ``x / s``, ties to even. A power of two divides exactly, so that ``q`` does not depend on the precision it is
computed in and ``q s`` is a bf16 number. NaN and infinities become NaN codes; the other values of their block keep their scale. A
finite value stays finite: where the nearest code would stand for 2^128, ``q`` is the one below.

``fp8_linear`` and ``fp8_lora_linear`` quantise their input once: the codes are the operand of the forward product and all that is
kept of the input for the backward pass, half of what bf16 takes. The backward pass quantises the output gradient the same way and
reads the same weight codes as the other operand order. The quantisers pass gradients straight through; one gradient is not the derivative
of what stands beside it: the low-rank product of an adapter reads the bf16 rows, ``y = x8 W8^T + s (x A^T) B^T``, and ``dA = (s dy B)^T x8``
the coded ones, the only ones that are kept.

``s x A^T`` and ``s dy B`` enter ``y`` and ``dx`` rounded to bf16, as in the bf16 layer (``ops.lora``), which leaves these within their own
rounding. For ``dB`` and ``dA``, where it would add as much again, both are held as two bf16 numbers up to rank 64 (off by 2^-16). All sums
of an adapter's gradients up to rank 64 are joined in a fixed order: the same bits every time.

The reference keeps such weights in FP8 only under adapters (src/axolotl/integrations/kernels/libs/dsv4/lora_fp8.py:1-147: a library
product in the forward pass, the weight expanded to bf16 in the backward pass) and expands them elsewhere
(src/axolotl/kernels/quantize.py:109-135).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
import struct
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK = 128
E4M3_MAX = 448.0
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _device_of(t):
    """Launches go to the current device: makes it the tensor's where it is another one."""
    return contextlib.nullcontext() if t.device.index == _current_device() else torch.cuda.device(t.device)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _padded(rows: int, cols: int, device):
    """Codes [rows, cols] whose rows start on 16 bytes (bulk tensor copies)."""
    ld = -(-cols // 16) * 16
    return torch.empty((rows, ld), dtype=torch.float8_e4m3fn, device=device)[:, :cols]


def _check_codes(codes, what):
    if codes.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{what}: codes are float8_e4m3fn, got {codes.dtype}")
    if codes.dim() != 2 or 0 in codes.shape[1:]:
        raise ValueError(f"{what}: codes are a matrix [rows, columns] with a column at least, got {tuple(codes.shape)}")


def _check_scale(scale, shape, device, what):
    if scale.dtype != torch.float32 or tuple(scale.shape) != shape or scale.device != device:
        raise ValueError(f"{what}: scales are float32 {shape} on {device}, got {scale.dtype} {tuple(scale.shape)} on {scale.device}")


def _rows16(codes):
    """``codes`` with rows of whole 16 bytes: as they are, or laid out again."""
    ld, unit = codes.stride()
    if unit == 1 and ld % 16 == 0 and ld >= codes.shape[1] and codes.data_ptr() % 16 == 0:
        return codes
    out = _padded(*codes.shape, codes.device)
    out.view(torch.uint8).copy_(codes.view(torch.uint8))
    return out


def _operand16(t):
    return t.dtype == torch.bfloat16 and t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0


def _operand(t, what):
    """A bf16 matrix as bulk tensor copies read it: rows of whole 16 bytes, on 16 bytes."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{what} takes bf16 matrices beside the codes, got {t.dtype}")
    if _operand16(t):
        return t
    out = t.new_empty((t.shape[0], (t.shape[1] + 7) & ~7))[:, :t.shape[1]]
    return out.copy_(t)


def _row_scales(scale, rows):
    """(tensor, row stride) of the scales [blocks, rows] as the kernels read them."""
    if scale.stride(1) != 1 or (scale.shape[0] > 1 and scale.stride(0) < rows):
        scale = scale.contiguous()
    return scale, max(scale.stride(0), rows)


# ------------------------------------------------------------------ rows
def quantize_fp8_rows(x: torch.Tensor):
    """x [rows, columns] (bf16, fp16 or fp32) -> (codes float8_e4m3fn [rows, columns], scales fp32 [ceil(columns / 128), rows]). Rows of
    codes start on 16 bytes, so that they are operands of the tensor-core kernels as they are."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"quantize_fp8_rows takes a matrix [rows, columns] with a column at least, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"quantize_fp8_rows takes bfloat16, float16 or float32, got {x.dtype}")
    return _unpacked(_pack(x.detach()), *x.shape)


def _lead(T, K):
    """Row lengths of a block of ``_pack``: codes in bytes, scales in numbers."""
    return (K + 15) & ~15, (T + 3) & ~3


def _packed_size(T, K):
    return T * ((K + 15) & ~15) + 4 * _blocks(K) * ((T + 3) & ~3)


_ROWS = struct.Struct("@3P2q2i")        # AxbFp8Rows of csrc/fp8_rows.cu


def _pack(x):
    """The 8-bit rows of x [T, K] as one block of bytes: T rows of codes, K rounded up to 16 bytes, and behind them the scales, fp32
    [ceil(K / 128)][T rounded up to 4]. What the layers and the checkpoint store keep."""
    T, K = x.shape
    if not x.is_cuda:
        return _pack_plain(x, *_lead(T, K))
    device = x.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return _pack(x)
    if x.stride(1) != 1 and K > 1:
        x = x.contiguous()
    q = x.new_empty(_packed_size(T, K), dtype=torch.uint8)
    _lib.check_rc(_lib.cuda_lib().axb_fp8_pack_rows(_ROWS.pack(x.data_ptr(), q.data_ptr(), torch._C._cuda_getCurrentRawStream(device.index),
                                                               x.stride(0), T, K, _DTYPES[x.dtype])), "fp8_quantize_rows")
    return q


def _unpacked(q, T, K):
    """(codes [T, K], scales [ceil(K / 128), T]): views of a block of ``_pack``."""
    ld, lds = _lead(T, K)
    if T == 0:
        return q.new_empty((0, K)).view(torch.float8_e4m3fn), torch.empty((_blocks(K), 0), device=q.device)
    codes = q[:T * ld].view(T, ld).view(torch.float8_e4m3fn)
    return (codes if ld == K else codes[:, :K]), q[T * ld:].view(torch.float32).view(_blocks(K), lds)[:, :T]


def _unpack(q, T, K, dtype):
    """The values of a block of ``_pack``, [T, K]."""
    if not q.is_cuda:
        return dequantize_fp8_rows(*_unpacked(q, T, K), dtype)
    device = q.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return _unpack(q, T, K, dtype)
    out = q.new_empty((T, K), dtype=dtype)
    _lib.check_rc(_lib.cuda_lib().axb_fp8_unpack_rows(_ROWS.pack(out.data_ptr(), q.data_ptr(), torch._C._cuda_getCurrentRawStream(device.index),
                                                                 K, T, K, _DTYPES[dtype])), "fp8_dequantize_rows")
    return out


def _pack_plain(x, ld, lds):
    T, K = x.shape
    kb = _blocks(K)
    v = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K)).view(T, kb, BLOCK)
    v = v.masked_fill(v.isinf(), float("nan"))
    top = v.nan_to_num(nan=0.0).abs().amax(-1)
    m, e = torch.frexp(top)                                # top = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.ones_like(top))
    v = v.clamp(-240 * 2.0 ** 120, 240 * 2.0 ** 120)
    codes = (v / scale[..., None]).to(torch.float8_e4m3fn).view(T, kb * BLOCK)[:, :ld]
    scale = torch.nn.functional.pad(scale.t(), (0, lds - T))
    return torch.cat([codes.reshape(-1).view(torch.uint8), scale.reshape(-1).view(torch.uint8)])


def dequantize_fp8_rows(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The values that the codes of ``quantize_fp8_rows`` stand for (exact in bf16 and fp32), [rows, columns]. In fp16 2^16, the nearest code
    of that type's largest values, comes back as the largest one, 65504."""
    _check_codes(codes, "dequantize_fp8_rows")
    T, K = codes.shape
    _check_scale(scale, (_blocks(K), T), codes.device, "dequantize_fp8_rows")
    if dtype not in _DTYPES:
        raise TypeError(f"dequantize_fp8_rows gives bfloat16, float16 or float32, not {dtype}")
    if not codes.is_cuda:
        v = codes.float() * scale.t().repeat_interleave(BLOCK, 1)[:, :K]
        return (torch.where(v.abs() == 65536, torch.copysign(torch.full_like(v, 65504.0), v), v) if dtype == torch.float16 else v).to(dtype)
    with _device_of(codes):
        codes = _rows16(codes)
        scale, lds = _row_scales(scale, T)
        out = torch.empty((T, K), dtype=dtype, device=codes.device)
        _lib.check_rc(_lib.cuda_lib().axb_fp8_dequantize_rows(codes.data_ptr(), codes.stride(0), scale.data_ptr(), lds, out.data_ptr(), K,
                                                              _DTYPES[dtype], T, K, _lib.stream_ptr()), "fp8_dequantize_rows")
    return out


# ------------------------------------------------------------------ weights
@dataclass
class Fp8State:
    """Scales of a frozen weight held as codes [N, K]: fp32 [ceil(N / 128), ceil(K / 128)]."""
    shape: tuple
    scale: torch.Tensor

    def to(self, device):
        return Fp8State(self.shape, self.scale.to(device))

    def nbytes(self):
        return self.scale.numel() * self.scale.element_size()


@torch.no_grad()
def quantize_fp8_weight(w: torch.Tensor):
    """w [N, K] -> (codes float8_e4m3fn [N, K] in rows of whole 16 bytes, scales fp32 [ceil(N / 128), ceil(K / 128)]): the block's largest
    finite magnitude becomes 448, NaN and infinities NaN codes. Done once, when a weight is loaded."""
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError(f"quantize_fp8_weight takes a matrix that is not empty, got {tuple(w.shape)}")
    N, K = w.shape
    codes = _padded(N, K, w.device)
    scale = torch.empty((_blocks(N), _blocks(K)), dtype=torch.float32, device=w.device)
    for i in range(scale.shape[0]):                       # 128 rows at a time: no fp32 copy of the whole weight
        rows = w[i * BLOCK:(i + 1) * BLOCK].float()
        pad = torch.nn.functional.pad(rows, (0, scale.shape[1] * BLOCK - K)).view(rows.shape[0], -1, BLOCK)
        pad = torch.where(torch.isfinite(pad), pad, float("nan"))
        s = pad.nan_to_num(nan=0.0).abs().amax((0, 2)) / E4M3_MAX
        s = torch.where(s > 0, s, torch.ones_like(s))
        scale[i] = s
        q = (pad / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        codes[i * BLOCK:(i + 1) * BLOCK].copy_(q.view(rows.shape[0], -1)[:, :K])
    return codes, scale


def dequantize_fp8_weight(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """codes [N, K] times their block's scale."""
    _check_weight(codes, scale, "dequantize_fp8_weight")
    from .nf4 import dequantize_fp8_block

    return dequantize_fp8_block(codes, scale, BLOCK, dtype)


def _check_weight(codes, scale, what):
    _check_codes(codes, what)
    _check_scale(scale, (_blocks(codes.shape[0]), _blocks(codes.shape[1])), codes.device, what)


# ------------------------------------------------------------------ products
def fp8_gemm(codes, row_scale, w_codes, w_scale, *, trans_w=False, a2=None, b2=None):
    """bf16 ``x8 W8^T`` (``trans_w``: ``x8 W8``) of quantised rows and a frozen weight, plus ``a2 b2^T`` (``a2 b2``) of a bf16
    K-extension: the low-rank update of an adapter, in the same accumulation."""
    _check_codes(codes, "fp8_gemm")
    _check_weight(w_codes, w_scale, "fp8_gemm")
    M, K = codes.shape
    Kw, N = w_codes.shape if trans_w else w_codes.shape[::-1]
    if K != Kw or w_codes.device != codes.device:
        raise ValueError(f"fp8_gemm: rows of {K} columns on {codes.device} against a weight of {Kw} on {w_codes.device}")
    _check_scale(row_scale, (_blocks(K), M), codes.device, "fp8_gemm")
    K2 = 0
    if a2 is not None or b2 is not None:
        if a2 is None or b2 is None or a2.dim() != 2 or a2.shape[0] != M or tuple(b2.shape) != ((a2.shape[1], N) if trans_w else (N, a2.shape[1])):
            raise ValueError("fp8_gemm: extension " + " x ".join(str(t if t is None else tuple(t.shape)) for t in (a2, b2))
                             + f" for a result [{M}, {N}]")
        if a2.device != codes.device or b2.device != codes.device:
            raise ValueError(f"fp8_gemm: extension on {a2.device} and {b2.device}, codes on {codes.device}")
        K2 = a2.shape[1]
    if not codes.is_cuda:
        w = w_codes.float() * w_scale.repeat_interleave(BLOCK, 0)[:w_codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :w_codes.shape[1]]
        y = dequantize_fp8_rows(codes, row_scale, torch.float32) @ (w if trans_w else w.t())
        if K2:
            y = y + a2.float() @ (b2 if trans_w else b2.t()).float()
        return y.to(torch.bfloat16)
    with _device_of(codes):
        codes, w_codes = _rows16(codes), _rows16(w_codes)
        row_scale, lds = _row_scales(row_scale, M)
        if K2:
            a2, b2 = _operand(a2, "fp8_gemm"), _operand(b2, "fp8_gemm")
        out = torch.empty((M, N), dtype=torch.bfloat16, device=codes.device)
        sn, sk = (w_scale.stride(1), w_scale.stride(0)) if trans_w else w_scale.stride()
        _lib.check_rc(_lib.cuda_lib().axb_fp8_gemm(
            codes.data_ptr(), codes.stride(0), row_scale.data_ptr(), lds, w_codes.data_ptr(), w_codes.stride(0), w_scale.data_ptr(), sn, sk,
            int(trans_w), out.data_ptr(), N, M, N, K, _lib.ptr(a2), a2.stride(0) if K2 else 0, _lib.ptr(b2), b2.stride(0) if K2 else 0, K2,
            _tile(M, N, K), _lib.status_word(codes.device).data_ptr(), _lib.stream_ptr()), "fp8_gemm")
    return out


def _tile(M, N, K) -> int:
    """Tiles of 256 x 256 (256) or 256 x 128 (192) by a CTA pair, or of 128 x 128: waves x (microseconds per block of K + microseconds per
    tile), by least squares over 105 products of 65 to 8192 rows; what it picks is 0.9 % above the best of the three on average (3.5 %
    without the middle one). 361 x 3048 by 6784 33.5 / 26.2 / 34.0 us (128 / 192 / 256), 3600 x 344 by 8304 35.6 / 31.1 / 35.6, 376 x 5512
    by 1304 15.7 / - / 14.8, 636 x 680 by 608 14.6 / - / 15.7, 8192 x 28672 by 4096 993 / - / 830."""
    nk, m1, m2, n1 = (K + 127) >> 7, (M + 127) >> 7, (M + 255) >> 8, (N + 127) >> 7
    small = -(-m1 * n1 // 148) * (0.326 * nk + 0.74) + 1.1
    mid = -(-m2 * n1 // 74) * (0.265 * nk + 0.73) + 1.8
    big = -(-m2 * ((N + 255) >> 8) // 74) * (0.393 * nk + 2.33)
    return 256 if big <= small and big <= mid else 192 if mid <= small else 128


def _few(T, N, K):
    """How the product of a few tokens runs: 2 in one launch, quantising inside (csrc/fp8_skinny.cu), 1 by the same kernel on rows that a
    launch before it has quantised, 0 by tiles. Inside, every CTA quantises the blocks of its part of K, 16 tokens at a time: some
    0.5 us each, against 3 us, most of them the host's, for the launch that does it once. Microseconds among others, inside / before /
    tiles, weights not in the L2: 1 x 4096 by 4096 (4 blocks a CTA, one pass) 10.9 / 15.6 / 17.5; 24 x 2048 by 11264 (6, two) 14.4 / 15.3 /
    15.5; 1 x 14336 by 4096 (14, one) 18.5 / 17.5 / 40.9, 16 tokens 22.6 / 18.6 / 36.7; 64 x 4096 by 4096 (4, four) 18.5 / 15.6 / 16.9; 1 x
    4096 by 28672 (32, one) 31.5 / 24.7 / 43.0; 64 x 14336 by 4096 (14, four) 36.9 / 24.5 / 41.0; 48 x 2048 by 11264 18.8 / 15.5 / 16.0 (on
    the device 18.0 / 14.2 / 12.3) and 64 x 4096 by 28672 66.6 / 34.8 / 30.4, where the tiles fill the chip by themselves. Replayed from a
    graph the launch before is the better one from some 6 blocks on: 24 x 4096 by 4096 11.5 / 10.8."""
    if T > 64:
        return 0
    tiles, nk = (N + 127) >> 7, (K + 127) >> 7
    # axb_cluster_split of csrc/axb_common.cuh
    splits = (8 if tiles <= 33 and nk >= 16 else 6 if tiles <= 44 and nk >= 12 else 5 if tiles <= 50 and nk >= 10 else
              4 if tiles <= 70 and nk >= 8 else 3 if tiles <= 92 and nk >= 6 else 2 if tiles <= 148 and nk >= 4 else 1)
    if -(-nk // splits) * (1 if T <= 16 else 2 if T <= 32 else 4) <= 12:
        return 2
    return 0 if T > 32 and tiles > 70 else 1


_LINEAR = struct.Struct("@9P6q6i")      # AxbFp8Linear of csrc/fp8_gemm.cu


def _product(x, codes, scale, trans=False, a2=None, b2=None, keep=False):
    """(x8 W8^T or x8 W8 (+ a2 b2) in bf16, block of ``_pack`` of x or None) of bf16 rows x [T, K]. One call, and
    for a few tokens whose codes nobody keeps one launch."""
    if not x.is_cuda:
        q = _pack(x)
        y = fp8_gemm(*_unpacked(q, *x.shape), codes, scale, trans_w=trans, a2=a2, b2=b2)
        return y, q
    device = x.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return _product(x, codes, scale, trans, a2, b2, keep)
    T, K = x.shape
    N = codes.shape[1] if trans else codes.shape[0]
    if T == 0:
        return x.new_empty((0, N)), _pack(x) if keep else None
    ldx, unit = x.stride()
    if unit != 1 and K > 1:
        x = x.contiguous()
        ldx = K
    codes = _rows16(codes)
    sn, sk = scale.stride()
    if trans:
        sn, sk = sk, sn
    a, lda, b, ldb, K2 = 0, 0, 0, 0, 0
    if a2 is not None:
        a2, b2 = _operand(a2, "8-bit product"), _operand(b2, "8-bit product")
        a, lda, b, ldb, K2 = a2.data_ptr(), a2.stride(0), b2.data_ptr(), b2.stride(0), a2.shape[1]
    few = 0 if trans or K2 % 8 else _few(T, N, K)
    y = x.new_empty((T, N))
    q = x.new_empty(_packed_size(T, K), dtype=torch.uint8) if keep or few < 2 else None
    status, stream = _lib.launch_args(device.index)
    _lib.check_rc(_lib.cuda_lib().axb_fp8_linear_packed(_LINEAR.pack(
        x.data_ptr(), 0 if q is None else q.data_ptr(), codes.data_ptr(), scale.data_ptr(), y.data_ptr(), a, b, status, stream, ldx,
        codes.stride(0), sn, sk, lda, ldb, T, N, K, K2, 0 if few else _tile(T, N, K), trans)), "fp8_linear")
    return y, q


def _as_codes(w):
    """The codes of a weight given as they are, or as the bytes of a frozen parameter. Autograd then saves the parameter and no view of
    its data, so that data which leave the device between the two passes are not kept alive there."""
    return w.data.view(torch.float8_e4m3fn) if w.dtype == torch.uint8 else w


def _once(backward):
    """A backward pass without a second derivative; the wrapper that refuses one costs the host 2 us and is entered where a graph of the
    backward pass is asked for."""
    refusing = once_differentiable(backward)
    return lambda ctx, dy: (refusing if torch.is_grad_enabled() else backward)(ctx, dy)


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scale, bias):
        y, _ = _product(x, _as_codes(codes), scale)
        if bias is not None:
            y += bias                                     # in place: bf16 whatever the bias is in, and so is the gradient that comes back
        ctx.save_for_backward(codes, scale)               # the weight is frozen: nothing of x is needed again
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        codes, scale = ctx.saved_tensors
        dx = _product(dy, _as_codes(codes), scale, trans=True)[0] if ctx.needs_input_grad[0] else None
        dbias = dy.float().sum(0).to(ctx.bias_dtype) if ctx.needs_input_grad[3] else None
        return dx, None, None, dbias


_LORA = struct.Struct("@17P8q10ifi")      # AxbFp8Lora of csrc/fp8_lora.cu


def _lora_call(entry, x, codes, scale, A16, B16, scaling, sizes, q, xa, y, qx=0, t_parts=0, dB_parts=0, t=0, dA=0, dB=0, dB16=0, blocks=0,
               ldda=0, lddb=0, n_blocks=0, splits=0, add_dA=False, add_dB=False, dA_bf16=False, two=True):
    """One call of csrc/fp8_lora.cu; ``q`` .. ``blocks`` are addresses, ``sizes`` is (T, N, K, R, tile)."""
    status, stream = _lib.launch_args(x.device.index)
    args = _LORA.pack(x.data_ptr(), q, codes.data_ptr(), scale.data_ptr(), A16.data_ptr(), B16.data_ptr(), xa, y, qx, t_parts, dB_parts, t, dA,
                      dB, dB16, blocks, status, x.stride(0), codes.stride(0), *scale.stride(), A16.stride(0), B16.stride(0), ldda, lddb, *sizes,
                      n_blocks, splits, add_dA, add_dB, dA_bf16, scaling, two)
    _lib.check_rc(entry(args, stream), "fp8_lora")


@functools.lru_cache(256)
def _flat_blocks(blocks, N, R):
    """The diagonal blocks (row0, rows, column0, columns) of an adapter's B [N, R] as the kernels take them."""
    if not blocks or any(len(b) != 4 or min(b) < 0 or b[0] + b[1] > N or b[2] + b[3] > R for b in blocks):
        raise ValueError(f"adapter blocks {blocks} of a matrix [{N}, {R}]")
    return (C.c_int * (4 * len(blocks)))(*[int(v) for b in blocks for v in b])


def _lora_forward(x, codes, scale, A16, B16, scaling, keep, two):
    """(y, scaling x A^T, block of ``_pack`` of x or None): one call up to rank 128. Where a gradient may follow, the low-rank product comes
    up to rank 64 as two bf16 numbers [2, T, R], the second what the first leaves of the fp32 sums."""
    if x.device.index != _current_device():
        with torch.cuda.device(x.device):
            return _lora_forward(x, codes, scale, A16, B16, scaling, keep, two)
    T, K = x.shape
    R, N = A16.shape[0], codes.shape[0]
    if R > 128:
        from .lora import skinny_gemm

        xa = skinny_gemm(x, A16, alpha=scaling)            # [T, R], of the bf16 input
        y, q = _product(x, codes, scale, a2=xa, b2=B16, keep=keep)
        return y, xa, q
    few = _few(T, N, K)
    two = two and R <= 64
    y, xa = x.new_empty((T, N)), x.new_empty((2, T, R) if two else (T, R))
    q = x.new_empty(_packed_size(T, K), dtype=torch.uint8) if keep or few < 2 else None
    _lora_call(_lib.cuda_lib().axb_fp8_lora_fwd, x, _rows16(codes), scale, A16, B16, scaling, (T, N, K, R, 0 if few else _tile(T, N, K)),
               0 if q is None else q.data_ptr(), xa.data_ptr(), y.data_ptr(), two=two)
    return y, xa, q


class _Fp8LoRALinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scale, A, B, A16, B16, scaling, blocks, bias):
        y, xa, q = _lora_forward(x, _as_codes(codes), scale, A16, B16, scaling, ctx.needs_input_grad[3], ctx.needs_input_grad[4])
        if bias is not None:
            y += bias
        ctx.save_for_backward(q if ctx.needs_input_grad[3] else None, codes, scale, A, B, A16, B16, xa)
        ctx.scaling, ctx.blocks, ctx.bias_dtype = scaling, blocks, None if bias is None else bias.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        from .lora import USE_FUSED_DY, _adapter_grads, _t_and_dB

        q, codes, scale, A, B, A16, B16, xa = ctx.saved_tensors
        codes = _as_codes(codes)
        need = ctx.needs_input_grad
        dy = _operand(dy, "fp8_lora_linear")
        (T, N), K, R = dy.shape, codes.shape[1], A16.shape[0]
        dbias = dy.float().sum(0).to(ctx.bias_dtype) if need[9] else None
        dx = dA = dB = None
        if need[4] and USE_FUSED_DY and R <= 64 and len(ctx.blocks) <= 8:
            # one pass over dy for t and dB, the product and dA behind it: one call. Scratch: the parts of t and of dB (a CTA of
            # csrc/lora_fused.cu holds 512 rows and one of `splits` ranges of dy's columns), dB in fp32 (where more than 8192 rows are summed
            # into a bf16 one), t as two bf16 numbers, the rows of dy in 8 bits
            tA, tB = getattr(A, "_axb_grad", None), getattr(B, "_axb_grad", None)
            low = [w is None and p.dtype == torch.bfloat16 for w, p in ((tA, A), (tB, B))]
            rows = min(T, 8192)
            chunks = -(-rows // 512)
            splits = min(148 // chunks, _blocks(N))
            at = [4 * splits * rows * R, 4 * chunks * N * R, 4 * N * R if low[1] and T > rows else 0, 4 * T * R]
            work = dy.new_empty(sum(at) + (_packed_size(T, N) if need[0] else 0), dtype=torch.uint8)
            p = work.data_ptr()
            args = dict(t_parts=p, dB_parts=p + at[0], t=p + sum(at[:3]), splits=splits)
            if need[0]:
                dx = dy.new_empty((T, K))
            if low[1]:
                dB = dy.new_empty((N, R))
                args.update(dB=p + at[0] + at[1] if at[2] else 0, dB16=dB.data_ptr(), lddb=R)
            else:
                dB = tB if tB is not None else dy.new_empty((N, R), dtype=torch.float32)
                args.update(dB=dB.data_ptr(), lddb=dB.stride(0), add_dB=tB is not None)
            if need[3] and low[0]:
                dA = dy.new_empty((R, K))
                args.update(qx=q.data_ptr(), dA=dA.data_ptr(), ldda=K, dA_bf16=True)
            elif need[3]:
                dA = tA if tA is not None else dy.new_empty((R, K), dtype=torch.float32)
                args.update(qx=q.data_ptr(), dA=dA.data_ptr(), ldda=dA.stride(0), add_dA=tA is not None)
            flat = _flat_blocks(ctx.blocks, N, R)
            _lora_call(_lib.cuda_lib().axb_fp8_lora_bwd, dy, _rows16(codes), scale, A16, B16, ctx.scaling, (T, N, K, R, _tile(T, K, N)),
                       p + sum(at), xa.data_ptr(), 0 if dx is None else dx.data_ptr(), blocks=C.addressof(flat), n_blocks=len(ctx.blocks), **args)
            dA = None if dA is None or tA is not None else dA if dA.dtype == A.dtype else dA.to(A.dtype)
            dB = None if tB is not None else dB if dB.dtype == B.dtype else dB.to(B.dtype)
            return dx, None, None, dA, dB, None, None, None, None, dbias
        xa = xa[0] if xa.dim() == 3 else xa
        t, dB_fused, dB_done = _t_and_dB(dy, B, B16, xa, ctx.blocks, ctx.scaling, need[4])
        dx = _product(dy, codes, scale, trans=True, a2=t, b2=A16)[0] if need[0] else None
        if need[3]:
            tgt = getattr(A, "_axb_grad", None)
            (ld, lds), at = _lead(T, K), q.data_ptr()
            buf = _adapter_grad(t, at, ld, at + T * ld, lds, K, tgt)
            dA = None if tgt is not None else buf.to(A.dtype)
        _, dB = _adapter_grads(None, B if need[4] else None, t, codes, dy, xa, ctx.blocks, dB_done, dB_fused)
        return dx, None, None, dA, dB, None, None, None, None, dbias


def fp8_adapter_grad(t, codes, row_scale, out=None):
    """``t^T x8`` [R, K] in fp32 for ``t`` [T, R] bf16 and the quantised rows [T, K] that a forward pass kept: the gradient of an adapter's
    A. ``out``: added to it in place."""
    _check_codes(codes, "fp8_adapter_grad")
    T, K = codes.shape
    _check_scale(row_scale, (_blocks(K), T), codes.device, "fp8_adapter_grad")
    if t.dim() != 2 or t.shape[0] != T or t.device != codes.device:
        raise ValueError(f"fp8_adapter_grad: {tuple(t.shape)} on {t.device} for {T} rows on {codes.device}")
    R = t.shape[1]
    if out is not None and (tuple(out.shape) != (R, K) or out.dtype != torch.float32 or out.device != codes.device):
        raise ValueError(f"fp8_adapter_grad: the result is float32 [{R}, {K}] on {codes.device}")
    if not codes.is_cuda:
        x = t.float().t() @ dequantize_fp8_rows(codes, row_scale, torch.float32)
        return x if out is None else out.add_(x)
    if t.dtype != torch.bfloat16:
        raise TypeError(f"fp8_adapter_grad takes bf16 on the device, got {t.dtype}")
    with _device_of(codes):
        codes = _rows16(codes)
        row_scale, lds = _row_scales(row_scale, T)
        if lds % 4 or row_scale.data_ptr() % 16:            # read by bulk copies
            row_scale = torch.nn.functional.pad(row_scale, (0, -T % 4))
            lds = row_scale.shape[1]
        return _adapter_grad(t, codes.data_ptr(), codes.stride(0), row_scale.data_ptr(), lds, K, out)


def _adapter_grad(t, q, ldq, s, lds, K, out):
    """The launch of ``fp8_adapter_grad`` on codes at ``q`` and scales at ``s``."""
    T, R = t.shape
    if T == 0 or R == 0:
        return torch.zeros((R, K), dtype=torch.float32, device=t.device) if out is None else out
    if out is not None and out.stride(1) != 1:
        return out.add_(_adapter_grad(t, q, ldq, s, lds, K, None))
    t = _operand(t, "fp8_adapter_grad")
    add = out is not None
    if not add:
        out = torch.empty((R, K), dtype=torch.float32, device=t.device)
    _lib.check_rc(_lib.cuda_lib().axb_fp8_adapter_grad(
        q, ldq, s, lds, t.data_ptr(), None, t.stride(0), out.data_ptr(), out.stride(0) if R > 1 else K, T, K, R, add,
        _lib.status_word(t.device).data_ptr(), _lib.stream_ptr()), "fp8_adapter_grad")
    return out


def _check_linear(x, codes, scale, bias, what):
    cs, ss = codes.shape, scale.shape
    if bias is not None and (bias.shape != cs[:1] or bias.device != x.device):
        raise ValueError(f"{what}: a bias {tuple(bias.shape)} on {bias.device} for a weight {tuple(cs)} and an input on {x.device}")
    if (len(cs) == 2 and len(ss) == 2 and cs[0] and cs[1] and x.dim() and x.shape[-1] == cs[1]
            and codes.dtype in (torch.float8_e4m3fn, torch.uint8) and scale.dtype == torch.float32 and ss[0] == _blocks(cs[0])
            and ss[1] == _blocks(cs[1]) and x.device == codes.device
            and x.device == scale.device and (x.dtype == torch.bfloat16 or not x.is_cuda)):
        return
    _check_weight(_as_codes(codes), scale, what)
    if 0 in cs or x.dim() < 1 or x.shape[-1] != cs[1]:
        raise ValueError(f"{what}: input {tuple(x.shape)} for a weight {tuple(cs)}")
    if x.device != codes.device:
        raise ValueError(f"{what}: input on {x.device}, weight on {codes.device}")
    raise TypeError(f"{what} takes bf16 on the device, got {x.dtype}")


def _rows_of(x):
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _shaped(y, x):
    y = y if y.dtype == x.dtype else y.to(x.dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[-1])


def _no_rows(x, codes, bias, A=None, B=None):
    """The result of no rows, connected to all that learns."""
    y = x[..., :1].expand(*x.shape[:-1], codes.shape[0])
    if A is not None:
        y = y + (x @ A.to(x.dtype).t()) @ B.to(x.dtype).t()
    return y if bias is None else y + bias.to(x.dtype)


def fp8_linear(x, codes, scale, bias=None):
    """``x8 W8^T (+ bias)`` of a frozen block-FP8 weight (codes [N, K], float8_e4m3fn or the same as bytes, and scales [ceil(N / 128),
    ceil(K / 128)]); ``x`` [..., K] in bf16. The input gradient is ``dy8 W8``; nothing of ``x`` is kept for it."""
    _check_linear(x, codes, scale, bias, "fp8_linear")
    if x.numel() == 0:
        return _no_rows(x, codes, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return _shaped(_Fp8LinearFn.apply(_rows_of(x), codes, scale, bias), x)
    y = _product(x if x.dim() == 2 else _rows_of(x), _as_codes(codes), scale)[0]
    if bias is not None:
        y += bias
    return y if x.dim() == 2 and y.dtype == x.dtype else _shaped(y, x)


def fp8_lora_linear(x, codes, scale, A, B, A16, B16, scaling, blocks, bias=None):
    """``x8 W8^T + scaling (x A^T) B^T (+ bias)``: ``fp8_linear`` with the adapter of ``ops.lora.lora_linear`` (same arguments). The 8-bit
    rows of ``x`` are kept for ``dA = (scaling dy B)^T x8``."""
    _check_linear(x, codes, scale, bias, "fp8_lora_linear")
    if x.numel() == 0:
        return _no_rows(x, codes, bias, A, B)
    x2 = _rows_of(x)
    if not x.is_cuda:
        y = _Fp8LinearFn.apply(x2, codes, scale, bias).to(x.dtype)
        return _shaped(y + scaling * ((x2 @ A.to(x2.dtype).t()) @ B.to(x2.dtype).t()), x)
    N, K = codes.shape
    R = A.shape[0]
    if (A.shape != (R, K) or B.shape != (N, R) or A16.shape != A.shape or B16.shape != B.shape or A16.dtype != torch.bfloat16
            or B16.dtype != torch.bfloat16 or not x.device == A.device == B.device == A16.device == B16.device):
        raise ValueError(f"fp8_lora_linear: adapter {tuple(A.shape)} {tuple(B.shape)} with bf16 copies {A16.dtype} {tuple(A16.shape)} "
                         f"{B16.dtype} {tuple(B16.shape)} for a weight [{N}, {K}] on {x.device}")
    if R % 8:
        raise ValueError(f"fp8_lora_linear: rank {R}, the device path needs a multiple of 8 (16-byte rows for the bulk tensor copies)")
    blocks = tuple(map(tuple, blocks))
    _flat_blocks(blocks, N, R)
    x2, A16, B16 = (_operand(t, "fp8_lora_linear") for t in (x2, A16, B16))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, A, B, bias)):
        return _shaped(_Fp8LoRALinearFn.apply(x2, codes, scale, A, B, A16, B16, float(scaling), blocks, bias), x)
    y = _lora_forward(x2, _as_codes(codes), scale, A16, B16, float(scaling), False, False)[0]
    if bias is not None:
        y += bias
    return _shaped(y, x)
