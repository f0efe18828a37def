"""Linears with 4-bit weights and group scales: ``mm_w4`` beside ``neokernel_b200.mm``.

    y[m, n] = bf16( sum_k x[m, k] * (q[n, k] - z[n, k // group]) * s[n, k // group] )

``W4Weight`` holds a weight in the kernel's storage (``include/nk_quant.h``): made once, when the
weights are loaded, from codes and scales (``pack``) or from a bf16 weight (``quantize``).
``mm_w4(x, w, out=y)`` takes it where ``mm(x, W.t(), out=y)`` takes ``W.t()``, with the same
conventions: the current stream, no allocation, no host synchronisation, capture-safe,
``ValueError`` before launching for an unsupported configuration. It needs no plan and no
workspace.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gemm import _raise, mm

GROUPS = (32, 64, 128)
_SCALE_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


class W4Weight:
    """A [N, K] weight as 4-bit codes with a scale (and a zero point) per row and group of K.

    Made by ``pack`` or ``quantize``; the arrays are not to be written afterwards, as a launch
    reads them ahead of the work queued before it on its stream.
    """

    __slots__ = ("N", "K", "group", "codes", "scales", "zeros", "scale_type", "device", "_c",
                 "_addr")

    def __init__(self, N, K, group, codes, scales, zeros, scale_type):
        self.N, self.K, self.group = N, K, group
        self.codes, self.scales, self.zeros, self.scale_type = codes, scales, zeros, scale_type
        self.device = codes.device
        self._c = _lib.NkW4Weight(codes.data_ptr(), scales.data_ptr(),
                                  zeros.data_ptr() if zeros is not None else None, N, K, group,
                                  scale_type)
        self._addr = ctypes.addressof(self._c)

    @property
    def shape(self):
        """Of the operand ``W.t()``: [K, N], as ``mm``'s second argument has it."""
        return (self.K, self.N)

    @property
    def nbytes(self):
        return (self.codes.nbytes + self.scales.nbytes
                + (self.zeros.nbytes if self.zeros is not None else 0))

    @classmethod
    def pack(cls, q, scales, zeros=None, *, K, group):
        """Lay out codes ``q`` (uint8 [N, ceil(K / 2)], element 2i in the low half of byte i),
        ``scales`` (bf16 or fp16 [N, ceil(K / group)]) and ``zeros`` (uint8 of the same shape,
        0..15; None: 8 throughout). Load time: waits for the device."""
        _need(group in GROUPS, f"W4Weight: group must be one of {GROUPS}, got {group}")
        _need(isinstance(q, torch.Tensor) and q.dtype == torch.uint8 and q.dim() == 2,
              "W4Weight: q must be a uint8 [N, ceil(K / 2)] tensor")
        N, G = q.shape[0], -(-K // group)
        _need(N >= 1 and K >= 1 and q.shape[1] == -(-K // 2),
              f"W4Weight: q is {tuple(q.shape)} for K={K}")
        _need(scales.dtype in _SCALE_TYPES, "W4Weight: scales must be bfloat16 or float16")
        _need(tuple(scales.shape) == (N, G) and scales.device == q.device,
              f"W4Weight: scales must be [{N}, {G}] on q's device, got {tuple(scales.shape)}")
        if zeros is not None:
            _need(zeros.dtype == torch.uint8 and tuple(zeros.shape) == (N, G)
                  and zeros.device == q.device,
                  f"W4Weight: zeros must be uint8 [{N}, {G}] on q's device")
            _need(int(zeros.max()) <= 15, "W4Weight: zero points must be 0..15")
        NB, KB = -(-N // 128), -(-K // 128)
        codes = torch.zeros(NB * 128, KB * 128, dtype=torch.uint8, device=q.device)
        codes[:N, 0:K:2] = q & 15
        codes[:N, 1:K:2] = (q >> 4)[:, :K // 2]
        # [tile, row, step, piece, word, element] -> [tile, step, piece, row, word], by byte
        c = codes.view(NB, 128, KB, 4, 4, 8).permute(0, 2, 3, 1, 4, 5)
        codes = torch.stack([c[..., a] | (c[..., b] << 4) for a, b in ((0, 2), (4, 6), (1, 3), (5, 7))],
                            dim=-1).contiguous().view(-1)

        def rows(t):  # [N, G] -> [tile, group, row]
            p = torch.zeros(NB * 128, KB * 128 // group, dtype=t.dtype, device=t.device)
            p[:N, :G] = t
            return p.view(NB, 128, -1).transpose(1, 2).contiguous().view(-1)

        w = cls(N, K, group, codes, rows(scales), rows(zeros) if zeros is not None else None,
                _SCALE_TYPES[scales.dtype])
        if q.is_cuda:
            torch.cuda.synchronize(q.device)  # launches read the weights ahead of their stream
        return w

    @classmethod
    def quantize(cls, weight, group=128, *, zeros=False, scale_dtype=torch.bfloat16):
        """Round a row-major [N, K] ``weight`` to 4 bits, nearest code of each group's range:
        symmetric around code 8, or with a zero point per group (``zeros``). Load time."""
        _need(isinstance(weight, torch.Tensor) and weight.dim() == 2 and weight.is_floating_point(),
              "W4Weight: weight must be a [N, K] floating-point tensor")
        _need(group in GROUPS, f"W4Weight: group must be one of {GROUPS}, got {group}")
        _need(scale_dtype in _SCALE_TYPES, "W4Weight: scales must be bfloat16 or float16")
        N, K = weight.shape
        G = -(-K // group)
        w = torch.zeros(N, G * group, dtype=torch.float32, device=weight.device)
        w[:, :K] = weight
        w = w.view(N, G, group)
        if zeros:
            lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
            s = ((hi - lo) / 15.0).to(scale_dtype)
            sf = torch.where(s > 0, s.float(), torch.ones_like(lo))
            z = torch.round(-lo / sf).clamp(0, 15)
        else:
            s = (w.abs().amax(-1) / 7.0).to(scale_dtype)
            sf = torch.where(s > 0, s.float(), torch.ones_like(w[..., 0]))
            z = torch.full_like(sf, 8.0)
        _need(bool(s.isfinite().all()), "W4Weight: weight must be finite, and its groups' scales "
              f"within {scale_dtype}")
        q = (torch.round(w / sf[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8)
        q = q.view(N, -1)[:, :K]
        if K % 2:
            q = torch.cat((q, torch.zeros_like(q[:, :1])), dim=1)
        return cls.pack(q[:, 0::2] | (q[:, 1::2] << 4), s, z.to(torch.uint8) if zeros else None,
                        K=K, group=group)

    def dequantize(self):
        """The weight it stands for, fp32 [N, K]."""
        NB, KB = -(-self.N // 128), -(-self.K // 128)
        b = self.codes.view(NB, KB, 4, 128, 4, 4)  # tile, step, piece, row, word, byte
        lo, hi = b & 15, b >> 4
        e = torch.stack((lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2],
                         lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]), dim=-1)
        q = e.permute(0, 3, 1, 2, 4, 5).reshape(NB * 128, KB * 128).float()

        def rows(t):
            t = t.view(NB, -1, 128).transpose(1, 2).reshape(NB * 128, -1).float()
            return t.repeat_interleave(self.group, dim=1)

        z = rows(self.zeros) if self.zeros is not None else 8.0
        return ((q - z) * rows(self.scales))[:self.N, :self.K]

    def __repr__(self):
        return (f"W4Weight(N={self.N}, K={self.K}, group={self.group}, "
                f"zeros={self.zeros is not None}, device={self.device})")


_BF16 = torch.bfloat16
_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(dev).cuda_stream, without the object


def mm_w4(a: torch.Tensor, w: W4Weight, *, out: torch.Tensor,
          stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """``out = a @ W.t()`` for a 4-bit weight ``w`` of W [N, K]: fp32 sums, one bf16 rounding.

    a: bf16 CUDA [M, K] with unit column stride; out: bf16 CUDA [M, N] with unit column stride, in
    memory that ``a`` does not share.
    Any M; made for decode batches and drafts of up to 64 tokens. Larger ones read and widen the
    weights once per 64 tokens: from some 128 tokens on (64 with groups of 32) ``mm`` with the bf16
    weight is faster, and a model that is not short of memory keeps that for them.
    """
    if not isinstance(w, W4Weight):
        raise ValueError(f"mm_w4: w must be a W4Weight, got {type(w).__name__}")
    if not (isinstance(a, torch.Tensor) and isinstance(out, torch.Tensor) and a.dtype is _BF16
            and out.dtype is _BF16 and a.dim() == 2 and out.dim() == 2):
        raise ValueError("mm_w4: a and out must be 2-D bfloat16 tensors")
    dev = w.device
    if not a.is_cuda or a.device != dev or out.device != dev:
        raise ValueError(f"mm_w4: a, w and out must be on the same CUDA device (a on {a.device}, "
                         f"w on {dev}, out on {out.device})")
    M, K = a.shape
    N = w.N
    if K != w.K:
        raise ValueError(f"mm_w4: a is [{M}, {K}] but w is [{w.K}, {N}]")
    if out.shape != (M, N):
        raise ValueError(f"mm_w4: out must be [{M}, {N}], got {tuple(out.shape)}")
    if M == 0:
        return out
    ldx, ca = a.stride()
    ldy, co = out.stride()
    if (ca != 1 and K > 1) or (co != 1 and N > 1):
        raise ValueError("mm_w4: a and out must have unit stride along their last dimension")
    if M == 1:
        ldx, ldy = K, N
    elif ldx < K or ldy < N:
        raise ValueError("mm_w4: rows of a and of out must not overlap")
    index = dev.index
    handle = _raw_stream(index) if stream is None else stream.cuda_stream
    fn = _lib.load().nk_gemm_w4
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            status = fn(a.data_ptr(), ldx, w._addr, out.data_ptr(), ldy, M, handle)
    else:
        status = fn(a.data_ptr(), ldx, w._addr, out.data_ptr(), ldy, M, handle)
    if status:
        _raise(status, f"nk_gemm_w4(M={M}, N={N}, K={K})")
    return out


def linear(a: torch.Tensor, b, *, out: torch.Tensor) -> torch.Tensor:
    """``out = a @ b`` for a ``W4Weight`` (``mm_w4``) or a bf16 ``W.t()`` (``mm``): the ``linear``
    of a decode step whose layers are in 4 bits and whose lm_head is not. (The tensor-parallel
    hooks sum unrounded partials of o_proj and down, which ``mm_w4`` does not give: they take bf16
    weights.)"""
    if isinstance(b, W4Weight):
        return mm_w4(a, b, out=out)
    return mm(a, b, out=out)
