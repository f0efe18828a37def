"""Python face of the fused decode kernels (include/nk_decode.h).

Same conventions as ``neokernel_b200.mm``: caller-owned CUDA tensors, launch on the current
stream, ``ValueError`` before launching for an unsupported configuration, no allocation, no
host synchronisation. Each replaces one of the reference engine's Triton wrappers:

* ``rmsnorm``            <- ``norm_out``            (engine/kernels/rmsnorm.py:28-41)
* ``qk_norm_rope_cache`` <- ``qk_rope_cache_out``   (engine/kernels/elementwise.py:63-78)
* ``qkv_rope_cache``     <- ``torch.mm(norm, w.qkv, out=qkv)`` + ``qk_rope_cache_out``
                            (engine/kernels/decode.py:54-55): the QKV linear and its consumer
                            in one launch, qkv never stored
* ``attention_decode``   <- ``attention_out``       (engine/kernels/attention.py:53-62)
* ``silu_mul``           <- ``silu_mul_out``        (engine/kernels/elementwise.py:91-101)

The KV cache can also be held in 8 bits (include/nk_quant.h; the reference has no such form):

* ``Q8Cache``                 e4m3 keys and values with a power-of-two scale per (sequence, kv
                              head, block of tokens)
* ``qk_norm_rope_cache_q8``   ``qk_norm_rope_cache`` appending to a ``Q8Cache``
* ``attention_decode_q8``     ``attention_decode`` over a ``Q8Cache``

Both take per-sequence positions, idle sequences and up to 16 new tokens a sequence.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .gemm import _raise

HEAD_DIM = 128


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _bf16_cuda(*ts):
    for t in ts:
        _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.bfloat16,
              "decode ops take bf16 CUDA tensors")


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, eps: float,
            branch: torch.Tensor | None = None) -> torch.Tensor:
    """out = bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight); with ``branch``, first
    x <- bf16(x + branch) in place (the fused residual add of the reference's
    ``norm_out(branch, w, out, eps, x, x)``)."""
    _bf16_cuda(x, weight, out, *([branch] if branch is not None else []))
    _need(x.dim() == 2 and x.is_contiguous() and out.shape == x.shape and out.is_contiguous(),
          "rmsnorm: x and out must be contiguous [rows, width]")
    _need(branch is None or (branch.shape == x.shape and branch.is_contiguous()),
          "rmsnorm: branch must match x")
    st = _lib.load().nk_rmsnorm_bf16(x.data_ptr(), branch.data_ptr() if branch is not None else None,
                                      weight.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1],
                                      float(eps), _stream(x))
    if st != _lib.NK_OK:
        _raise(st, "nk_rmsnorm_bf16")
    return out


def qk_norm_rope_cache(qkv, q_norm, k_norm, cos, sin, position, q_out, k_cache, v_cache,
                       heads: int, kv_heads: int, eps: float):
    """Q/K head RMSNorm + RoPE at ``position`` (device int64 [1]); queries to ``q_out``
    [B, heads*128], keys and values into the [B, kv_heads, capacity, 128] caches. A position
    outside the caches writes nothing and is reported by ``device_error()``."""
    _bf16_cuda(qkv, q_norm, k_norm, cos, sin, q_out, k_cache, v_cache)
    _need(position.is_cuda and position.dtype == torch.int64, "position: CUDA int64 tensor")
    B = qkv.shape[0]
    _need(qkv.stride(1) == 1 and q_out.is_contiguous() and cos.is_contiguous()
          and sin.is_contiguous() and k_cache.stride(3) == 1 and v_cache.stride() == k_cache.stride(),
          "qk_norm_rope_cache: unsupported layout")
    st = _lib.load().nk_qk_norm_rope_cache_bf16(
        qkv.data_ptr(), qkv.stride(0), q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(),
        sin.data_ptr(), position.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), B, heads, kv_heads, HEAD_DIM, k_cache.shape[2], k_cache.stride(0),
        k_cache.stride(1), k_cache.stride(2), float(eps), _stream(qkv))
    if st != _lib.NK_OK:
        _raise(st, "nk_qk_norm_rope_cache_bf16")


def qkv_rope_cache(x, w_qkv_t, q_norm, k_norm, cos, sin, position, q_out, k_cache, v_cache,
                   heads: int, kv_heads: int, eps: float, plan=None):
    """``qk_norm_rope_cache`` of ``x @ w_qkv_t`` without storing the product: the QKV linear
    (``w_qkv_t`` = Wqkv.t() of the packed row-major weight, as ``mm`` takes it) whose kernel
    finishes each 128-row head tile with that head's RMSNorm + RoPE and writes queries, keys
    and values where the attention reads them. Same bits as ``mm`` then
    ``qk_norm_rope_cache``. Decode batches of up to 16 tokens."""
    from . import gemm
    gemm._check_tensor(x, "x")
    gemm._check_tensor(w_qkv_t, "w_qkv_t")
    _bf16_cuda(q_norm, k_norm, cos, sin, q_out, k_cache, v_cache)
    _need(position.is_cuda and position.dtype == torch.int64, "position: CUDA int64 tensor")
    M, K = x.shape
    K2, N = w_qkv_t.shape
    _need(K2 == K and N == (heads + 2 * kv_heads) * HEAD_DIM,
          f"qkv_rope_cache: x [{M}, {K}] and w_qkv_t [{K2}, {N}] for {heads}+2x{kv_heads} heads")
    _need(1 <= M <= 16, "qkv_rope_cache: decode batches of 1 to 16 tokens")
    _need(x.stride(1) == 1 and w_qkv_t.stride(0) == 1 and q_out.is_contiguous()
          and cos.is_contiguous() and sin.is_contiguous() and k_cache.stride(3) == 1
          and v_cache.stride() == k_cache.stride(), "qkv_rope_cache: unsupported layout")
    plan = plan or gemm.plan_for(M, N, K)
    dev = x.device
    stream = torch.cuda.current_stream(dev)
    ws = gemm.workspace(plan.ws_bytes, dev, stream) if plan.ws_bytes else None
    st = _lib.load().nk_gemm_bf16_qkv_rope_cache(
        x.data_ptr(), x.stride(0) if M > 1 else K, w_qkv_t.data_ptr(), w_qkv_t.stride(1), M, N, K,
        plan._ref, ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
        q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(), position.data_ptr(),
        q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), heads, kv_heads,
        k_cache.shape[2], k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), float(eps),
        stream.cuda_stream)
    if st != _lib.NK_OK:
        _raise(st, "nk_gemm_bf16_qkv_rope_cache")


def attention_workspace(batch: int, heads: int, capacity: int, device) -> torch.Tensor:
    n = _lib.load().nk_attention_ws_bytes(batch, heads, capacity)
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=device)


def attention_decode(q, k_cache, v_cache, position, out, ws, heads: int, kv_heads: int,
                     scale: float | None = None):
    """Grouped split-KV decode attention over slots [0, position]: q, out [B, heads*128]."""
    _bf16_cuda(q, k_cache, v_cache, out)
    _need(q.is_contiguous() and out.is_contiguous() and k_cache.stride(3) == 1
          and v_cache.stride() == k_cache.stride(), "attention_decode: unsupported layout")
    B, cap = q.shape[0], k_cache.shape[2]
    scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else scale
    st = _lib.load().nk_attention_decode_bf16(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), position.data_ptr(),
        out.data_ptr(), B, heads, kv_heads, HEAD_DIM, cap, k_cache.stride(0), k_cache.stride(1),
        k_cache.stride(2), float(scale), ws.data_ptr(), ws.numel(), _stream(q))
    if st != _lib.NK_OK:
        _raise(st, "nk_attention_decode_bf16")


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor):
    """out = bf16(bf16(silu(gate)) * up) for gate_up = [gate | up] rows."""
    _bf16_cuda(gate_up, out)
    _need(gate_up.is_contiguous() and out.is_contiguous()
          and gate_up.shape[1] == 2 * out.shape[1] and gate_up.shape[0] == out.shape[0],
          "silu_mul: gate_up [rows, 2I] and out [rows, I] contiguous")
    st = _lib.load().nk_silu_mul_bf16(gate_up.data_ptr(), out.data_ptr(), out.shape[0],
                                       out.shape[1], _stream(out))
    if st != _lib.NK_OK:
        _raise(st, "nk_silu_mul_bf16")


Q8_MAX_TOKENS = 16   # new tokens per sequence and call (NK_Q8_MAX_TOKENS)
Q8_MAX_BATCH = 1024  # NK_Q8_MAX_BATCH
Q8_BLOCKS = (16, 32, 64, 128)


def _meets(dims, lo: int, hi: int) -> bool:
    """Whether some sum of i * stride over the (stride, count) pairs ``dims`` (largest stride first),
    0 <= i < count, lies strictly between ``lo`` and ``hi``."""
    if not dims:
        return lo < 0 < hi
    (stride, count), rest = dims[0], dims[1:]
    first = max(lo // stride + 1, 0)            # the least i whose own multiple is past lo
    if first < count and first * stride < hi:
        return True
    reach = sum(s * (n - 1) for s, n in rest)   # smaller ones can still get there with the others' help
    least = max((lo - reach) // stride + 1, 0)
    return any(_meets(rest, lo - i * stride, hi - i * stride)
               for i in range(least, min(first, count)))


class Q8Cache:
    """A layer's KV cache in 8 bits: e4m3 codes ``k``, ``v`` [batch, kv_heads, capacity, 128] and
    fp32 scales ``k_scale``, ``v_scale`` [batch, kv_heads, ceil(capacity / block)]; the value held
    at slot j is ``k[..., j, :] * k_scale[..., j // block]``. The codes may have any batch, head
    and token strides that are multiples of 16, the same for ``k`` and ``v``; the scales are
    contiguous, and no two of the four share memory (keys and values may lie between each other's rows,
    as in one [.., 2, 128] tensor). The tensors are the caller's and are read and written in place."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "block", "batch", "kv_heads", "capacity",
                 "device", "_c", "_addr")

    def __init__(self, k, v, k_scale, v_scale, block: int):
        for t in (k, v):
            _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float8_e4m3fn
                  and t.dim() == 4 and t.shape[3] == HEAD_DIM,
                  "Q8Cache: k and v must be float8_e4m3fn CUDA tensors [batch, kv_heads, "
                  "capacity, 128]")
        _need(v.shape == k.shape and v.stride() == k.stride() and v.device == k.device,
              "Q8Cache: k and v must have the same shape, strides and device")
        _need(block in Q8_BLOCKS, f"Q8Cache: block must be one of {Q8_BLOCKS}, got {block}")
        B, H, S, _ = k.shape
        _need(1 <= B <= Q8_MAX_BATCH and H >= 1 and S >= 1,
              f"Q8Cache: batch 1..{Q8_MAX_BATCH}, kv_heads >= 1 and capacity >= 1")
        sb, sh, ss, sd = k.stride()
        # sorted by stride, each dimension starts past the extent of the ones below it
        extent, dense = HEAD_DIM, sd == 1
        for st, n in sorted((st, n) for st, n in ((sb, B), (sh, H), (ss, S)) if n > 1):
            dense = dense and st >= extent and st % 16 == 0
            extent = st * n
        _need(dense and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0,
              "Q8Cache: unsupported layout (unit stride along the head, other strides multiples "
              "of 16 that do not overlap, 16-byte aligned)")
        shape = (B, H, -(-S // block))
        for t in (k_scale, v_scale):
            _need(isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.device == k.device
                  and tuple(t.shape) == shape and t.is_contiguous(),
                  f"Q8Cache: scales must be contiguous fp32 {list(shape)} on the codes' device")
        _need(abs(v_scale.data_ptr() - k_scale.data_ptr()) >= k_scale.nbytes,
              "Q8Cache: k_scale and v_scale must not share memory")
        # rows of 128 bytes at these strides; between two of them, the differences of two indexes
        dims = sorted(((st, n) for st, n in ((sb, B), (sh, H), (ss, S)) if n > 1), reverse=True)
        mid = v.data_ptr() - k.data_ptr() + sum(st * (n - 1) for st, n in dims)
        _need(not _meets([(st, 2 * n - 1) for st, n in dims], mid - HEAD_DIM, mid + HEAD_DIM),
              "Q8Cache: k and v must not share memory")
        for t in (k, v):
            for s in (k_scale, v_scale):
                at = s.data_ptr() - t.data_ptr()
                _need(not _meets(dims, at - HEAD_DIM, at + s.nbytes),
                      "Q8Cache: codes and scales must not share memory")
        self.k, self.v, self.k_scale, self.v_scale, self.block = k, v, k_scale, v_scale, block
        self.batch, self.kv_heads, self.capacity, self.device = B, H, S, k.device
        self._c = _lib.NkQ8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                 B, H, HEAD_DIM, S, block, 0, sb if B > 1 else 0,
                                 sh if H > 1 else 0, ss if S > 1 else HEAD_DIM)
        self._addr = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, device, block: int = 64,
              layout: str = "bhsd"):
        """A zeroed cache; ``layout`` "bhsd" keeps a head's tokens adjacent, "bshd" a token's
        heads (the reference supports both for its bf16 cache)."""
        _need(layout in ("bhsd", "bshd"), f"Q8Cache: layout must be bhsd or bshd, not {layout!r}")
        _need(block in Q8_BLOCKS, f"Q8Cache: block must be one of {Q8_BLOCKS}, got {block}")

        def codes():
            shape = ((batch, kv_heads, capacity) if layout == "bhsd"
                     else (batch, capacity, kv_heads))
            t = torch.zeros(*shape, HEAD_DIM, dtype=torch.uint8, device=device)
            return (t if layout == "bhsd" else t.transpose(1, 2)).view(torch.float8_e4m3fn)

        def scales():
            return torch.zeros(batch, kv_heads, -(-capacity // block), dtype=torch.float32,
                               device=device)

        return cls(codes(), codes(), scales(), scales(), block)

    def zero_(self):
        for t in (self.k, self.v):
            t.view(torch.uint8).zero_()
        self.k_scale.zero_()
        self.v_scale.zero_()
        return self

    def dequantize(self):
        """Keys and values, fp32 [batch, kv_heads, capacity, 128]."""
        def full(codes, scale):
            return codes.float() * scale.repeat_interleave(self.block, dim=2)[:, :, :self.capacity,
                                                                              None]
        return full(self.k, self.k_scale), full(self.v, self.v_scale)


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(dev).cuda_stream, without the object
_BF16, _INT64 = torch.bfloat16, torch.int64


def _q8_tokens(x, cache, width, name):
    """New tokens per sequence of a [batch * tokens, width] bf16 operand."""
    if not (isinstance(x, torch.Tensor) and x.dtype is _BF16 and x.dim() == 2
            and x.device == cache.device):
        raise ValueError(f"{name} must be a 2-D bf16 tensor on the cache's device")
    rows, cols = x.shape
    T, rest = divmod(rows, cache.batch)
    if rest or cols != width or not 1 <= T <= Q8_MAX_TOKENS or T > cache.capacity:
        raise ValueError(f"{name} must be [batch * tokens, {width}] for batch {cache.batch}, tokens "
                         f"1..{Q8_MAX_TOKENS} within the capacity {cache.capacity}, got "
                         f"[{rows}, {cols}]")
    return T


def _q8_position(position, cache, name):
    """1 if the int64 ``position`` has an entry per sequence, 0 if one for all."""
    if (isinstance(position, torch.Tensor) and position.dtype is _INT64 and position.dim() == 1
            and position.device == cache.device and position.is_contiguous()):
        n = position.numel()
        if n == cache.batch:
            return 1
        if n == 1:
            return 0
    raise ValueError(f"{name}: position must be a contiguous int64 tensor [1] or [{cache.batch}] on "
                     "the cache's device")


def _on(device, fn, args):
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return fn(*args)
    return fn(*args)


def qk_norm_rope_cache_q8(qkv, q_norm, k_norm, cos, sin, position, q_out, cache: Q8Cache,
                          heads: int, eps: float):
    """``qk_norm_rope_cache`` for T = 1..16 new tokens per sequence, appending to a ``Q8Cache``.

    qkv [batch * T, (heads + 2 kv_heads) * 128] (row b * T + t, unit column stride); ``position``
    [batch] (or [1], shared): slot of each sequence's first new token, negative for an idle
    sequence, of which nothing is read or written. q_out [batch * T, heads * 128] contiguous, not
    in qkv's memory. A
    block's scale is the smallest power of two that keeps its new tokens within e4m3's range,
    and at least its former one where it holds earlier tokens; these are rounded anew when it
    rises. A position past capacity - T is an idle sequence too and is reported by
    ``device_error()``. ``heads`` is 1 to 16 times the cache's kv_heads."""
    name = "qk_norm_rope_cache_q8"
    Hkv, dev = cache.kv_heads, cache.device
    T = _q8_tokens(qkv, cache, (heads + 2 * Hkv) * HEAD_DIM, "qk_norm_rope_cache_q8: qkv")
    if _q8_tokens(q_out, cache, heads * HEAD_DIM, "qk_norm_rope_cache_q8: q_out") != T \
            or not q_out.is_contiguous():
        raise ValueError(f"{name}: q_out must be contiguous, with as many rows as qkv")
    per = _q8_position(position, cache, name)
    ld, unit = qkv.stride()
    if T * cache.batch == 1:
        ld = qkv.shape[1]
    if unit != 1 or ld < qkv.shape[1]:
        raise ValueError(f"{name}: qkv rows must have unit column stride and not overlap")
    for t in (q_norm, k_norm):
        if not (isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.device == dev
                and t.shape == (HEAD_DIM,) and t.is_contiguous()):
            raise ValueError(f"{name}: q_norm and k_norm must be contiguous bf16 [128] on the "
                             "cache's device")
    for t in (cos, sin):
        if not (isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.device == dev
                and t.dim() == 2 and t.shape[1] == HEAD_DIM and t.shape[0] >= cache.capacity
                and t.is_contiguous()):
            raise ValueError(f"{name}: cos and sin must be contiguous bf16 [capacity, 128] on the "
                             "cache's device")
    status = _on(dev, _lib.load().nk_qk_norm_rope_cache_q8, (
        qkv.data_ptr(), ld, q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        position.data_ptr(), per, q_out.data_ptr(), cache._addr, T, heads, eps,
        _raw_stream(dev.index)))
    if status:
        _raise(status, "nk_qk_norm_rope_cache_q8")
    return q_out


def attention_q8_workspace(cache: Q8Cache, heads: int, tokens: int = 1) -> torch.Tensor:
    """Workspace of ``attention_decode_q8`` for up to ``tokens`` new tokens per sequence, on the
    cache's device. Its size does not depend on the batch or the capacity, so the layers of a
    model, whose calls are ordered, share one. Two streams (or graphs) that may run at once need
    one each."""
    n = int(_lib.load().nk_attention_q8_ws_bytes(tokens, heads, cache.kv_heads))
    _need(n > 0, f"attention_q8_workspace: tokens 1..{Q8_MAX_TOKENS}, heads 1..16 times "
                 f"{cache.kv_heads}; got tokens={tokens}, heads={heads}")
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


_ATTN_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def attention_decode_q8(q, cache: Q8Cache, position, out, ws, heads: int,
                        scale: float | None = None):
    """``attention_decode`` of T = 1..16 new tokens per sequence over a ``Q8Cache`` that already
    holds them: row b * T + t of q, out [batch * T, heads * 128] attends over slots
    [0, position[b] + t]. ``position`` as in ``qk_norm_rope_cache_q8``; rows of idle sequences
    come out zero. ``heads`` is 1 to 16 times the cache's kv_heads. fp32 throughout but for the
    probabilities and the queries as the matrix instructions take them (f16; include/nk_quant.h says
    what that keeps)."""
    name = "attention_decode_q8"
    T = _q8_tokens(q, cache, heads * HEAD_DIM, "attention_decode_q8: q")
    if _q8_tokens(out, cache, heads * HEAD_DIM, "attention_decode_q8: out") != T \
            or not (q.is_contiguous() and out.is_contiguous()):
        raise ValueError(f"{name}: q and out must be contiguous and of the same shape")
    per = _q8_position(position, cache, name)
    if not (isinstance(ws, torch.Tensor) and ws.device == cache.device and ws.is_contiguous()):
        raise ValueError(f"{name}: ws must be a workspace on the cache's device")
    status = _on(cache.device, _lib.load().nk_attention_decode_q8, (
        q.data_ptr(), cache._addr, position.data_ptr(), per, out.data_ptr(), T, heads,
        _ATTN_SCALE if scale is None else scale, ws.data_ptr(), ws.nbytes,
        _raw_stream(cache.device.index)))
    if status:
        _raise(status, "nk_attention_decode_q8")
    return out
