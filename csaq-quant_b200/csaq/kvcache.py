"""csaq.kvcache — a quantised KV cache and the attention that reads it.

The reference keeps the HF module's cache in the model's dtype; this is the
package's own extension for long contexts and large batches: keys and values
as 8- or 4-bit codes with one scale and zero point per (token, head, group of
head elements), a half or a quarter of the bytes that decode attention has to
read. ``DecodeRuntime(..., kv_bits=8)`` uses it for a whole model; the class
below is one layer's cache for callers with a loop of their own. It is for
inference: no call records a gradient, whatever its inputs require.

Token (b, s) of a step is row ``b*S + s`` of its matrices and sits at position
``pos0[b] + s``, as everywhere in the package.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import CsaqKvqCache, check, dtype_code, lib, ptr, raw_stream

__all__ = ["KVWorkspace", "QuantizedKVCache", "cache_positions"]


_CODES = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}


def cache_positions(n: int) -> int:
    """The cache length that holds n positions (the kernels want a multiple of 16)."""
    return (int(n) + 15) // 16 * 16


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """t and its row stride when the kernels can read its rows where they are, else a copy's."""
    ld, one = t.stride()
    if t.shape[0] == 1:  # of a single row the stride says nothing
        ld = t.shape[1]
    if one != 1 or ld % 8 or ld < t.shape[1] or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:  # a contiguous view at an odd offset
            t = t.clone()
        ld = t.shape[1]
    return t, ld


@dataclass
class KVWorkspace:
    """Scratch of ``QuantizedKVCache.attend``: calls that share one must be
    ordered on the GPU (one stream, or one captured graph replayed at a time)."""

    part: torch.Tensor


class QuantizedKVCache:
    """One layer's keys and values in 8 or 4 bits.

    ``group_size`` elements of a head share a scale and a zero point: 64 or
    ``head_dim`` (64 or 128); the default is one group per head for 8 bits and
    64 for 4. ``max_len`` is rounded up to a multiple of 16. The buffers
    (``k_codes``, ``k_params``, ``v_codes``, ``v_params``) are ordinary tensors;
    include/csaq_b200.h documents their layout (csaq_kvq_cache).
    """

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, bits: int = 8,
                 group_size: Optional[int] = None, device=None) -> None:
        if bits not in (8, 4):
            raise ValueError(f"csaq-b200: a KV cache holds 8 or 4 bits, not {bits}")
        if min(batch, kv_heads, max_len) < 1:
            raise ValueError("csaq-b200: batch, kv_heads and max_len must be positive")
        group = group_size if group_size is not None else (head_dim if bits == 8 else 64)
        dev = torch.device(device) if device is not None else _lib.cuda_device()
        L = cache_positions(max_len)
        code = lambda: torch.zeros(batch, kv_heads, L, head_dim * bits // 8, dtype=torch.uint8, device=dev)  # noqa: E731
        word = lambda: torch.zeros(batch, kv_heads, L, max(head_dim // max(group, 1), 1), dtype=torch.int32,  # noqa: E731
                                   device=dev)
        if group not in (64, head_dim) or head_dim not in (64, 128):
            raise ValueError("csaq-b200: head_dim must be 64 or 128 and group_size 64 or head_dim")
        self._adopt(code(), word(), code(), word(), bits)

    @classmethod
    def from_buffers(cls, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                     v_params: torch.Tensor, bits: int) -> "QuantizedKVCache":
        """A cache over existing buffers (kept, not copied)."""
        if bits not in (8, 4):
            raise ValueError(f"csaq-b200: a KV cache holds 8 or 4 bits, not {bits}")
        self = cls.__new__(cls)
        self._adopt(k_codes, k_params, v_codes, v_params, bits)
        return self

    def _adopt(self, kc, kp, vc, vp, bits: int) -> None:
        for t, dt, what in ((kc, torch.uint8, "k_codes"), (kp, torch.int32, "k_params"), (vc, torch.uint8, "v_codes"),
                            (vp, torch.int32, "v_params")):
            if t.dtype != dt or t.dim() != 4 or not t.is_contiguous():
                raise ValueError(f"csaq-b200: {what} must be a contiguous 4-D {dt} tensor")
            if t.device != kc.device:
                raise ValueError("csaq-b200: a cache's buffers live on one device")
        if kc.shape != vc.shape or kp.shape != vp.shape or kc.shape[:3] != kp.shape[:3]:
            raise ValueError("csaq-b200: the cache buffers do not belong together: "
                             f"{[tuple(t.shape) for t in (kc, kp, vc, vp)]}")
        B, Hkv, L, rowb = kc.shape
        D = rowb * 8 // bits
        if min(B, Hkv, L) < 1:
            raise ValueError("csaq-b200: a cache holds at least one sequence, KV head and position")
        if D not in (64, 128) or kp.shape[3] not in (1, D // 64) or L % 16:
            raise ValueError("csaq-b200: head_dim must be 64 or 128, group_size 64 or head_dim and the length a "
                             "multiple of 16")
        self.k_codes, self.k_params, self.v_codes, self.v_params = kc, kp, vc, vp
        self.batch, self.kv_heads, self.max_len, self.head_dim = B, Hkv, L, D
        self.bits, self.group_size = bits, D // kp.shape[3]
        self.device = kc.device
        self._c = CsaqKvqCache(kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), L, bits, self.group_size)
        self._ref = ctypes.byref(self._c)
        self._sizes = {}  # (tokens, heads) -> floats of attend's scratch
        self._pos_shape = (B,)
        self._scale = 1.0 / math.sqrt(D)

    def buffers(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.k_codes, self.k_params, self.v_codes, self.v_params

    def zero_(self) -> "QuantizedKVCache":
        for t in self.buffers():
            t.zero_()
        return self

    # ── argument checks shared by the calls ─────────────────────────────────
    def _tokens(self, t: torch.Tensor, what: str) -> Tuple[int, int, int]:
        """(tokens per sequence, columns, dtype code) of a step's matrix t (B*S rows)."""
        if t.device != self.device or not t.is_cuda:
            raise RuntimeError(f"csaq-b200: {what} must be on the cache's CUDA device {self.device}, not {t.device}")
        code = _CODES.get(t.dtype)
        if code is None:
            raise TypeError(f"csaq-b200: {what} must be float16 or bfloat16, not {t.dtype}")
        shape = t.shape
        if len(shape) != 2 or shape[0] < self.batch or shape[0] % self.batch:
            raise ValueError(f"csaq-b200: {what} needs batch * tokens rows (batch {self.batch}), got {tuple(shape)}")
        return shape[0] // self.batch, shape[1], code

    def _heads(self, columns: int) -> int:
        step = self.kv_heads * self.head_dim
        if columns < step or columns % step:
            raise ValueError(f"csaq-b200: q needs a multiple of {step} columns (kv_heads * head_dim), got {columns}")
        return columns // self.head_dim

    def _positions(self, pos0: torch.Tensor) -> int:
        if pos0.dtype is not torch.int32 or pos0.shape != self._pos_shape or pos0.device != self.device \
                or not pos0.is_contiguous():
            raise ValueError(f"csaq-b200: pos0 must be {self.batch} contiguous int32 values on {self.device}")
        return pos0.data_ptr()

    def _run(self, fn, what: str, *args) -> None:
        """fn(*args, the current stream of the cache's device), with that device current."""
        index = self.device.index
        if index == torch.cuda.current_device():
            rc = fn(*args, raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, raw_stream(index))
        if rc:
            check(rc, what)

    # ── the operators ────────────────────────────────────────────────────────
    def write(self, k: torch.Tensor, v: torch.Tensor, pos0: torch.Tensor, cos: Optional[torch.Tensor] = None,
              sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Quantise a step's keys and values (B*S, kv_heads*head_dim) into
        positions pos0[b] .. pos0[b]+S-1.

        With cos and sin (fp32 tables of one row per position, head_dim wide)
        the keys are rotated first, and q (B*S, heads*head_dim), when given, is
        rotated into q_out, which is returned. Positions outside the cache or
        the tables are not stored (their queries pass unrotated)."""
        width = self.kv_heads * self.head_dim
        kind = S, columns, code = self._tokens(k, "k")
        if self._tokens(v, "v") != kind or columns != width:
            raise ValueError(f"csaq-b200: k and v must have one dtype and batch * tokens rows of {width} columns")
        at = self._positions(pos0)
        (k, ldk), (v, ldv) = _rows(k), _rows(v)
        Hq, n_rope, ldq = 0, 0, 0
        if (cos is None) != (sin is None):
            raise ValueError("csaq-b200: cos and sin come together")
        if cos is not None:
            for t in (cos, sin):
                if t.dtype is not torch.float32 or t.shape != cos.shape or t.dim() != 2 or t.shape[1] != self.head_dim \
                        or t.device != self.device or not t.is_contiguous() or t.shape[0] == 0:
                    raise ValueError(f"csaq-b200: cos and sin must be contiguous fp32 (positions, {self.head_dim}) "
                                     f"tables on {self.device}")
            n_rope = cos.shape[0]
        if q is not None:
            if cos is None:
                raise ValueError("csaq-b200: q is only rotated: pass cos and sin with it")
            Sq, columns, code_q = self._tokens(q, "q")
            if Sq != S or code_q != code:
                raise ValueError("csaq-b200: q must have k's rows and dtype")
            Hq = self._heads(columns)
            q, ldq = _rows(q)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.device != q.device \
                    or not q_out.is_contiguous():
                raise ValueError("csaq-b200: q_out must be contiguous with q's shape and dtype")
        elif q_out is not None:
            raise ValueError("csaq-b200: q_out without q")
        self._run(lib().csaq_kvq_write, "kvq_write", ptr(q), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, at,
                  self.batch, S, Hq, self.kv_heads, self.head_dim, ptr(cos), ptr(sin), n_rope, ptr(q_out),
                  self._ref, code)
        return q_out

    def read(self, start: int, end: int, dtype: torch.dtype = torch.bfloat16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Positions [start, end) as (k, v), each (B, kv_heads, end-start,
        head_dim) in dtype (float32, float16 or bfloat16)."""
        if not 0 <= start <= end <= self.max_len:
            raise ValueError(f"csaq-b200: positions [{start}, {end}) are not inside the cache's {self.max_len}")
        if self.device.type != "cuda":
            raise RuntimeError(f"csaq-b200: the cache must be on a CUDA device, not {self.device}")
        code = dtype_code(dtype)
        shape = (self.batch, self.kv_heads, end - start, self.head_dim)
        if out is None:
            k = torch.empty(shape, dtype=dtype, device=self.device)
            out = k, torch.empty_like(k)
        else:
            for t in out:
                if tuple(t.shape) != shape or t.dtype != dtype or t.device != self.device or not t.is_contiguous():
                    raise ValueError(f"csaq-b200: out must be two contiguous {dtype} tensors of shape {shape}")
        k, v = out
        if end > start:
            self._run(lib().csaq_kvq_read, "kvq_read", self._ref, self.batch, self.kv_heads, self.head_dim, start,
                      end - start, k.data_ptr(), v.data_ptr(), code)
        return k, v

    def workspace(self, tokens: int, heads: int) -> KVWorkspace:
        """Scratch for ``attend`` with up to `tokens` tokens per sequence and `heads` query heads."""
        return KVWorkspace(torch.empty(self._floats(tokens, heads), dtype=torch.float32, device=self.device))

    def _floats(self, tokens: int, heads: int) -> int:
        n = self._sizes.get((tokens, heads))
        if n is None:
            n = lib().csaq_kvq_attention_workspace_floats(self.batch, tokens, heads, self.kv_heads, self.head_dim,
                                                          self.max_len)
            if n < 0:
                raise ValueError(f"csaq-b200: no attention of {tokens} tokens and {heads} heads over "
                                 f"{self.kv_heads} KV heads")
            self._sizes[(tokens, heads)] = n
        return n

    def attend(self, q: torch.Tensor, pos0: torch.Tensor, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, workspace: Optional[KVWorkspace] = None) -> torch.Tensor:
        """Causal attention of a step's (rotated) queries, (B*S, heads*head_dim):
        token (b, s) attends positions 0 .. pos0[b]+s. A token at a negative
        position sees nothing and gets zeros. S is at most 65535. scale defaults
        to 1/sqrt(head_dim). Without a workspace one is allocated for the call."""
        S, columns, code = self._tokens(q, "q")
        Hq = self._heads(columns)
        at = self._positions(pos0)
        q, ldq = _rows(q)
        ldo = columns
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(1) != 1:
                raise ValueError("csaq-b200: out must have q's shape and dtype and rows of even stride")
            if out.shape[0] > 1:
                ldo = out.stride(0)
                if ldo < columns or ldo % 2:
                    raise ValueError("csaq-b200: out must have q's shape and dtype and rows of even stride")
        floats, part = self._floats(S, Hq), None
        if workspace is not None:
            part = workspace.part
            if part.device != self.device or part.numel() < floats or part.dtype is not torch.float32 \
                    or not part.is_contiguous():
                raise ValueError(f"csaq-b200: the workspace must be {floats} contiguous fp32 values on {self.device} "
                                 f"for {S} tokens and {Hq} heads of this cache")
        elif floats:
            part = torch.empty(floats, dtype=torch.float32, device=self.device)
        self._run(lib().csaq_kvq_attention, "kvq_attention", q.data_ptr(), ldq, self._ref, at, self.batch, S, Hq,
                  self.kv_heads, self.head_dim, self._scale if scale is None else float(scale), ptr(part) if floats else None,
                  out.data_ptr(), ldo, code)
        return out
