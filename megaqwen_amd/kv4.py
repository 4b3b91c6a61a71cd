"""A key/value cache held in 4 bits, and the attention over it.

    cache = KV4Cache(batch, num_kv_heads, max_seq_len)
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")     # with the new rows
    cache.append(k, v, lengths)                                       # [batch, t, kv_heads, head_dim]
    out = cache.attend(q, lengths)                                    # [batch, t, q_heads, head_dim]

Every call works on the last t positions of each sequence: row i of t is at position
lengths[b] - t + i.  Rows whose position is negative do not exist (a batch of unequal prompts is
padded at its front): append skips them, read and attend give 0 for them.  `lengths` stays on the
device, so a decode loop can be captured into a HIP graph and replayed with new lengths.

A row's values are held in groups (32, 64 or 128 of the head's dimensions): scale = bf16(max|x| / 7),
code = 8 + round(x / scale) in 1..15, two codes to a byte, the even dimension in the low half.  A row
of 128 takes 72 bytes in groups of 32, against 256 in bf16.

The compute is the hand-written gfx950 kernels behind `mq_kv4_append`, `mq_kv4_read` and
`mq_kv4_attend` (include/megaqwen_hip.h, megaqwen_amd/csrc/kv4.hip); there is no PyTorch fallback.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._launch import DTYPES, call, no_grad
from .spec import COMPILED_LAYER_SHAPE

HEAD_DIMS = (64, 128)
GROUP_SIZES = (32, 64, 128)
_Strides = ctypes.c_int64 * 3


class KV4Cache:
    """Codes and scales of `batch` sequences of up to max_seq_len positions (one layer).

    Tensors: k_codes, v_codes uint8 [batch, kv_heads, max_seq_len, head_dim / 2] and scales bf16
    [batch, kv_heads, max_seq_len, 2, head_dim / group_size] (key scales, then value scales)."""

    def __init__(self, batch: int, num_kv_heads: int = COMPILED_LAYER_SHAPE["num_kv_heads"],
                 max_seq_len: int = 2048, head_dim: int = COMPILED_LAYER_SHAPE["head_dim"],
                 group_size: int = 32, *, device="cuda"):
        shape = (int(batch), int(num_kv_heads), int(max_seq_len))
        if min(shape) < 1 or shape[1] > 256:
            raise ValueError("batch, num_kv_heads and max_seq_len must be positive, and num_kv_heads at most 256, "
                             f"got {shape}")
        if head_dim not in HEAD_DIMS or group_size not in GROUP_SIZES or group_size > head_dim:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS} and group_size one of {GROUP_SIZES}, "
                             f"at most head_dim; got {head_dim} and {group_size}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("KV4Cache expects a CUDA device")
        codes = torch.full((2, *shape, head_dim // 2), 0x88, dtype=torch.uint8, device=device)
        self._bind(codes[0], codes[1], torch.zeros((*shape, 2, head_dim // group_size),
                                                   dtype=torch.bfloat16, device=device))

    @classmethod
    def from_tensors(cls, k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor) -> "KV4Cache":
        """A cache over caller-owned tensors of the shapes above (they are used in place)."""
        if k_codes.ndim != 4 or k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 \
                or v_codes.shape != k_codes.shape or k_codes.shape[-1] * 2 not in HEAD_DIMS \
                or min(k_codes.shape) < 1 or k_codes.shape[1] > 256:
            raise ValueError("k_codes and v_codes must be uint8 [batch, kv_heads, max_seq_len, head_dim / 2] with "
                             f"head_dim one of {HEAD_DIMS} and at most 256 kv_heads; got {k_codes.dtype} {tuple(k_codes.shape)} and "
                             f"{v_codes.dtype} {tuple(v_codes.shape)}")
        dim = 2 * k_codes.shape[-1]
        if scales.ndim != 5 or scales.dtype != torch.bfloat16 or scales.shape[:4] != (*k_codes.shape[:3], 2) \
                or scales.shape[4] not in [dim // g for g in GROUP_SIZES if g <= dim]:
            raise ValueError("scales must be bfloat16 [batch, kv_heads, max_seq_len, 2, head_dim / group_size], got "
                             f"{scales.dtype} {tuple(scales.shape)}")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes), ("scales", scales)):
            if t.device.type != "cuda" or t.device != k_codes.device:
                raise ValueError(f"{name} is on {t.device}; the cache's tensors must be on one CUDA device")
            if not t.is_contiguous() or t.data_ptr() % (4 if name == "scales" else 16) != 0:
                raise ValueError(f"{name} must be contiguous and aligned (codes 16 bytes, scales 4)")
        cache = cls.__new__(cls)
        cache._bind(k_codes, v_codes, scales)
        return cache

    def _bind(self, k_codes, v_codes, scales) -> None:
        self.k_codes, self.v_codes, self.scales = k_codes, v_codes, scales
        self.batch, self.num_kv_heads, self.max_seq_len, half = k_codes.shape
        self.head_dim, self.device = 2 * half, k_codes.device
        self.group_size = self.head_dim // scales.shape[-1]
        self._dev = k_codes.get_device()
        lib = _lib.load()
        self._append, self._read, self._attend = lib.mq_kv4_append, lib.mq_kv4_read, lib.mq_kv4_attend
        self._workspace = lib.mq_kv4_attend_workspace_bytes
        self._desc = _lib.Kv4Cache(k_codes.data_ptr(), v_codes.data_ptr(), scales.data_ptr(), self.batch,
                                   self.num_kv_heads, self.max_seq_len, self.head_dim, self.group_size)
        self._ref = ctypes.byref(self._desc)

    # ------------------------------------------------------------------------------ checks
    def _rows(self, what: str, name: str, x: torch.Tensor, heads: Optional[int]):
        """x as [batch, t, heads, head_dim] with a contiguous last dimension."""
        if x.get_device() != self._dev:
            raise ValueError(f"{name} is on {x.device}, the cache on {self.device}")
        if x.dtype != torch.bfloat16 and x.dtype != torch.float16:
            raise ValueError(f"{what} only supports fp16/bf16, got {x.dtype}")
        s = x.shape
        if len(s) != 4 or s[0] != self.batch or s[3] != self.head_dim or (heads is not None and s[2] != heads):
            raise ValueError(f"{name} must be [batch={self.batch}, t, {'heads' if heads is None else heads}, "
                             f"head_dim={self.head_dim}], got {tuple(s)}")
        return x if x.stride(3) == 1 else x.contiguous()

    def _lengths(self, lengths: torch.Tensor) -> int:
        if lengths.get_device() != self._dev or lengths.dtype != torch.int32 or lengths.shape != (self.batch,) \
                or not lengths.is_contiguous():
            raise ValueError(f"lengths must be a contiguous int32 tensor [{self.batch}] on {self.device}, got "
                             f"{lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
        return lengths.data_ptr()

    # --------------------------------------------------------------------------- operators
    def append(self, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor) -> None:
        """Quantises k and v [batch, t, kv_heads, head_dim] (bf16 or fp16; any strides of the first
        three dimensions) into positions lengths[b] - t .. lengths[b] - 1; positions outside
        [0, max_seq_len) are skipped.  A group that holds an infinity or a NaN reads as NaN."""
        k = self._rows("KV4Cache.append", "k", k, self.num_kv_heads)
        v = self._rows("KV4Cache.append", "v", v, self.num_kv_heads)
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"Shape mismatch k={k.dtype} {tuple(k.shape)} v={v.dtype} {tuple(v.shape)}")
        at = self._lengths(lengths)
        if torch.is_grad_enabled():
            no_grad("KV4Cache.append", k, v)
        call(self._append, self._dev, self._ref, k.data_ptr(), _Strides(*k.stride()[:3]), v.data_ptr(),
             _Strides(*v.stride()[:3]), at, k.shape[1], DTYPES[k.dtype])

    def read(self, lengths: torch.Tensor, t: int, dtype: torch.dtype = torch.bfloat16
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [batch, t, kv_heads, head_dim]: the values held for positions lengths[b] - t ..
        lengths[b] - 1, rounded to `dtype` (bf16, fp16, or fp32, which is exact); positions outside
        [0, max_seq_len) read as 0."""
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        t = int(t)
        if t < 0:
            raise ValueError(f"t must not be negative, got {t}")
        at = self._lengths(lengths)
        k = self.scales.new_empty((self.batch, t, self.num_kv_heads, self.head_dim), dtype=dtype)
        v = torch.empty_like(k)
        call(self._read, self._dev, self._ref, at, t, k.data_ptr(), v.data_ptr(), DTYPES[dtype])
        return k, v

    def attend(self, q: torch.Tensor, lengths: torch.Tensor, *, scale: Optional[float] = None,
               max_length: Optional[int] = None) -> torch.Tensor:
        """Causal attention of q [batch, t, q_heads, head_dim] (bf16 or fp16, q_heads a multiple of
        kv_heads, by at most 256) over the cache: query i of t looks at positions
        0 .. lengths[b] - t + i.  The output has q's type and shape; a query with no position to look at gives 0.  `scale`
        defaults to 1/sqrt(head_dim).  max_length, if known, is an upper bound of `lengths`: the
        work is split for it, and positions from there on are not looked at."""
        q = self._rows("KV4Cache.attend", "q", q, None)
        _, t, heads, _ = q.shape
        if heads < 1 or heads % self.num_kv_heads != 0:
            raise ValueError(f"q has {heads} heads, not a multiple of {self.num_kv_heads}")
        at = self._lengths(lengths)
        n = self.max_seq_len if max_length is None else int(max_length)
        if not 0 <= n <= self.max_seq_len:
            raise ValueError(f"max_length {n} outside [0, max_seq_len={self.max_seq_len}]")
        if torch.is_grad_enabled():
            no_grad("KV4Cache.attend", q)
        if n == 0 or t == 0:
            return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        out = q.new_empty(q.shape)
        # scratch of this call alone, in stream order: calls on other streams and captured graphs
        # have theirs
        size = self._workspace(self._ref, t, heads, n)
        ws = self.k_codes.new_empty(size) if size else None
        call(self._attend, self._dev, self._ref, q.data_ptr(), _Strides(*q.stride()[:3]), at, t, heads, n,
             DTYPES[q.dtype], scale, out.data_ptr(), None if ws is None else ws.data_ptr(), size)
        return out
