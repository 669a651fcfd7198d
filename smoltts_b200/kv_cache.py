"""A paged key/value cache in 8 bits: ``KVCache8`` holds one attention layer's keys and values as e4m3 codes with a
power-of-two scale per 16 positions and head, appends to them (rotating keys and queries by position on the way) and
attends to them.

Half the bytes of a bf16 cache: twice the positions in the same pool, and half the traffic of decoding.  Pages are the
indices of a ``pool.PagePool``; a batch is ragged, as in an engine step: sequence ``s`` brings the rows ``seq_start[s] ..
seq_start[s + 1] - 1``, which are its positions ``seq_pos0[s], seq_pos0[s] + 1, ...`` (below 2^31 - 128).  The arrays are looked at on the device: a sequence
whose rows or positions do not fit is left out, a page outside the cache not touched, and ``check_device_errors`` tells.  Everything runs on the current stream
of the cache's device and nothing synchronises, so that calls can be captured into a CUDA graph; results carry no gradient.  ``lm.HybridLM`` serves
its softmax attention layers from such a cache with ``kv_bits=8``.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Dict, Optional, Tuple

import torch

from . import _capi_lm
from ._errors import SMOL_ERR_CAPACITY, SMOL_ERR_CUDA, SMOL_OK, SmolError

BLOCK = 16          # positions that share a scale
_DTYPES = {torch.bfloat16: _capi_lm.SMOL_LM_BF16, torch.float32: _capi_lm.SMOL_LM_F32}
# The arguments' structs of include/smoltts_b200_lm.h as native layouts: packing one takes a microsecond, filling a ctypes structure several.
_BATCH = struct.Struct("@5i4P")
_APPEND = struct.Struct("@i2P4Ni2P4N2iPf0P")
_ATTEND = struct.Struct("@2i2P4N3f2i5PN0P")
for _s, _m in ((_BATCH, _capi_lm.SmolLmCache8Batch), (_APPEND, _capi_lm.SmolLmCache8Append), (_ATTEND, _capi_lm.SmolLmCache8Attend)):
    assert _s.size == C.sizeof(_m)


def _pack(layout: struct.Struct, *fields) -> bytes:
    """The fields in their native types; an integer that its type does not hold is the caller's."""
    try:
        return layout.pack(*fields)
    except struct.error as e:
        raise ValueError(f"an integer outside its range: {e}") from e


def _float(x: float, what: str) -> float:
    if not abs(x) <= 3.4028234663852886e38:      # (packing would make an infinity of it)
        raise ValueError(f"{what} {x} is outside the range of float32")
    return x


def _padded(n: int) -> int:
    return (n + 15) // 16 * 16


def _extent(x: torch.Tensor) -> Tuple[int, int]:
    """First byte and the one behind the last that a tensor reaches."""
    at = x.data_ptr()
    return at, at + (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))) * x.element_size()


def _check_written(out: torch.Tensor, what: str, **read: torch.Tensor) -> None:
    """A result must not overlap itself, nor what is read while it is written."""
    (tokens, heads, width), (row, head, _) = out.shape, out.stride()
    if not ((heads == 1 or head >= width) and (tokens == 1 or row >= (heads - 1) * head + width) or
            (tokens == 1 or row >= width) and (heads == 1 or head >= (tokens - 1) * row + width)):
        raise ValueError(f"{what}: rows must not overlap")
    lo, hi = _extent(out)
    for name, x in read.items():
        a, b = _extent(x)
        if a < hi and lo < b:
            raise ValueError(f"{what} must not reach into {name}'s memory: it is read while {what} is written")


class KVCache8:
    """Codes ``k [pages, kv_heads, page_size, dim rounded up to 16]`` and ``v`` (e4m3), scales ``k_scale`` / ``v_scale``
    ``[pages, kv_heads, page_size / 16]`` (fp32; a position's values are its codes times the magnitude of its block's scale,
    and a negative scale says that the block holds a NaN).  All four are contiguous tensors of one CUDA device that the
    caller may make (``allocate`` makes them); codes behind ``dim`` / ``vdim`` are zeros."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, dim: Optional[int] = None, vdim: Optional[int] = None):
        if k.dim() != 4 or v.dim() != 4 or k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
            raise ValueError("k and v must be float8_e4m3fn [pages, kv_heads, page_size, padded head size]")
        n, g, page, ld = k.shape
        self.dim, self.vdim = ld if dim is None else int(dim), v.shape[3] if vdim is None else int(vdim)
        if tuple(v.shape[:3]) != (n, g, page) or ld != _padded(self.dim) or v.shape[3] != _padded(self.vdim):
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not hold heads of {self.dim} and {self.vdim} in the same pages")
        if page % BLOCK or page < BLOCK or n < 1 or g < 1:
            raise ValueError("page_size must be a multiple of 16, with at least one page and head")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or tuple(s.shape) != (n, g, page // BLOCK):
                raise ValueError(f"scales must be float32 {(n, g, page // BLOCK)}")
        if not k.is_cuda or any(t.device != k.device or not t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("codes and scales must be contiguous tensors of one CUDA device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.kv_heads, self.page_size = n, g, page
        self.device, self._index = k.device, k.device.index
        self._err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = bytes(_capi_lm.SmolLmCache8(k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(), n_pages=n, page_size=page,
                                              kv_heads=g, dim=self.dim, vdim=self.vdim, err=self._err.data_ptr()))
        lib = _capi_lm.load()
        # (functions of this module's own: their arguments are packed structs)
        self._append, self._attend, self._workspace = lib["smol_lm_cache8_append"], lib["smol_lm_cache8_attend"], lib["smol_lm_cache8_workspace_bytes"]
        self._append.argtypes = [C.c_char_p, C.c_char_p, C.c_char_p, C.c_void_p]
        self._attend.argtypes = [C.c_char_p, C.c_char_p, C.c_char_p, C.c_void_p, C.c_size_t, C.c_void_p]
        self._workspace.argtypes = [C.c_char_p, C.c_char_p, C.c_char_p, C.c_void_p]
        self._need: Dict[tuple, int] = {}      # bytes of workspace by what they depend on

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, kv_heads: int, dim: int, vdim: Optional[int] = None, device=None) -> "KVCache8":
        """An empty cache of ``n_pages`` pages."""
        device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        vdim = dim if vdim is None else vdim
        if n_pages < 1 or kv_heads < 1 or page_size < BLOCK or page_size % BLOCK or dim < 1 or vdim < 1:
            raise ValueError("page_size must be a multiple of 16, and all sizes positive")
        codes = [torch.zeros(n_pages, kv_heads, page_size, _padded(w), dtype=torch.float8_e4m3fn, device=device) for w in (dim, vdim)]
        scales = [torch.zeros(n_pages, kv_heads, page_size // BLOCK, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1], dim=dim, vdim=vdim)

    # ------------------------------------------------------------------ arguments
    def _rows(self, x: torch.Tensor, tokens: Optional[int], heads: Optional[int], width: int, dtype: Optional[torch.dtype], what: str) -> Tuple[int, int]:
        """Checks a ``[tokens, heads, width]`` tensor and returns its strides; rows may be slices of something wider."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != width or (heads is not None and shape[1] != heads) or (tokens is not None and shape[0] != tokens):
            raise ValueError(f"{what} must be [{'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, {width}], got {tuple(shape)}")
        if x.dtype not in _DTYPES or (dtype is not None and x.dtype != dtype) or x.device != self.device:
            raise ValueError(f"{what} must be {'bfloat16 or float32' if dtype is None else dtype} on {self.device}, got {x.dtype} on {x.device}")
        row, head, one = x.stride()
        if one != 1 and width > 1:
            raise ValueError(f"{what}: the last dimension must be contiguous")
        return row, head

    def _ints(self, x: torch.Tensor, shape: tuple, what: str) -> int:
        if x.dtype != torch.int32 or x.shape != shape or x.device != self.device or not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous int32 {shape} on {self.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x.data_ptr()

    def _floats(self, x: Optional[torch.Tensor], n: int, what: str) -> int:
        if x is None:
            return 0
        if x.dtype != torch.float32 or x.shape != (n,) or x.device != self.device or not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous float32 [{n}] on {self.device}")
        return x.data_ptr()

    def _batch(self, tokens: int, seq_start, seq_pos0, block_table, max_new: int, max_len: int, kv_len=None) -> bytes:
        if block_table.dim() != 2:
            raise ValueError("block_table must be [sequences, pages]")
        n, pages = block_table.shape
        if tokens < 1 or n < 1 or pages < 1 or max_new < 1 or max_len < 1:
            raise ValueError("a batch needs at least one row, sequence and page, max_new and max_len at least 1")
        return _pack(_BATCH, tokens, n, pages, max_new, max_len, self._ints(seq_start, (n + 1,), "seq_start"), self._ints(seq_pos0, (n,), "seq_pos0"),
                     self._ints(block_table, (n, pages), "block_table"), 0 if kv_len is None else self._ints(kv_len, (n,), "kv_len"))

    def _call(self, call, *args) -> None:
        """On the cache's device and its current stream."""
        if self._index == torch._C._cuda_getDevice():      # (a few tenths of a microsecond; torch.cuda's own two functions take four)
            rc = call(self._c, *args, torch._C._cuda_getCurrentRawStream(self._index))
        else:
            with torch.cuda.device(self._index):
                rc = call(self._c, *args, torch._C._cuda_getCurrentRawStream(self._index))
        if rc != SMOL_OK:
            _capi_lm.check(rc)

    # ------------------------------------------------------------------ operators
    def append(self, k: torch.Tensor, v: torch.Tensor, seq_start: torch.Tensor, seq_pos0: torch.Tensor, block_table: torch.Tensor, max_new: int,
               q: Optional[torch.Tensor] = None, freq: Optional[torch.Tensor] = None, rot_half: bool = True, rot_mult: float = 1.0,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes the rows' keys ``k [tokens, kv_heads, dim]`` and values ``v [tokens, kv_heads, vdim]`` into their pages.

        With ``freq [pairs]`` (fp32) keys, and queries ``q [tokens, heads, dim]``, are rotated first: pair ``i`` by the angle position *
        ``freq[i]`` (computed in 64 bits), ``rot_half`` pairing coordinate ``i`` with ``i + pairs``, otherwise ``2i`` with ``2i + 1``; coordinates
        behind the pairs pass unchanged; ``rot_mult`` multiplies cosine and sine.  Returns the queries (in ``q_out``, or a new tensor), or None
        without ``q``.  ``max_new``: most rows a sequence brings (a host number).  Rows outside every sequence are left alone.

        A block's 16 positions share the smallest power of two with |value| <= 448 * scale; where an earlier call began the block the
        scale never shrinks, and the older codes follow it when it grows.  Magnitudes above 2^100 are clamped; a NaN stays a NaN.  Two
        sequences of a batch must not write the same page, nor one write a page twice.  The rows of a sequence have to follow what it already holds."""
        tokens, dtype = k.shape[0], k.dtype
        k_row, k_head = self._rows(k, None, self.kv_heads, self.dim, None, "k")
        v_row, v_head = self._rows(v, tokens, self.kv_heads, self.vdim, dtype, "v")
        batch = self._batch(tokens, seq_start, seq_pos0, block_table, max_new, max_new)
        pairs = freq_ptr = heads = q_ptr = q_row = q_head = out_ptr = out_row = out_head = 0
        if freq is not None:
            if freq.dim() != 1 or 2 * freq.shape[0] > self.dim:
                raise ValueError(f"freq must be [pairs] with at most {self.dim // 2} pairs")
            pairs = freq.shape[0]
            freq_ptr = self._floats(freq, pairs, "freq") if pairs else 0
        if q is not None:
            q_row, q_head = self._rows(q, tokens, None, self.dim, dtype, "q")
            heads = q.shape[1]
            if heads < 1:
                raise ValueError("q without heads")
            if q_out is None:
                q_out = q.new_empty((tokens, heads, self.dim))
                out_row, out_head = heads * self.dim, self.dim
            else:
                out_row, out_head = self._rows(q_out, tokens, heads, self.dim, dtype, "q_out")
                _check_written(q_out, "q_out", q=q, k=k, v=v)
            q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        self._call(self._append, batch, _pack(_APPEND, _DTYPES[dtype], k.data_ptr(), v.data_ptr(), k_row, k_head, v_row, v_head, heads, q_ptr, out_ptr, q_row, q_head,
                                              out_row, out_head, 2 * pairs, 1 if rot_half else 0, freq_ptr, _float(rot_mult, "rot_mult")))
        return q_out

    def attend(self, q: torch.Tensor, seq_start: torch.Tensor, seq_pos0: torch.Tensor, block_table: torch.Tensor, max_new: int, max_len: int,
               scale: Optional[float] = None, window: int = 0, first: int = 0, softcap: float = 0.0, sink: Optional[torch.Tensor] = None,
               slope: Optional[torch.Tensor] = None, penalty: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
               kv_len: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal softmax attention of the rows ``q [tokens, heads, dim]`` over the cache (which holds the rows' own positions already).

        A row at position ``i`` sees the keys ``j <= i``; with ``window`` only ``i - j < window``, and the sequence's first ``first``
        positions whatever their distance; ``kv_len [sequences]`` hides keys from that position on.  Score: ``scale`` (default
        ``dim ** -0.5``) times q.k, bent by ``softcap * tanh(s / softcap)``, less ``penalty[0] * ln(1 + penalty[1] * (i - j))`` and ``slope * (i - j)``;
        ``sink``, a logit without a key, joins the denominator (all per query head, fp32).  A row that sees no key gives zeros.

        ``max_new``: most rows a sequence brings; ``max_len``: most positions a sequence holds, the rows included (host numbers;
        the grid is chosen by them -- a longer sequence is attended to as a whole all the same, rows beyond ``max_new`` are left alone).
        Returns ``[tokens, heads, vdim]`` of q's type, in ``out`` if given (which must not reach into q's memory); rows outside every sequence are left as
        they were, which in a new tensor is anything."""
        q_row, q_head = self._rows(q, None, None, self.dim, None, "q")
        tokens, heads, dtype = q.shape[0], q.shape[1], q.dtype
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads over {self.kv_heads} key/value heads")
        if window < 0 or first < 0 or not 0.0 <= softcap < math.inf:
            raise ValueError("window, first and softcap must not be negative, and softcap finite")
        batch = self._batch(tokens, seq_start, seq_pos0, block_table, max_new, max_len, kv_len)
        if out is None:
            out = q.new_empty((tokens, heads, self.vdim))
            out_row, out_head = heads * self.vdim, self.vdim
        else:
            out_row, out_head = self._rows(out, tokens, heads, self.vdim, dtype, "out")
            _check_written(out, "out", q=q)
        r1 = r2 = 0
        if penalty is not None:
            r1, r2 = self._floats(penalty[0], heads, "penalty[0]"), self._floats(penalty[1], heads, "penalty[1]")
        a = _pack(_ATTEND, _DTYPES[dtype], heads, q.data_ptr(), out.data_ptr(), q_row, q_head, out_row, out_head, self.dim ** -0.5 if scale is None else _float(scale, "scale"), _float(softcap, "softcap"), 1.0,
                  window, first, self._floats(sink, heads, "sink"), self._floats(slope, heads, "slope"), r1, r2, 0, 0)
        key = (dtype, tokens, heads, block_table.shape, max_new, max_len, window, first)
        need = self._need.get(key)
        if need is None:
            size = C.c_size_t()
            with torch.cuda.device(self._index):
                _capi_lm.check(self._workspace(self._c, batch, a, C.byref(size)))
            if len(self._need) >= 4096:
                self._need.clear()
            need = self._need[key] = size.value
        # of the call's own: from torch's allocator for this stream, or for the graph that is being captured
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._call(self._attend, batch, a, work.data_ptr() if need else None, need)
        return out

    # ------------------------------------------------------------------ looking in
    def values(self, pages: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """What ``pages`` (an index tensor) hold: keys and values ``[pages, kv_heads, page_size, dim / vdim]`` in fp32."""
        got = []
        for codes, scale, width in ((self.k, self.k_scale, self.dim), (self.v, self.v_scale, self.vdim)):
            x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.float32)
            got.append((x[..., :width] * scale[pages].abs().repeat_interleave(BLOCK, -1).unsqueeze(-1)))
        return got[0], got[1]

    def check_device_errors(self) -> None:
        """Raises if a call met a page outside the cache or arrays that contradict one another (reads a device word; synchronises)."""
        word = int(self._err.item())
        if word == 3:
            raise SmolError(SMOL_ERR_CUDA, "device-side error word 3: a wait inside a kernel ran out, results of that call are missing")
        if word:
            raise SmolError(SMOL_ERR_CAPACITY, f"device-side error word {word}: " + ("a block table names a page outside the cache" if word == 1 else "a batch's arrays do not fit its sizes"))
