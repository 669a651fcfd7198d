"""A paged key/value cache in 8 bits: ``KVCache8`` holds one attention layer's keys and values as e4m3 codes with a
power-of-two scale per 16 positions and head, appends to them (rotating keys and queries by position on the way) and
attends to them.

Half the bytes of a bf16 cache: twice the positions in the same pool, and half the traffic of decoding.  Pages are the
indices of a ``pool.PagePool``; a batch is ragged, as in an engine step: sequence ``s`` brings the rows ``seq_start[s] ..
seq_start[s + 1] - 1``, which are its positions ``seq_pos0[s], seq_pos0[s] + 1, ...``.  Everything runs on the current stream
of the cache's device and nothing synchronises, so that calls can be captured into a CUDA graph.  ``lm.HybridLM`` serves
its softmax attention layers from such a cache with ``kv_bits=8``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _capi_lm
from ._errors import SMOL_ERR_CAPACITY, SMOL_OK, SmolError

BLOCK = 16          # positions that share a scale
_DTYPES = {torch.bfloat16: _capi_lm.SMOL_LM_BF16, torch.float32: _capi_lm.SMOL_LM_F32}


def _padded(n: int) -> int:
    return (n + 15) // 16 * 16


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
        self.lib = _capi_lm.load()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.kv_heads, self.page_size, self.device = n, g, page, k.device
        self._err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = _capi_lm.SmolLmCache8(k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(), n_pages=n, page_size=page,
                                        kv_heads=g, dim=self.dim, vdim=self.vdim, err=self._err.data_ptr())

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
    def _rows(self, x: torch.Tensor, heads: Optional[int], width: int, what: str) -> Tuple[int, int]:
        """Checks a ``[tokens, heads, width]`` tensor and returns its strides; rows may be slices of something wider."""
        if x.dim() != 3 or x.shape[2] != width or (heads is not None and x.shape[1] != heads):
            raise ValueError(f"{what} must be [tokens, {heads if heads is not None else 'heads'}, {width}], got {tuple(x.shape)}")
        if x.dtype not in _DTYPES or x.device != self.device:
            raise ValueError(f"{what} must be bfloat16 or float32 on {self.device}, got {x.dtype} on {x.device}")
        row, head, one = x.stride()
        if (one != 1 and width > 1) or row < 0 or head < 0:
            raise ValueError(f"{what}: the last dimension must be contiguous")
        return row, head

    def _ints(self, x: torch.Tensor, shape: tuple, what: str) -> int:
        if x.dtype != torch.int32 or x.device != self.device or tuple(x.shape) != shape or not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous int32 {shape} on {self.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x.data_ptr()

    def _floats(self, x: Optional[torch.Tensor], n: int, what: str) -> Optional[int]:
        if x is None:
            return None
        if x.dtype != torch.float32 or x.device != self.device or tuple(x.shape) != (n,) or not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous float32 [{n}] on {self.device}")
        return x.data_ptr()

    def _batch(self, tokens: int, seq_start, seq_pos0, block_table, max_new: int, max_len: int, kv_len=None) -> "_capi_lm.SmolLmCache8Batch":
        if block_table.dim() != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1:
            raise ValueError("block_table must be [sequences, pages]")
        n, pages = block_table.shape
        if tokens < 1 or max_new < 1 or max_len < 1:
            raise ValueError("a batch needs at least one row, max_new and max_len at least 1")
        return _capi_lm.SmolLmCache8Batch(tokens, n, pages, max_new, max_len, self._ints(seq_start, (n + 1,), "seq_start"), self._ints(seq_pos0, (n,), "seq_pos0"),
                                          self._ints(block_table, (n, pages), "block_table"), None if kv_len is None else self._ints(kv_len, (n,), "kv_len"))

    def _call(self, call, *args) -> None:
        """On the cache's device and its current stream."""
        index = self.device.index
        if index == torch.cuda.current_device():
            rc = call(*args, torch.cuda.current_stream().cuda_stream)
        else:
            with torch.cuda.device(index):
                rc = call(*args, torch.cuda.current_stream().cuda_stream)
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
        sequences of a batch must not write the same page.  The rows of a sequence have to follow what it already holds."""
        k_row, k_head = self._rows(k, self.kv_heads, self.dim, "k")
        v_row, v_head = self._rows(v, self.kv_heads, self.vdim, "v")
        tokens = k.shape[0]
        if v.shape[0] != tokens or v.dtype != k.dtype:
            raise ValueError("k and v must have the same rows and type")
        batch = self._batch(tokens, seq_start, seq_pos0, block_table, max_new, max_new)
        a = _capi_lm.SmolLmCache8Append(dtype=_DTYPES[k.dtype], k=k.data_ptr(), v=v.data_ptr(), k_row=k_row, k_head=k_head, v_row=v_row, v_head=v_head,
                                        rot_half=1 if rot_half else 0, rot_mult=rot_mult)
        if freq is not None:
            if freq.dim() != 1 or 2 * freq.shape[0] > self.dim:
                raise ValueError(f"freq must be [pairs] with at most {self.dim // 2} pairs")
            a.rot_dims, a.freq = 2 * freq.shape[0], self._floats(freq, freq.shape[0], "freq")
        if q is not None:
            a.q_row, a.q_head = self._rows(q, None, self.dim, "q")
            if q.shape[0] != tokens or q.dtype != k.dtype or q.shape[1] < 1:
                raise ValueError("q must have k's rows and type")
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            elif q_out.dtype != q.dtype or q_out.shape[0] != tokens:
                raise ValueError("q_out must have q's rows and type")
            elif q_out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
                raise ValueError("q_out must not share q's memory: a row is read while others are written")
            a.heads, a.q, a.q_out = q.shape[1], q.data_ptr(), q_out.data_ptr()
            a.q_out_row, a.q_out_head = self._rows(q_out, q.shape[1], self.dim, "q_out")
        elif q_out is not None:
            raise ValueError("q_out without q")
        self._call(self.lib.smol_lm_cache8_append, self._c, batch, a)
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
        Returns ``[tokens, heads, vdim]`` of q's type, in ``out`` if given; rows outside every sequence are left as they were."""
        q_row, q_head = self._rows(q, None, self.dim, "q")
        tokens, heads = q.shape[0], q.shape[1]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads over {self.kv_heads} key/value heads")
        if window < 0 or first < 0 or not softcap >= 0.0:
            raise ValueError("window, first and softcap must not be negative")
        batch = self._batch(tokens, seq_start, seq_pos0, block_table, max_new, max_len, kv_len)
        if out is None:
            out = torch.empty((tokens, heads, self.vdim), dtype=q.dtype, device=q.device)
        elif out.dtype != q.dtype or out.shape[0] != tokens:
            raise ValueError("out must have q's rows and type")
        out_row, out_head = self._rows(out, heads, self.vdim, "out")
        if (out_row < self.vdim and tokens > 1) or (out_head < self.vdim and heads > 1):
            raise ValueError("out: rows must not overlap")
        a = _capi_lm.SmolLmCache8Attend(_DTYPES[q.dtype], heads, q.data_ptr(), out.data_ptr(), q_row, q_head, out_row, out_head,
                                        self.dim ** -0.5 if scale is None else scale, softcap, 1.0, window, first, self._floats(sink, heads, "sink"),
                                        self._floats(slope, heads, "slope"))
        if penalty is not None:
            a.dist_r1, a.dist_r2 = self._floats(penalty[0], heads, "penalty[0]"), self._floats(penalty[1], heads, "penalty[1]")
        need = C.c_size_t()
        if self.device.index == torch.cuda.current_device():
            rc = self.lib.smol_lm_cache8_workspace_bytes(self._c, batch, a, need)
        else:
            with torch.cuda.device(self.device):
                rc = self.lib.smol_lm_cache8_workspace_bytes(self._c, batch, a, need)
        if rc != SMOL_OK:
            _capi_lm.check(rc)
        # of the call's own: from torch's allocator for this stream, or for the graph that is being captured
        work = torch.empty(need.value, dtype=torch.uint8, device=self.device) if need.value else None
        self._call(self.lib.smol_lm_cache8_attend, self._c, batch, a, work.data_ptr() if work is not None else None, need.value)
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
        if word:
            raise SmolError(SMOL_ERR_CAPACITY, f"device-side error word {word}: " + ("a block table names a page outside the cache" if word == 1 else "a batch's arrays do not fit its sizes"))
