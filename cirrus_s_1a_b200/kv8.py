"""A K/V cache in 8 bits (``CbKv8`` of ``include/cirrus_b200.h``): append,
attention, and eviction by accumulated attention weight.

    cache = Kv8Cache(batch, n_kv_heads, head_dim, max_len, fmt="e4m3")
    cache.append(k, v, pos)                    # T tokens per sequence behind pos[b]
    out, lse = cache.attend(q, pos)            # their queries, causal
    kept, pos = cache.evict(pos + T, keep, recent)

Keys and values are held as E4M3 or int8 codes with one scale, a power of two,
for each block of 64 slots and KV head.  ``pos`` is a device int32 tensor: the
slots of each sequence in use before the call.  Calls enqueue work on the
current stream and do not synchronise.  The attention's scratch belongs to the
cache and to one stream: calls of one cache from several streams get one each, and
a call that a CUDA graph captures gets its own, from the graph's memory.

The reference keeps the shared K/V in the model's type
(``cirrus/model/model.py:41-51``); this is its bounded form for long texts.
"""

from __future__ import annotations

import ctypes as C

import torch

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200._lib import CB_KV8_BLOCK, CbKv8

FORMATS = {"e4m3": (_lib.CB_KV8_E4M3, torch.float8_e4m3fn), "int8": (_lib.CB_KV8_INT8, torch.int8)}
DTYPES = {torch.float32: _lib.CB_F32, torch.bfloat16: _lib.CB_BF16, torch.float16: _lib.CB_F16}
HEAD_DIMS = (16, 32, 64, 128)

_Strides = C.c_int64 * 3


#: device index -> the current stream's pointer (what ``torch.cuda.current_stream`` wraps, without the object)
raw_stream = torch._C._cuda_getCurrentRawStream if torch.cuda.is_available() else None
#: whether the current stream is being captured (``torch.cuda.is_current_stream_capturing`` without its wrapper)
capturing = torch._C._cuda_isCurrentStreamCapturing if torch.cuda.is_available() else None
current_device = torch._C._cuda_getDevice if torch.cuda.is_available() else None


def _dtype(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


class Kv8Cache:
    """``batch`` sequences of up to ``max_len`` slots (rounded up to whole blocks of 64)."""

    def __init__(self, batch: int, n_kv_heads: int, head_dim: int, max_len: int, fmt: str = "e4m3", device="cuda",
                 mass: bool = True):
        if fmt not in FORMATS:
            raise ValueError(f"unknown format {fmt!r}; choose from {sorted(FORMATS)}")
        if min(batch, n_kv_heads, max_len) <= 0:
            raise ValueError("batch, n_kv_heads and max_len must be positive")
        if not torch.cuda.is_available():
            raise _lib.CbError("Kv8Cache needs a CUDA device (there is no CPU path)")
        L = -(-max_len // CB_KV8_BLOCK) * CB_KV8_BLOCK
        k, v = (torch.zeros(batch, n_kv_heads, L, head_dim, dtype=torch.uint8, device=device).view(FORMATS[fmt][1])
                for _ in range(2))
        ks, vs = (torch.ones(batch, n_kv_heads, L // CB_KV8_BLOCK, device=device) for _ in range(2))
        self._bind(k, v, ks, vs, torch.zeros(batch, n_kv_heads, L, device=device) if mass else None)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     mass: torch.Tensor | None = None) -> "Kv8Cache":
        """A cache over existing tensors (not copied): codes [B, H, L, D] as
        float8_e4m3fn or int8, scales float32 [B, H, L / 64], mass float32 [B, H, L]."""
        c = cls.__new__(cls)
        c._bind(k, v, k_scale, v_scale, mass)
        return c

    def _bind(self, k, v, k_scale, v_scale, mass) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [batch, heads, slots, dim] of one shape and type")
        fmt = next((n for n, (_, dt) in FORMATS.items() if dt == k.dtype), None)
        if fmt is None:
            raise ValueError(f"codes are float8_e4m3fn or int8, not {k.dtype}")
        B, H, L, D = k.shape
        if min(B, H, L) <= 0 or L % CB_KV8_BLOCK:
            raise ValueError(f"the slots ({L}) must be a positive multiple of {CB_KV8_BLOCK}")
        if D not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, not {D}")
        for name, t, shape in (("k_scale", k_scale, (B, H, L // CB_KV8_BLOCK)),
                               ("v_scale", v_scale, (B, H, L // CB_KV8_BLOCK)), ("mass", mass, (B, H, L))):
            if t is not None and (t.shape != shape or t.dtype != torch.float32):
                raise ValueError(f"{name} must be float32 of shape {shape}")
        for t in (k, v, k_scale, v_scale, mass):
            if t is not None and (not t.is_cuda or t.device != k.device or not t.is_contiguous()):
                raise ValueError("the cache's tensors must be contiguous and on one CUDA device")
        self.batch, self.n_kv_heads, self.max_len, self.head_dim, self.fmt = B, H, L, D, fmt
        self.k, self.v, self.k_scale, self.v_scale, self.mass = k, v, k_scale, v_scale, mass
        self.device = k.device
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._struct = CbKv8(B, H, D, L, FORMATS[fmt][0], k.data_ptr(), v.data_ptr(), k_scale.data_ptr(),
                             v_scale.data_ptr(), _lib.ptr(mass))
        self._ref = C.addressof(self._struct)
        self._lib = _lib.lib()
        self._scratch: dict = {}  # stream -> buffer; one serves every shape
        self._sizes: dict = {}  # shape -> bytes
        self._hits: dict = {}  # (stream, *shape) -> the stream's buffer, once it is known to be long enough
        self.workspaces: dict = {}  # of the model's forward over this cache, by chunk length

    # ------------------------------------------------------------- helpers
    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.mass)
                   if t is not None)

    def clone(self) -> "Kv8Cache":
        return Kv8Cache.from_tensors(*(None if t is None else t.clone()
                                       for t in (self.k, self.v, self.k_scale, self.v_scale, self.mass)))

    def values(self) -> tuple:
        """(k, v) as float32 [B, H, L, D]: code * scale of every slot, in use or not."""
        def of(codes, scale):
            return (codes.float().unflatten(2, (-1, CB_KV8_BLOCK)) * scale[..., None, None]).flatten(2, 3)

        return of(self.k, self.k_scale), of(self.v, self.v_scale)

    def read_status(self) -> int:
        """The device status (0; 5 when an append passed ``max_len``; 8 when a wait gave up); synchronises."""
        return int(self.status.item())

    def clear_status(self) -> None:
        self.status.zero_()

    def _ints(self, t, name: str) -> int | None:
        if t is None:
            return None
        if t.dtype != torch.int32 or t.shape != (self.batch,) or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor [{self.batch}] on {self.device}")
        return t.data_ptr()

    def _rows(self, t, name: str, heads: int | None):
        """(T, heads, strides) of a [B, T, heads, D] tensor with contiguous dims."""
        if t.dim() != 4 or t.shape[0] != self.batch or t.shape[3] != self.head_dim or t.device != self.device:
            raise ValueError(f"{name} must be [{self.batch}, T, heads, {self.head_dim}] on {self.device}")
        if heads is not None and t.shape[2] != heads:
            raise ValueError(f"{name} must have {heads} heads, not {t.shape[2]}")
        if t.shape[1] <= 0:
            raise ValueError(f"{name} must hold at least one token")
        sb, st, sh, sd = t.stride()
        if sd != 1:
            raise ValueError(f"{name}'s last dimension must be contiguous")
        return t.shape[1], t.shape[2], _Strides(sb, st, sh)

    def _stream(self) -> int:
        return raw_stream(self.device.index)

    def _call(self, fn, what: str, *args) -> None:
        if current_device() == self.device.index:
            rc = fn(*args)
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args)
        if rc:
            _lib.check(rc, what)

    # ----------------------------------------------------------- operators
    def append(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """Writes the T tokens of ``k`` / ``v`` [B, T, heads, D] (``counts[b]`` of
        them) to slots ``pos[b]`` .. and zeroes their mass (``cb_kv8_append``).
        ``pos`` is not advanced; tokens past ``max_len`` are dropped and noted in
        the device status."""
        T, _, ks = self._rows(k, "k", self.n_kv_heads)
        Tv, _, vs = self._rows(v, "v", self.n_kv_heads)
        if T != Tv or k.dtype != v.dtype:
            raise ValueError("k and v must hold the same tokens in one type")
        if T > self.max_len:
            raise _lib.CbError(f"context full: {T} tokens > max_len {self.max_len}")
        self._call(self._lib.cb_kv8_append, "cb_kv8_append", self._ref, k.data_ptr(), v.data_ptr(), _dtype(k, "k"), ks,
                   vs, T, self._ints(pos, "pos"), self._ints(counts, "counts"), self.status.data_ptr(),
                   self._stream())

    def attend(self, q: torch.Tensor, pos: torch.Tensor, counts: torch.Tensor | None = None, *,
               scale: float | None = None, add_mass: bool = False, longest: int | None = None,
               out: torch.Tensor | None = None) -> tuple:
        """Causal attention of the queries ``q`` [B, T, query heads, D] of the T
        tokens behind ``pos[b]``: row t sees slots up to ``pos[b] + t``.  Returns
        (out [B, T, query heads, D] in q's type, lse float32 [B, T, query heads]);
        rows that see nothing give 0 and -inf, rows whose query is not finite or that see
        a NaN key give NaN.  ``scale`` defaults to D ** -0.5;
        ``add_mass`` adds each slot's probabilities to ``mass``; ``longest`` bounds
        ``pos + T`` and sizes the launch (default ``max_len``) (``cb_kv8_attend``)."""
        if current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.attend(q, pos, counts, scale=scale, add_mass=add_mass, longest=longest, out=out)
        T, heads, qs = self._rows(q, "q", None)
        if heads % self.n_kv_heads:
            raise ValueError(f"{heads} query heads do not divide among {self.n_kv_heads} KV heads")
        if add_mass and self.mass is None:
            raise ValueError("this cache keeps no mass")
        longest = self.max_len if longest is None else min(int(longest), self.max_len)
        dtype = _dtype(q, "q")
        if out is None:
            out = torch.empty(self.batch, T, heads, self.head_dim, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError("out must be contiguous, of q's shape, type and device")
        lse = torch.empty(self.batch, T, heads, dtype=torch.float32, device=self.device)
        st = self._stream()
        key = (st, dtype, heads, T, longest, add_mass)
        scratch = None if capturing() else self._hits.get(key)
        if scratch is None:
            scratch = self._scratch_of(*key)
        rc = self._lib.cb_kv8_attend(self._ref, q.data_ptr(), dtype, qs, heads, T, self._ints(pos, "pos"),
                                     self._ints(counts, "counts"), longest,
                                     self.head_dim ** -0.5 if scale is None else float(scale), int(add_mass),
                                     out.data_ptr(), lse.data_ptr(), scratch.data_ptr(), scratch.numel(),
                                     self.status.data_ptr(), st)
        if rc:
            _lib.check(rc, "cb_kv8_attend")
        return out, lse

    def _scratch_of(self, stream: int, dtype: int, heads: int, T: int, longest: int, add_mass: bool) -> torch.Tensor:
        key = (dtype, heads, T, longest, add_mass)
        nbytes = self._sizes.get(key)
        if nbytes is None:
            nbytes = self._lib.cb_kv8_attend_scratch_bytes(self._ref, dtype, heads, T, longest, int(add_mass))
            if nbytes == 0:
                raise _lib.CbError("cb_kv8_attend_scratch_bytes: shape not supported")
            if len(self._sizes) >= 256:  # a caller's ``longest`` may change with every token
                self._sizes.clear()
                self._hits.clear()
            self._sizes[key] = nbytes
        if capturing():
            # from the graph's pool, and zeroed by each replay: the stream's buffer may be replaced by a
            # longer one, and what it holds is not zero before the graph's own first replay
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            scratch[:_lib.CB_KV8_ZEROED].zero_()
            return scratch
        scratch = self._scratch.get(stream)
        if scratch is None or scratch.numel() < nbytes:
            scratch = self._scratch[stream] = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
            self._hits.clear()
        self._hits[(stream, *key)] = scratch
        return scratch

    def evict(self, pos: torch.Tensor, keep: int, recent: int) -> tuple:
        """Brings every sequence of more than ``keep`` tokens down to ``keep``, per
        KV head: the ``recent`` last slots and the older ones of largest mass, ties
        to the lowest slot, moved to slots 0 .. keep - 1 in order (``cb_kv8_evict``).
        Returns (kept int32 [B, heads, keep]: the slots they came from, -1 past the
        end of a shorter sequence; pos int32 [B]: min(pos, keep))."""
        if self.mass is None:
            raise ValueError("this cache keeps no mass")
        if not 0 < keep <= self.max_len or not 0 <= recent <= keep:
            raise ValueError("eviction needs 0 < keep <= max_len and 0 <= recent <= keep")
        kept = torch.empty(self.batch, self.n_kv_heads, keep, dtype=torch.int32, device=self.device)
        new_pos = torch.empty(self.batch, dtype=torch.int32, device=self.device)
        self._call(self._lib.cb_kv8_evict, "cb_kv8_evict", self._ref, self._ints(pos, "pos"), int(keep), int(recent),
                   kept.data_ptr(), new_pos.data_ptr(), self._stream())
        return kept, new_pos
