"""ctypes binding of the attention part of libabq_gemm.so (the C ABI in include/abq_attention.h).

Works as abq_gemm.py does and on top of it: device buffers are torch tensors, there is no CPU fallback, and a call that the
library refuses raises AbqError.  Import torch before this module.
"""
import ctypes
import importlib.util
import math
import os
import struct
import sys

if "abq_gemm" not in sys.modules:
    _spec = importlib.util.spec_from_file_location("abq_gemm", os.path.join(os.path.dirname(os.path.abspath(__file__)), "abq_gemm.py"))
    _module = importlib.util.module_from_spec(_spec)
    sys.modules["abq_gemm"] = _module
    _spec.loader.exec_module(_module)
import abq_gemm  # noqa: E402
import torch  # noqa: E402

AbqError = abq_gemm.AbqError
F16, BF16 = 0, 1

# every symbol include/abq_attention.h declares
EXPORTED = [
    "abq_kv_codes_bytes", "abq_kv_scales_bytes", "abq_kv_append", "abq_kv_read",
    "abq_attn_prompt_init", "abq_attn_tree_init", "abq_attn_workspace_bytes", "abq_attn_set_workspace", "abq_attn_exec",
    "abq_rotary_apply", "abq_kv_append_rotary",
    "abq_kv_pages_fork", "abq_kv_pages_extend", "abq_kv_pages_compact", "abq_kv_copy_pages",
    "abq_kv_bound_codes_bytes", "abq_kv_bound_scales_bytes", "abq_kv_bound", "abq_attn_choose_workspace_bytes", "abq_attn_choose",
    "abq_attn_sparse_init", "abq_attn_sparse_workspace_bytes", "abq_attn_sparse_set_workspace", "abq_attn_sparse_exec",
]


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("rows", ctypes.c_int64), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class KvCacheDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("bits", "symmetric", "kv_heads", "head_dim", "page_size", "num_pages")] + \
               [(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "k_scales", "v_scales")]


class AttnState(ctypes.Structure):
    _fields_ = [
        ("init_success", ctypes.c_int), ("kind", ctypes.c_int), ("dtype", ctypes.c_int),
        ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
        ("seqs", ctypes.c_int), ("max_q", ctypes.c_int), ("max_k", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows),
        ("q_starts", ctypes.c_void_p), ("k_starts", ctypes.c_void_p),
        ("cache", KvCacheDesc),
        ("page_table", ctypes.c_void_p), ("context", ctypes.c_void_p), ("mask", ctypes.c_void_p),
        ("max_pages", ctypes.c_int), ("parts", ctypes.c_int), ("block_rows", ctypes.c_int),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class RotaryDesc(ctypes.Structure):
    _fields_ = [("rotary_dim", ctypes.c_int), ("axes", ctypes.c_int), ("interleaved", ctypes.c_int), ("turns", ctypes.c_void_p), ("axis", ctypes.c_void_p)]


class KvPagesDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("seqs", "max_pages", "page_size", "num_pages")] + [(n, ctypes.c_void_p) for n in ("table", "lengths", "refs")]


class KvBoundsDesc(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


class SparseState(ctypes.Structure):
    _fields_ = [("attn", AttnState), ("blocks", ctypes.c_void_p), ("count", ctypes.c_int)]


_lib = None


def lib():
    """libabq_gemm.so with the signatures of this part; raises if it has not been built (no fallback)."""
    global _lib
    if _lib is None:
        L = abq_gemm.lib()
        vp, ci, P = ctypes.c_void_p, ctypes.c_int, ctypes.POINTER
        for name in ("abq_kv_codes_bytes", "abq_kv_scales_bytes"):
            getattr(L, name).argtypes = [P(KvCacheDesc)]
            getattr(L, name).restype = ctypes.c_size_t
        for name in ("abq_kv_append", "abq_kv_read"):
            getattr(L, name).argtypes = [P(KvCacheDesc), P(Rows), P(Rows), ci, vp, vp]
        L.abq_attn_prompt_init.argtypes = [P(Rows)] * 4 + [ci] * 4 + [vp, vp] + [ci] * 3 + [ctypes.c_float, P(AttnState)]
        L.abq_attn_tree_init.argtypes = [P(KvCacheDesc), P(Rows), P(Rows), ci, ci, vp, ci, vp, vp, vp, ci, ci, ci, ctypes.c_float, P(AttnState)]
        L.abq_attn_workspace_bytes.argtypes = [P(AttnState)]
        L.abq_attn_workspace_bytes.restype = ctypes.c_size_t
        L.abq_attn_set_workspace.argtypes = [P(AttnState), vp, ctypes.c_size_t]
        L.abq_attn_exec.argtypes = [P(AttnState), vp]
        i64 = ctypes.c_int64
        # (rows as structures or as their bytes)
        L.abq_rotary_apply.argtypes = [P(RotaryDesc), vp, vp, ci, vp, vp, ci, ci, ci, vp, i64, vp]
        L.abq_kv_append_rotary.argtypes = [P(KvCacheDesc), P(RotaryDesc), vp, vp, ci, vp, vp, vp, ci, vp, i64, vp, vp]
        L.abq_kv_pages_fork.argtypes = [P(KvPagesDesc), vp, vp]
        L.abq_kv_pages_extend.argtypes = [P(KvPagesDesc), vp, vp, i64, vp, vp, vp, vp]
        L.abq_kv_pages_compact.argtypes = [P(KvPagesDesc), vp, vp]
        L.abq_kv_copy_pages.argtypes = [P(KvCacheDesc), P(KvBoundsDesc), vp, i64, vp]
        for name in ("abq_kv_bound_codes_bytes", "abq_kv_bound_scales_bytes"):
            getattr(L, name).argtypes = [P(KvCacheDesc)]
            getattr(L, name).restype = ctypes.c_size_t
        L.abq_kv_bound.argtypes = [P(KvCacheDesc), P(KvBoundsDesc), vp, i64, vp]
        L.abq_attn_choose_workspace_bytes.argtypes = [P(KvCacheDesc), ci, ci, ci, ci]
        L.abq_attn_choose_workspace_bytes.restype = ctypes.c_size_t
        L.abq_attn_choose.argtypes = [P(KvCacheDesc), P(KvBoundsDesc), P(Rows), ci, ci, vp, ci, vp, vp, ci, ci, ci, ci, ci, ci, vp, vp, ctypes.c_size_t, vp]
        L.abq_attn_sparse_init.argtypes = [P(KvCacheDesc), P(Rows), P(Rows), ci, ci, vp, ci, vp, vp, vp, vp, ci, ci, ci, ci, ctypes.c_float, P(SparseState)]
        L.abq_attn_sparse_workspace_bytes.argtypes = [P(SparseState)]
        L.abq_attn_sparse_workspace_bytes.restype = ctypes.c_size_t
        L.abq_attn_sparse_set_workspace.argtypes = [P(SparseState), vp, ctypes.c_size_t]
        L.abq_attn_sparse_exec.argtypes = [P(SparseState), vp]
        _lib = L
    return _lib


def _check(status, what):
    if status != abq_gemm.ABQ_OK:
        raise AbqError(status, what)


_DTYPES = {torch.float16: F16, torch.bfloat16: BF16}


def _dtype(t):
    if t.dtype not in _DTYPES:
        raise TypeError("fp16 or bf16 is wanted, got %s" % t.dtype)
    return _DTYPES[t.dtype]


def _rows(t):
    """A device tensor [rows, heads, head dim] as the library sees it"""
    strides = t.stride()
    if len(strides) != 3 or not t.is_cuda:
        raise ValueError("a device tensor [rows, heads, head dim] is wanted")
    if strides[2] != 1:
        raise ValueError("the elements of a head have to lie beside each other")
    return Rows(t.data_ptr(), t.shape[0], strides[0], strides[1])


_ROWS = struct.Struct("Pqqq").pack


def _row_bytes(t):
    """The same as the bytes of the structure, which take less time to make"""
    if t is None:
        return None
    strides = t.stride()
    if len(strides) != 3 or not t.is_cuda:
        raise ValueError("a device tensor [rows, heads, head dim] is wanted")
    if strides[2] != 1:
        raise ValueError("the elements of a head have to lie beside each other")
    return _ROWS(t.data_ptr(), t.shape[0], strides[0], strides[1])


def _index(t, dtype, numel, what):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous() or t.numel() != numel:
        raise ValueError("%s: a contiguous device tensor of %d %s is wanted" % (what, numel, dtype))
    return t.data_ptr()


# (with one device there is nowhere else to be)
_many_devices = torch.cuda.device_count() > 1


def _together(stream, *tensors):
    """Refuses tensors on another device than the one that a call on this stream runs on (a number as the stream does not say)"""
    if _many_devices:
        device = torch._C._cuda_getDevice() if stream is None else getattr(stream, "device_index", None)
        if device is not None and any(t is not None and t.get_device() not in (-1, device) for t in tensors):
            raise ValueError("a tensor is on another device than device %d, which the call runs on" % device)


def _stream_of(stream):
    """The torch stream that a call's argument stands for"""
    if stream is None:
        return torch.cuda.current_stream()
    return torch.cuda.ExternalStream(stream) if isinstance(stream, int) else stream


class _Memory:
    """Tensors that an object of this module allocated.  They belong to the stream that was current then.  A call on another stream first
    has that one wait for what still goes on with them here (once), and keeps them from being handed out again before it is done."""

    def __init__(self, tensors):
        self.tensors, self.home = tensors, torch.cuda.current_stream()
        self.known = {self.home.cuda_stream or None}  # (as ctypes has a null pointer)

    def use(self, stream):
        other = _stream_of(stream)
        with torch.cuda.stream(other):
            captured = torch.cuda.is_current_stream_capturing()
        for t in self.tensors:
            t.record_stream(other)
        if self.tensors and not captured:
            other.wait_stream(self.home)
        if not captured:  # (a capture may not wait for what is outside of it, and is replayed behind it)
            self.known.add(other.cuda_stream or None)


class _OnStream:
    """Objects whose calls take a stream and whose memory (self._memory) is safe on any"""

    def _on(self, stream):
        on = abq_gemm._stream_ptr(stream)
        if on.value not in self._memory.known:
            self._memory.use(stream)
        return on


class Rotary(_OnStream):
    """Rotary positions of a head's first 2 * len(turns) elements: pair i turns by turns[i] revolutions per position (float64), of the
    axis axis[i] (default: one axis).  Pairs are element i and i + len(turns), or neighbours if interleaved.  Both are copied to the device."""

    def __init__(self, turns, axis=None, axes=None, interleaved=False, device="cuda"):
        if torch.device(device).type != "cuda":
            raise ValueError("the angles have to be on the device, not on %s" % device)
        turns = torch.as_tensor(turns, dtype=torch.float64)
        if turns.dim() != 1 or not turns.numel() or turns.numel() % 8:
            raise ValueError("one number of revolutions for each of a multiple of 8 pairs is wanted")
        if axis is not None:
            axis = torch.as_tensor(axis, dtype=torch.int32)
            if axis.shape != turns.shape or int(axis.min()) < 0:
                raise ValueError("an axis, from 0, for each pair is wanted")
            axes = axes or int(axis.max()) + 1
            if int(axis.max()) >= axes:
                raise ValueError("there are %d axes" % axes)
        self.turns, self.axes = turns.to(device, copy=True).contiguous(), axes or 1  # (what is there already as well)
        self.axis = None if axis is None else axis.to(device, copy=True).contiguous()
        self.desc = RotaryDesc(2 * turns.numel(), self.axes, int(bool(interleaved)), self.turns.data_ptr(), None if axis is None else self.axis.data_ptr())
        self._ref = ctypes.byref(self.desc)
        self._memory = _Memory(tuple(t for t in (self.turns, self.axis) if t is not None))

    @classmethod
    def of_base(cls, dim, base=10000.0, sections=None, interleaved=False, device="cuda"):
        """The usual angles, base^(-2 i / dim) per position; sections: how many pairs each axis has, in order, if there are several."""
        pairs = dim // 2
        turns = torch.tensor([base ** (-i / pairs) / (2 * math.pi) for i in range(pairs)], dtype=torch.float64)
        axis = None
        if sections is not None:
            if sum(sections) != pairs:
                raise ValueError("sections of %d pairs in all are wanted" % pairs)
            axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
        return cls(turns, axis, None if sections is None else len(sections), interleaved, device)

    def _positions(self, positions, tokens):
        """(address, stride) of positions int32 [tokens], or [axes, tokens] with the tokens beside each other"""
        shape, strides = tuple(positions.shape), positions.stride()
        if shape != (self.axes, tokens) and (shape != (tokens,) or self.axes > 1) or not positions.is_cuda or positions.dtype != torch.int32 or (
                tokens > 1 and strides[-1] != 1):
            raise ValueError("positions: a device tensor [%d, %d] of torch.int32 is wanted" % (self.axes, tokens))
        return positions.data_ptr(), strides[0] if self.axes > 1 else tokens

    def apply(self, q, k, positions, out=None, stream=None):
        """(q, k) turned, [tokens, heads, dim] each, into out = (q, k), which may be q and k themselves; k may be None."""
        _together(stream, self.turns, q, k, positions, *(out or ()))
        on = self._on(stream)
        if k is not None and (k.dtype is not q.dtype or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]):
            raise ValueError("q [tokens, heads, dim] and k [tokens, kv heads, dim] of one type are wanted")
        if out is None:
            with torch.cuda.stream(None if stream is None else _stream_of(stream)):  # (tensors of the stream that they are written on)
                out = (torch.empty(q.shape, dtype=q.dtype, device=q.device), None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device))
        for x, y in zip((q, k), out):
            if (x is None) != (y is None) or (x is not None and (x.shape != y.shape or x.dtype is not y.dtype)):
                raise ValueError("out has to be of the inputs' shapes and type")
        at, step = self._positions(positions, q.shape[0])
        _check(lib().abq_rotary_apply(self._ref, _row_bytes(q), _row_bytes(out[0]), q.shape[1], _row_bytes(k), _row_bytes(out[1]),
                                      0 if k is None else k.shape[1], q.shape[2], _dtype(q), at, step, on), "abq_rotary_apply")
        return out


class Extension:
    """What PageTable.extend gives: slots [rows] of the new tokens, one sequence behind the other, starts [sequences + 1], granted [sequences]
    and copies [sequences, 2], the pages that KvCache.copy_pages has to copy in every layer before anything is written; int32."""

    def __init__(self, rows, sequences, whole):
        self.sizes, self.whole, self._parts = (rows, sequences + 1, sequences, 2 * sequences), whole, None
        first = whole.data_ptr()
        self.at = (first, first + 4 * rows, first + 4 * (rows + sequences + 1), first + 4 * (rows + 2 * sequences + 1))

    def _part(self, i):
        if self._parts is None:  # (views are made where they are looked at: four take as long as a launch)
            self._parts = self.whole.split(self.sizes)
        return self._parts[i]

    slots = property(lambda self: self._part(0))
    starts = property(lambda self: self._part(1))
    granted = property(lambda self: self._part(2))
    copies = property(lambda self: self._part(3).view(-1, 2))


class PageTable(_OnStream):
    """Which pages hold which sequence's tokens: table int32 [sequences, max_pages] (-1: none), lengths [sequences] and refs [num_pages], how
    many entries name each page, on the device.  Every sequence is empty at first."""

    def __init__(self, num_pages, page_size, sequences, max_pages, device="cuda"):
        if torch.device(device).type != "cuda":
            raise ValueError("the table has to be on the device, not on %s" % device)
        if min(num_pages, page_size, sequences, max_pages) < 1:
            raise ValueError("no such table: %d sequences of %d pages, of %d of %d tokens" % (sequences, max_pages, num_pages, page_size))
        self.table = torch.full((sequences, max_pages), -1, dtype=torch.int32, device=device)
        self.lengths, self.refs = (torch.zeros(n, dtype=torch.int32, device=device) for n in (sequences, num_pages))
        self.desc = KvPagesDesc(sequences, max_pages, page_size, num_pages, *(t.data_ptr() for t in (self.table, self.lengths, self.refs)))
        self._ref = ctypes.byref(self.desc)
        self._extend, self._fork = lib().abq_kv_pages_extend, lib().abq_kv_pages_fork
        self._memory = _Memory((self.table, self.lengths, self.refs))

    def _made(self, numbers, stream):
        if stream is None:
            return torch.empty(numbers, dtype=torch.int32, device=self.table.device)
        with torch.cuda.stream(_stream_of(stream)):  # (a tensor of the stream that it is written on)
            return torch.empty(numbers, dtype=torch.int32, device=self.table.device)

    def fork(self, parents, stream=None):
        """Sequence s takes over the tokens of sequence parents[s] (int32 [sequences]; -1: none) as they were before, on the same pages."""
        _together(stream, self.table, parents)
        at, on = _index(parents, torch.int32, self.desc.seqs, "parents"), self._on(stream)
        _check(self._fork(self._ref, at, on), "abq_kv_pages_fork")

    def extend(self, counts, rows, out=None, stream=None):
        """Room for counts[s] more tokens in sequence s (int32 [sequences]), or counts[s] < 0 taken away.  Returns an Extension, a new one or
        out, which an earlier call with as many rows has given."""
        _together(stream, self.table, counts, None if out is None else out.whole)
        at, on = _index(counts, torch.int32, self.desc.seqs, "counts"), self._on(stream)
        if out is None:
            out = Extension(rows, self.desc.seqs, self._made(rows + 4 * self.desc.seqs + 1, stream))
        elif out.sizes != (rows, self.desc.seqs + 1, self.desc.seqs, 2 * self.desc.seqs):
            raise ValueError("an Extension of %d rows and %d sequences is wanted" % (rows, self.desc.seqs))
        _check(self._extend(self._ref, at, out.at[0], rows, out.at[1], out.at[2], out.at[3], on), "abq_kv_pages_extend")
        return out

    def compact(self, out=None, stream=None):
        """Moves the live pages to the front; returns (or fills out with) moves [num_pages // 2, 2] for KvCache.copy_pages of every layer."""
        _together(stream, self.table, out)
        on, half = self._on(stream), self.desc.num_pages // 2
        out = self._made(2 * half, stream).view(half, 2) if out is None else out
        _check(lib().abq_kv_pages_compact(self._ref, _index(out, torch.int32, 2 * half, "moves"), on), "abq_kv_pages_compact")
        return out


class KvCache(_OnStream):
    """A paged cache of keys and values in codes of 8 or 4 bits with a scale (and a zero point) per token and head.

    A token's place is its slot, page * page_size + offset.  With zero points (symmetric=False) a row that lies more than 39 of its spreads
    from zero (8 bits; 667 with 4) is not held as what it is: zero points end at 1e4, scales begin at 1e-5.

    With bounds=True it has room for bounds of every page's keys (bound_codes int8 [pages, kv heads, 2, head dim], bound_scales [pages,
    kv heads]), which bound() writes and SparseAttention chooses pages by."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, bits=8, symmetric=True, device="cuda", bounds=False):
        if torch.device(device).type != "cuda":
            raise ValueError("the cache has to be on the device, not on %s" % device)
        d = KvCacheDesc(bits, int(bool(symmetric)), kv_heads, head_dim, page_size, num_pages)
        codes, scales = lib().abq_kv_codes_bytes(ctypes.byref(d)), lib().abq_kv_scales_bytes(ctypes.byref(d))
        if not codes:
            raise ValueError("no such cache: %d pages of %d tokens, %d heads of %d, %d bits" % (num_pages, page_size, kv_heads, head_dim, bits))
        self.k_codes, self.v_codes = (torch.zeros(codes, dtype=torch.uint8, device=device) for _ in range(2))
        self.k_scales, self.v_scales = (torch.ones(scales // 4, dtype=torch.float32, device=device) for _ in range(2))
        d.k_codes, d.v_codes, d.k_scales, d.v_scales = (t.data_ptr() for t in (self.k_codes, self.v_codes, self.k_scales, self.v_scales))
        self.desc = d
        self._ref, self._row = ctypes.byref(d), (kv_heads, head_dim)
        self._append, self._read, self._append_rotary = lib().abq_kv_append, lib().abq_kv_read, lib().abq_kv_append_rotary
        held = (self.k_codes, self.v_codes, self.k_scales, self.v_scales)
        self.bounds = self._bounds = None
        if bounds:
            self.bound_codes = torch.zeros((num_pages, kv_heads, 2, head_dim), dtype=torch.int8, device=device)
            self.bound_scales = torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=device)
            self.bounds = KvBoundsDesc(self.bound_codes.data_ptr(), self.bound_scales.data_ptr())
            self._bounds = ctypes.byref(self.bounds)
            held += (self.bound_codes, self.bound_scales)
        self._memory = _Memory(held)
        self._known = self._memory.known

    def _call(self, call, name, k, v, slots, stream):
        shape = k.shape
        if shape != v.shape or k.dtype is not v.dtype or shape[1:] != self._row:
            raise ValueError("keys and values [tokens, %d, %d] of one type are wanted" % self._row)
        at, on = _index(slots, torch.int32, shape[0], "slots"), abq_gemm._stream_ptr(stream)
        if on.value not in self._known:
            self._memory.use(stream)
        status = call(self._ref, ctypes.byref(_rows(k)), ctypes.byref(_rows(v)), _dtype(k), at, on)
        if status:
            raise AbqError(status, name)

    def append(self, k, v, slots, stream=None):
        """Quantises k and v [tokens, kv heads, head dim] and writes token i at slots[i] (int32; outside the cache: dropped)."""
        self._call(self._append, "abq_kv_append", k, v, slots, stream)

    def read(self, slots, dtype=None, out=None, stream=None):
        """(k, v) [tokens, kv heads, head dim] of the tokens at these slots, in fp16 (or dtype), or into out = (k, v)."""
        if out is None:
            shape = (slots.numel(),) + self._row
            with torch.cuda.stream(None if stream is None else _stream_of(stream)):  # (tensors of the stream that they are written on)
                out = tuple(torch.empty(shape, dtype=dtype or torch.float16, device=slots.device) for _ in range(2))
        self._call(self._read, "abq_kv_read", out[0], out[1], slots, stream)
        return out


    def append_rotated(self, rotary, q, k, v, positions, slots, q_out=None, k_out=None, stream=None):
        """Turns q and k by their positions and appends the turned k and v, in one launch.  Returns (q_out, k_out): the turned q, in a new
        tensor by default (None without q), and the turned k if k_out is given (the same tensors as q and k turn them in place)."""
        shape, dtype = k.shape, k.dtype
        if shape != v.shape or dtype is not v.dtype or shape[1:] != self._row:
            raise ValueError("keys and values [tokens, %d, %d] of one type are wanted" % self._row)
        heads = 0
        if q is not None:
            if q.dim() != 3 or q.dtype is not dtype or q.shape[::2] != shape[::2]:
                raise ValueError("q [%d, heads, %d] of the keys' type is wanted" % shape[::2])
            heads = q.shape[1]
            if q_out is None:
                with torch.cuda.stream(None if stream is None else _stream_of(stream)):
                    q_out = torch.empty(q.shape, dtype=dtype, device=q.device)
        for x, y in ((q, q_out), (k, k_out)):
            if y is not None and (x is None or x.shape != y.shape or y.dtype is not dtype):
                raise ValueError("q_out and k_out have to be of the inputs' shapes and type")
        _together(stream, self.k_codes, rotary.turns, q, k, v, q_out, k_out, positions, slots)
        at, on = _index(slots, torch.int32, shape[0], "slots"), self._on(stream)
        if on.value not in rotary._memory.known:
            rotary._memory.use(stream)
        turns, step = rotary._positions(positions, shape[0])
        status = self._append_rotary(self._ref, rotary._ref, _row_bytes(q), _row_bytes(q_out), heads, _row_bytes(k), _row_bytes(k_out), _row_bytes(v), _dtype(k),
                                     turns, step, at, on)
        if status:
            raise AbqError(status, "abq_kv_append_rotary")
        return q_out, k_out

    def copy_pages(self, pairs, stream=None):
        """Copies page pairs[i, 0] to page pairs[i, 1] (int32 [n, 2]; -1: nothing), bounds included."""
        if pairs.dim() != 2 or pairs.shape[1] != 2:
            raise ValueError("pairs of pages [n, 2] are wanted")
        _together(stream, self.k_codes, pairs)
        at, on = _index(pairs, torch.int32, pairs.numel(), "pairs"), self._on(stream)
        _check(lib().abq_kv_copy_pages(self._ref, self._bounds, at, pairs.shape[0], on), "abq_kv_copy_pages")

    def bound(self, slots, stream=None):
        """Writes the bounds of the pages that these slots complete: behind an append, with its slots."""
        if self.bounds is None:
            raise ValueError("this cache has no bounds")
        _together(stream, self.k_codes, slots)
        at, on = _index(slots, torch.int32, slots.numel(), "slots"), self._on(stream)
        _check(lib().abq_kv_bound(self._ref, self._bounds, at, slots.numel(), on), "abq_kv_bound")


class _Attention:
    _calls = ("abq_attn_workspace_bytes", "abq_attn_set_workspace", "abq_attn_exec")

    def _finish(self, out, workspace, *made):
        self.out = out
        need = self.workspace_bytes
        if workspace is not None and workspace.numel() and not (workspace.is_cuda and workspace.is_contiguous()):
            raise ValueError("a contiguous device tensor is wanted as the workspace")
        if workspace is None and need:
            workspace = torch.empty(need, dtype=torch.uint8, device=out.device)
            made += (workspace,)
        self.workspace = workspace
        self._memory = _Memory(made)
        self._known = self._memory.known
        if workspace is not None and workspace.numel():
            _check(getattr(lib(), self._calls[1])(ctypes.byref(self.state), workspace.data_ptr(), workspace.numel() * workspace.element_size()),
                   self._calls[1])
        self._exec, self._state = getattr(lib(), self._calls[2]), ctypes.byref(self.state)

    @property
    def workspace_bytes(self):
        return getattr(lib(), self._calls[0])(ctypes.byref(self.state))

    def run(self, stream=None):
        """One pass over what the tensors hold now; returns out.  A graph that captures it needs the object for as long as it is replayed."""
        on = abq_gemm._stream_ptr(stream)
        if on.value not in self._known:
            self._memory.use(stream)
        status = self._exec(self._state, on)
        if status:
            raise AbqError(status, self._calls[2])
        return self.out


class PromptAttention(_Attention):
    """Causal attention of packed prompts: q [tokens, heads, head dim], k and v [tokens, kv heads, head dim], sequence s in rows
    starts[s] .. starts[s + 1] - 1 (int32 on the device).  With k_starts, the queries are the last tokens of each sequence's keys.
    max_q, max_k: bounds of a sequence's queries (those beyond are not computed) and keys.  workspace: a device tensor of at least
    workspace_bytes; by default one is made, an empty tensor means none."""

    def __init__(self, q, k, v, q_starts, k_starts=None, max_q=None, max_k=None, scale=None, out=None, workspace=None):
        if k.shape != v.shape or k.shape[2] != q.shape[2] or not (q.dtype == k.dtype == v.dtype):
            raise ValueError("q [tokens, heads, head dim], k and v [tokens, kv heads, head dim] of one type are wanted")
        made = ()
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            made = (out,)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out has to be of q's shape and type")
        seqs = q_starts.numel() - 1
        max_q, max_k = max_q or q.shape[0] or 1, max_k or k.shape[0] or 1
        rows = [_rows(t) for t in (q, k, v, out)]
        at = [_index(t, torch.int32, seqs + 1, "starts") if t is not None else None for t in (q_starts, k_starts)]
        self.held = (q, k, v, q_starts, k_starts)
        self.state = AttnState()
        _check(lib().abq_attn_prompt_init(*[ctypes.byref(r) for r in rows], _dtype(q), q.shape[1], k.shape[1], q.shape[2], at[0], at[1],
                                          seqs, max_q, max_k, q.shape[2] ** -0.5 if scale is None else scale, ctypes.byref(self.state)), "abq_attn_prompt_init")
        self._finish(out, workspace, *made)


class TreeAttention(_Attention):
    """Attention of drafted tokens (ordinary decoding: one per sequence) over a KvCache: q [drafts, heads, head dim], sequence s in rows
    q_starts[s] .. q_starts[s + 1] - 1; page_table int32 [sequences, pages], context int32 [sequences]: tokens in front of the
    drafts, which stand behind them in the cache.  mask: int64 [drafts], bit j: sees draft j of its sequence; without one a draft sees
    those before it and itself.  max_q, max_context: bounds of a sequence's drafts (at most 64; those beyond are seen, not computed) and context."""

    def __init__(self, q, cache, page_table, context, q_starts, max_q, max_context, mask=None, scale=None, out=None, workspace=None):
        d = cache.desc
        if q.dim() != 3 or q.shape[2] != d.head_dim:
            raise ValueError("q [drafts, heads, %d] is wanted" % d.head_dim)
        made = ()
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            made = (out,)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out has to be of q's shape and type")
        seqs = context.numel()
        rows = [_rows(t) for t in (q, out)]
        table = _index(page_table, torch.int32, seqs * page_table.shape[-1], "page_table")
        self.held = (q, cache, page_table, context, q_starts, mask)
        self.state = AttnState()
        _check(lib().abq_attn_tree_init(ctypes.byref(d), ctypes.byref(rows[0]), ctypes.byref(rows[1]), _dtype(q), q.shape[1], table, page_table.shape[-1],
                                        _index(context, torch.int32, seqs, "context"), _index(q_starts, torch.int32, seqs + 1, "q_starts"),
                                        None if mask is None else _index(mask, torch.int64, q.shape[0], "mask"), seqs, max_q, max_context,
                                        q.shape[2] ** -0.5 if scale is None else scale, ctypes.byref(self.state)), "abq_attn_tree_init")
        self._finish(out, workspace, *made, *cache._memory.tensors)


class SparseAttention(_Attention):
    """Attention of drafted tokens as TreeAttention's, but every draft and key head sees only `count` of the context's complete pages, and what
    stands behind them: the first `first`, the last `last` (one each by default, as far as `count` has room, the last before the first), and
    those whose bounds promise the largest scores for its queries.  Each pass chooses them anew into blocks, int32 [drafts, kv heads, count];
    with blocks given, those are seen and nothing is chosen.  Passes on two streams at once need an object each."""

    _calls = ("abq_attn_sparse_workspace_bytes", "abq_attn_sparse_set_workspace", "abq_attn_sparse_exec")

    def __init__(self, q, cache, page_table, context, q_starts, max_q, max_context, count, first=None, last=None, mask=None, scale=None, out=None, workspace=None,
                 blocks=None):
        d = cache.desc
        if q.dim() != 3 or q.shape[2] != d.head_dim:
            raise ValueError("q [drafts, heads, %d] is wanted" % d.head_dim)
        if blocks is None and cache.bounds is None:
            raise ValueError("this cache has no bounds to choose pages by")
        last = min(1, max(0, count - (first or 0))) if last is None else last
        first = min(1, max(0, count - last)) if first is None else first
        if count < 1 or min(first, last) < 0 or first + last > count:
            raise ValueError("count >= first + last pages, one at least, are wanted")
        made = ()
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            made = (out,)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out has to be of q's shape and type")
        self._choose = blocks is None
        if blocks is None:
            blocks = torch.full((q.shape[0], d.kv_heads, count), -1, dtype=torch.int32, device=q.device)
            made += (blocks,)
        self.blocks, seqs = blocks, context.numel()
        rows = [_rows(t) for t in (q, out)]
        table = _index(page_table, torch.int32, seqs * page_table.shape[-1], "page_table")
        at = [_index(blocks, torch.int32, q.shape[0] * d.kv_heads * count, "blocks"), _index(context, torch.int32, seqs, "context"),
              _index(q_starts, torch.int32, seqs + 1, "q_starts")]
        _together(None, cache.k_codes, q, out, page_table, context, q_starts, mask, blocks, workspace)
        self.held = (q, cache, page_table, context, q_starts, mask, blocks)
        self.state = SparseState()
        _check(lib().abq_attn_sparse_init(ctypes.byref(d), ctypes.byref(rows[0]), ctypes.byref(rows[1]), _dtype(q), q.shape[1], table, page_table.shape[-1],
                                          at[1], at[2], None if mask is None else _index(mask, torch.int64, q.shape[0], "mask"), at[0], count, seqs, max_q,
                                          max_context, q.shape[2] ** -0.5 if scale is None else scale, ctypes.byref(self.state)), "abq_attn_sparse_init")
        if self._choose:
            if page_table.shape[-1] > 32768:
                raise AbqError(abq_gemm.ABQ_ERR_TOO_LARGE, "abq_attn_choose")
            need = lib().abq_attn_choose_workspace_bytes(ctypes.byref(d), page_table.shape[-1], seqs, max_q, max_context)
            scores = torch.empty(need // 4, dtype=torch.int32, device=q.device) if need else None
            made += (scores,) if need else ()
            self._chosen = (ctypes.byref(d), cache._bounds, ctypes.byref(rows[0]), _dtype(q), q.shape[1], table, page_table.shape[-1], at[1], at[2], seqs, max_q,
                            max_context, first, last, count, at[0], scores.data_ptr() if need else None, need)
        self._finish(out, workspace, *made, *cache._memory.tensors)

    def run(self, stream=None):
        """One pass over what the tensors hold now; returns out.  A graph that captures it needs the object for as long as it is replayed."""
        _together(stream, self.out)
        if self._choose:
            on = abq_gemm._stream_ptr(stream)
            if on.value not in self._known:
                self._memory.use(stream)
            _check(lib().abq_attn_choose(*self._chosen, on), "abq_attn_choose")
        return super().run(stream)
