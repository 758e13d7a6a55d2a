"""ctypes binding of the attention part of libabq_gemm.so (the C ABI in include/abq_attention.h).

Works as abq_gemm.py does and on top of it: device buffers are torch tensors, there is no CPU fallback, and a call that the
library refuses raises AbqError.  Import torch before this module.
"""
import ctypes
import importlib.util
import os
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


def _index(t, dtype, numel, what):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous() or t.numel() != numel:
        raise ValueError("%s: a contiguous device tensor of %d %s is wanted" % (what, numel, dtype))
    return t.data_ptr()


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


class KvCache:
    """A paged cache of keys and values in codes of 8 or 4 bits with a scale (and a zero point) per token and head.

    A token's place is its slot, page * page_size + offset.  With zero points (symmetric=False) a row that lies more than 39 of its spreads
    from zero (8 bits; 667 with 4) is not held as what it is: zero points end at 1e4, scales begin at 1e-5."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, bits=8, symmetric=True, device="cuda"):
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
        self._append, self._read = lib().abq_kv_append, lib().abq_kv_read
        self._memory = _Memory((self.k_codes, self.v_codes, self.k_scales, self.v_scales))
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


class _Attention:
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
            _check(lib().abq_attn_set_workspace(ctypes.byref(self.state), workspace.data_ptr(), workspace.numel() * workspace.element_size()),
                   "abq_attn_set_workspace")
        self._exec, self._state = lib().abq_attn_exec, ctypes.byref(self.state)

    @property
    def workspace_bytes(self):
        return lib().abq_attn_workspace_bytes(ctypes.byref(self.state))

    def run(self, stream=None):
        """One pass over what the tensors hold now; returns out.  A graph that captures it needs the object for as long as it is replayed."""
        on = abq_gemm._stream_ptr(stream)
        if on.value not in self._known:
            self._memory.use(stream)
        status = self._exec(self._state, on)
        if status:
            raise AbqError(status, "abq_attn_exec")
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
