"""Host side of attention on the quantised cache: symbols, structures, refusals, and how work is laid out.  No GPU."""
import ctypes
import os
import re
import subprocess

import pytest

pytest.importorskip("torch")

from attention_launch_probe import launches  # noqa: E402
from attention_reference import load_abq_attention  # noqa: E402
from conftest import ROOT  # noqa: E402


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def test_library_exports_every_declared_symbol(attn):
    header = open(os.path.join(ROOT, "include", "abq_attention.h")).read()
    declared = set(re.findall(r"^(?:abq_status|size_t)\s+(abq_\w+)\(", header, re.M))
    assert declared == set(attn.EXPORTED)
    for name in attn.EXPORTED:
        getattr(attn.lib(), name)


def test_structures_match_the_header(attn, tmp_path):
    src = '#include "abq_attention.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu %zu %zu", sizeof(abq_rows), ' \
          'sizeof(abq_kv_cache), sizeof(abq_attn_state), offsetof(abq_attn_state, q), offsetof(abq_attn_state, mask), ' \
          'offsetof(abq_attn_state, workspace));return 0;}'
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-x", "c", "-I" + os.path.join(ROOT, "include"), "-o", exe, "-"], input=src.encode(), check=True)
    want = [int(x) for x in subprocess.check_output([exe]).split()]
    assert want == [ctypes.sizeof(attn.Rows), ctypes.sizeof(attn.KvCacheDesc), ctypes.sizeof(attn.AttnState), attn.AttnState.q.offset,
                    attn.AttnState.mask.offset, attn.AttnState.workspace.offset]


A = 0x10000  # an address no call may reach: every check comes before


def cache_desc(attn, **kw):
    d = dict(bits=8, symmetric=1, kv_heads=2, head_dim=128, page_size=64, num_pages=10, k_codes=A, v_codes=2 * A, k_scales=3 * A, v_scales=4 * A)
    d.update(kw)
    return attn.KvCacheDesc(*d.values())


def test_cache_sizes(attn):
    L = attn.lib()
    for kw, codes, scales in [({}, 10 * 64 * 2 * 128, 10 * 64 * 2 * 4), ({"bits": 4, "symmetric": 0}, 10 * 64 * 2 * 64, 10 * 64 * 2 * 8),
                              ({"head_dim": 64, "page_size": 16, "kv_heads": 7}, 10 * 16 * 7 * 64, 10 * 16 * 7 * 4),
                              ({"num_pages": 1 << 24, "kv_heads": 40}, (1 << 30) * 40 * 128, (1 << 30) * 40 * 4),
                              ({"bits": 5}, 0, 0), ({"head_dim": 96}, 0, 0), ({"page_size": 8}, 0, 0), ({"page_size": 48}, 0, 0), ({"page_size": 8192}, 0, 0),
                              ({"num_pages": 0}, 0, 0), ({"kv_heads": -1}, 0, 0), ({"num_pages": 1 << 25}, 0, 0)]:
        d = cache_desc(attn, **kw)
        assert (L.abq_kv_codes_bytes(ctypes.byref(d)), L.abq_kv_scales_bytes(ctypes.byref(d))) == (codes, scales), kw
    assert L.abq_kv_codes_bytes(None) == 0
    with pytest.raises(ValueError):
        attn.KvCache(3, 20, 2, 128, device="cpu")


def rows(attn, **kw):
    d = dict(data=8 * A, rows=12, row_stride=256, head_stride=128)
    d.update(kw)
    return attn.Rows(*d.values())


BAD_ROWS = [{"data": None}, {"data": 8 * A + 8}, {"rows": -1}, {"rows": 11}, {"row_stride": 255}, {"head_stride": 130}, {"head_stride": 64}, {"row_stride": -256}]


def test_cache_calls_are_refused(attn):
    L, ok = attn.lib(), attn.abq_gemm
    for fn in (L.abq_kv_append, L.abq_kv_read):
        def call(c={}, k={}, v={}, dtype=0, slots=5 * A):
            return fn(ctypes.byref(cache_desc(attn, **c)), ctypes.byref(rows(attn, **k)), ctypes.byref(rows(attn, **v)), dtype, slots, None)
        for c in ({"bits": 3}, {"bits": 16}, {"head_dim": 80}):
            assert call(c=c) == ok.ABQ_ERR_UNSUPPORTED, c
        for c in ({"page_size": 20}, {"num_pages": 0}, {"kv_heads": 0}, {"k_codes": None}, {"v_codes": A + 4}, {"k_scales": None}, {"v_scales": A + 8}):
            assert call(c=c) == ok.ABQ_ERR_INVALID_ARG, c
        for bad in BAD_ROWS:
            assert call(v=bad) == ok.ABQ_ERR_INVALID_ARG, bad
            if "rows" not in bad:
                assert call(k=bad) == ok.ABQ_ERR_INVALID_ARG, bad
        assert call(dtype=2) == ok.ABQ_ERR_INVALID_ARG and call(slots=None) == ok.ABQ_ERR_INVALID_ARG
        assert call(k={"rows": 1 << 31}, v={"rows": 1 << 31}) == ok.ABQ_ERR_TOO_LARGE
        assert call(k={"rows": 0}, v={"rows": 0}, slots=None) == ok.ABQ_OK  # nothing to do: no launch
        assert fn(None, ctypes.byref(rows(attn)), ctypes.byref(rows(attn)), 0, A, None) == ok.ABQ_ERR_INVALID_ARG
        assert fn(ctypes.byref(cache_desc(attn)), None, ctypes.byref(rows(attn)), 0, A, None) == ok.ABQ_ERR_INVALID_ARG


def prompt(attn, q={}, k={}, v={}, out={}, dtype=0, heads=2, kv_heads=2, head_dim=128, q_starts=A, k_starts=A, seqs=2, max_q=10, max_k=10, scale=0.1):
    st = attn.AttnState()
    return attn.lib().abq_attn_prompt_init(*[ctypes.byref(rows(attn, **r)) for r in (q, k, v, out)], dtype, heads, kv_heads, head_dim, q_starts, k_starts,
                                           seqs, max_q, max_k, scale, ctypes.byref(st)), st


def tree(attn, cache={}, q={}, out={}, dtype=0, heads=2, page_table=A, max_pages=4, context=A, q_starts=A, mask=A, seqs=2, max_q=10, max_context=100, scale=0.1):
    st = attn.AttnState()
    return attn.lib().abq_attn_tree_init(ctypes.byref(cache_desc(attn, **cache)), ctypes.byref(rows(attn, **q)), ctypes.byref(rows(attn, **out)), dtype, heads,
                                         page_table, max_pages, context, q_starts, mask, seqs, max_q, max_context, scale, ctypes.byref(st)), st


def test_attention_calls_are_refused(attn):
    ok = attn.abq_gemm
    common = [{"dtype": 2}, {"dtype": -1}, {"heads": 0}, {"heads": 3}, {"q_starts": None}, {"seqs": 0}, {"max_q": 0}, {"scale": 0.0}, {"scale": -1.0},
              {"scale": float("nan")}, {"scale": float("inf")}] + [{"out": b} for b in BAD_ROWS] + [{"q": b} for b in BAD_ROWS]
    for kw in common + [{"kv_heads": 0}, {"max_k": 0}, {"k_starts": None, "k": {"rows": 13}, "v": {"rows": 13}}] + [{"v": b} for b in BAD_ROWS]:
        assert prompt(attn, **kw)[0] == ok.ABQ_ERR_INVALID_ARG and not prompt(attn, **kw)[1].init_success, kw
    for kw in common + [{"page_table": None}, {"context": None}, {"max_pages": 0}, {"max_context": -1}, {"cache": {"k_codes": None}}]:
        assert tree(attn, **kw)[0] == ok.ABQ_ERR_INVALID_ARG and not tree(attn, **kw)[1].init_success, kw
    assert prompt(attn, head_dim=96)[0] == ok.ABQ_ERR_UNSUPPORTED and tree(attn, cache={"bits": 2})[0] == ok.ABQ_ERR_UNSUPPORTED
    assert tree(attn, max_q=65)[0] == ok.ABQ_ERR_TOO_LARGE and tree(attn, max_pages=1 << 26)[0] == ok.ABQ_ERR_TOO_LARGE
    assert prompt(attn, max_q=2 ** 31 - 1, seqs=100000)[0] == ok.ABQ_ERR_TOO_LARGE
    assert tree(attn, max_q=64, seqs=2 ** 31 - 1)[0] == ok.ABQ_ERR_TOO_LARGE
    L, st = attn.lib(), attn.AttnState()
    assert L.abq_attn_exec(ctypes.byref(st), None) == ok.ABQ_ERR_NOT_INITIALIZED and L.abq_attn_exec(None, None) == ok.ABQ_ERR_INVALID_ARG
    assert L.abq_attn_set_workspace(ctypes.byref(st), A, 100) == ok.ABQ_ERR_NOT_INITIALIZED and L.abq_attn_workspace_bytes(ctypes.byref(st)) == 0
    assert L.abq_attn_prompt_init(None, None, None, None, 0, 1, 1, 64, None, None, 1, 1, 1, 1.0, None) == ok.ABQ_ERR_INVALID_ARG
    s, st = tree(attn)
    assert s == ok.ABQ_OK and st.init_success
    assert L.abq_attn_set_workspace(ctypes.byref(st), A + 8, 100) == ok.ABQ_ERR_INVALID_ARG
    assert L.abq_attn_set_workspace(ctypes.byref(st), None, 100) == ok.ABQ_ERR_INVALID_ARG
    s, st = tree(attn, q={"rows": 0}, out={"rows": 0})
    assert s == ok.ABQ_OK and L.abq_attn_exec(ctypes.byref(st), None) == ok.ABQ_OK  # no rows: no launch


def test_parts_follow_the_workspace(attn):
    L = attn.lib()
    s, st = tree(attn, max_q=1, max_context=30000, max_pages=600)
    need = L.abq_attn_workspace_bytes(ctypes.byref(st))
    assert st.parts == 1 and need > 0
    assert L.abq_attn_set_workspace(ctypes.byref(st), A, need) == 0 and st.parts > 1
    per_part = 12 * 2 * (128 + 2) * 4
    assert need == st.parts * per_part
    for parts in (1, 2, 3):
        assert L.abq_attn_set_workspace(ctypes.byref(st), A, parts * per_part + 5) == 0 and st.parts == parts
    assert L.abq_attn_set_workspace(ctypes.byref(st), None, 0) == 0 and st.parts == 1
    assert L.abq_attn_workspace_bytes(ctypes.byref(st)) == need  # what it would take is not what it has


def test_sizes_beyond_32_and_64_bits_are_refused(attn):
    ok = attn.abq_gemm
    most = 1 << 25  # 63 strides of 2-byte elements, a tile's last row, stay below 2^32
    assert prompt(attn, k={"row_stride": most}, v={"row_stride": most})[0] == ok.ABQ_OK
    for name in ("k", "v"):
        assert prompt(attn, **{name: {"row_stride": most + 8}})[0] == ok.ABQ_ERR_TOO_LARGE
    assert prompt(attn, q={"row_stride": 1 << 40}, out={"row_stride": 1 << 40})[0] == ok.ABQ_OK  # (addressed in 64 bits)
    top = 2 ** 31 - 1
    for kw in ({"max_q": top, "heads": top, "kv_heads": top, "seqs": top}, {"max_q": 1 << 26, "heads": 1 << 25, "kv_heads": 1, "seqs": 1 << 18},
               {"heads": top, "kv_heads": top, "seqs": top}):  # (the second is 2^64 blocks)
        assert prompt(attn, **kw)[0] == ok.ABQ_ERR_TOO_LARGE, kw
    for kw in ({"max_q": 64, "heads": top - 1, "seqs": top}, {"max_q": 64, "heads": 1 << 31 - 6, "cache": {"kv_heads": 1}, "seqs": top}):
        assert tree(attn, **kw)[0] == ok.ABQ_ERR_TOO_LARGE, kw


def test_parts_keep_launches_within_their_limit(attn):
    L, blocks = attn.lib(), 0xffffffff // 256
    # a generous bound of the contexts asks for many parts; many sequences leave room for few
    for seqs, max_q, heads, kv_heads in ((2000, 1, 32, 32), (70000, 1, 32, 8), (300, 64, 32, 8), (20000, 64, 32, 8), (1 << 20, 1, 8, 8)):
        s, st = tree(attn, cache={"kv_heads": kv_heads}, heads=heads, seqs=seqs, max_q=max_q, max_context=2 ** 31 - 100)
        assert s == attn.abq_gemm.ABQ_OK, (seqs, max_q)
        need = L.abq_attn_workspace_bytes(ctypes.byref(st))
        assert L.abq_attn_set_workspace(ctypes.byref(st), A, need) == 0
        rows = (max_q * heads // kv_heads + st.block_rows - 1) // st.block_rows
        assert (seqs * kv_heads * st.parts + 7) // 8 * 8 * rows <= blocks, (seqs, st.parts)
        assert st.parts == 1 or (seqs * max_q * heads + 3) // 4 <= blocks, (seqs, st.parts)


def test_a_scale_of_zero_is_refused_not_replaced(attn):
    class Fake(attn.torch.Tensor):  # a CPU tensor that says it is on the device: no launch is made
        is_cuda = True
    def fake(*shape, dtype=attn.torch.float16):
        return attn.torch.zeros(shape, dtype=dtype).as_subclass(Fake)
    q, starts = fake(4, 2, 64), fake(2, dtype=attn.torch.int32)
    with pytest.raises(attn.AbqError):
        attn.PromptAttention(q, q, q, starts, scale=0.0, out=q)


def test_scales_whose_product_with_a_tokens_is_beyond_fp32_are_refused(attn):
    ok = attn.abq_gemm
    for scale in (1e-38, 1e20, 2e30):
        assert prompt(attn, scale=scale)[0] == ok.ABQ_OK and tree(attn, scale=scale)[0] == ok.ABQ_OK, scale
    for scale in (3e30, 2e38):  # a token's scale and zero point may be 1e4 each
        assert prompt(attn, scale=scale)[0] == ok.ABQ_OK and tree(attn, scale=scale)[0] == ok.ABQ_ERR_INVALID_ARG, scale
    for scale in (2.5e38, 3e38):  # beyond fp32 once it is taken in powers of two
        assert prompt(attn, scale=scale)[0] == ok.ABQ_ERR_INVALID_ARG and tree(attn, scale=scale)[0] == ok.ABQ_ERR_INVALID_ARG, scale


def test_launches_stay_within_the_threads_that_hip_counts(attn, tmp_path):
    """Grid times workgroup of every launch below 2^32, whatever bound of the contexts is given"""
    sizes = [(64, 1, 32, 32, 1 << 25), (128, 1, 32, 32, 2 ** 31 - 164), (2000, 1, 32, 32, 2 ** 31 - 164), (70000, 1, 32, 8, 2 ** 31 - 164),
             (1 << 20, 1, 8, 8, 100), (1 << 20, 1, 8, 8, 2 ** 31 - 164), (131071, 1, 64, 64, 100), (131072, 1, 64, 64, 100), (262143, 4, 64, 32, 100),
             (20000, 64, 32, 8, 2 ** 31 - 164), (300, 64, 32, 8, 2 ** 31 - 164)]
    calls = [dict(kind="tree", rows=s * n, seqs=s, max_q=n, heads=h, kv_heads=kv, max_k=m) for s, n, h, kv, m in sizes]
    for c, r in zip(calls, launches(tmp_path, calls)):
        assert r["status"] == [0, 0, 0] and len(r["launches"]) == (1 if r["parts"] == 1 else 2), (c, r)
        for made in r["launches"]:
            assert made["grid"][0] * made["block"][0] < 2 ** 32 and made["grid"][1:] == made["block"][1:] == [1, 1], (c, made)
        rows = c["max_q"] * c["heads"] // c["kv_heads"]  # every row block of every part has its workgroup
        blocks = (rows + r["block_rows"] - 1) // r["block_rows"]
        assert r["launches"][0]["grid"][0] >= c["seqs"] * c["kv_heads"] * r["parts"] * blocks, (c, r)
    for c, r in zip(calls, launches(tmp_path, [dict(c, workspace=0) for c in calls])):
        assert r["status"] == [0, 0, 0] and r["parts"] == 1 and r["launches"][0]["grid"][0] * r["launches"][0]["block"][0] < 2 ** 32, (c, r)


def test_a_bound_of_the_keys_as_large_as_its_type_splits_them_as_any_large_one(attn, tmp_path):
    base = dict(kind="prompt", rows=64, heads=4, kv_heads=4, seqs=1, max_q=64)
    large = [dict(base, max_k=m) for m in (1 << 30, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1)]
    made = launches(tmp_path, large)
    assert all(r["status"] == [0, 0, 0] and r == made[0] and r["parts"] == 64 for r in made), made


class StreamsOfHand:
    """torch.cuda's streams, written down instead of made: what the binding asks of them, in order"""

    class Stream:
        def __init__(self, streams, at):
            self.cuda_stream, self.streams = at, streams

        def wait_stream(self, other):
            self.streams.log.append(("wait", self.cuda_stream, other.cuda_stream))

    def __init__(self, torch, monkeypatch):
        self.log, self.captured, self.current = [], False, None
        self.current = self.home = self.Stream(self, 0x10)

        class Inside:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(inside):
                inside.before, self.current = self.current, inside.stream or self.current

            def __exit__(inside, *_):
                self.current = inside.before

        empty = torch.empty

        def make(*shape, **kw):
            t = empty(*shape, **kw)
            self.log.append(("made", self.current.cuda_stream))
            return t
        monkeypatch.setattr(torch, "empty", make)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: self.current)
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda at, *_: self.Stream(self, at))
        monkeypatch.setattr(torch.cuda, "stream", Inside)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.captured)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.log.append(("keep", t.data_ptr(), s.cuda_stream)))

    def taken(self):
        log, self.log = self.log, []
        return log


def test_memory_that_the_binding_makes_is_safe_on_other_streams(attn, monkeypatch):
    """The workspace and the result belong to the stream that was current: another one waits for it once before the first launch, and
    keeps the memory from being handed out"""
    torch = attn.torch

    class Fake(torch.Tensor):  # a CPU tensor that says it is on the device: no launch is made
        is_cuda = True
    on_device = lambda t: t.as_subclass(Fake)  # noqa: E731
    streams = StreamsOfHand(torch, monkeypatch)
    monkeypatch.setattr(attn, "_rows", lambda t: attn.Rows(t.data_ptr(), t.shape[0], t.stride(0), t.stride(1)))
    q, k = on_device(torch.zeros(40, 2, 128).half()), on_device(torch.zeros(1500, 2, 128).half())
    starts = [on_device(torch.tensor([0, n], dtype=torch.int32)) for n in (40, 1500)]
    call = attn.PromptAttention(q, k, k, *starts, 40, 1500)
    assert call.state.parts > 1 and streams.taken() == [("made", 0x10)] * 2
    call._exec = lambda state, on: streams.log.append(("run", on.value)) or 0
    memory = {call.workspace.data_ptr(), call.out.data_ptr()}
    other = streams.Stream(streams, 0x20)

    def kept(log, at):
        assert {e[1] for e in log if e[0] == "keep"} == memory and all(e[2] == at for e in log if e[0] == "keep"), log
        return [e for e in log if e[0] != "keep"]

    call.run(stream=streams.home)
    assert streams.taken() == [("run", 0x10)]
    call.run(stream=other)
    assert kept(streams.taken(), 0x20) == [("wait", 0x20, 0x10), ("run", 0x20)]
    call.run(stream=other)
    call.run(stream=0x20)
    assert streams.taken() == [("run", 0x20)] * 2
    streams.captured = True  # a capture does not wait for what is outside of it
    call.run(stream=0x30)
    assert kept(streams.taken(), 0x30) == [("run", 0x30)]
    streams.captured = False
    call.run(stream=0x30)
    assert kept(streams.taken(), 0x30) == [("wait", 0x30, 0x10), ("run", 0x30)]

    # what the caller brings is the caller's
    mine = attn.PromptAttention(q, k, k, *starts, 40, 1500, out=on_device(torch.zeros(40, 2, 128).half()),
                                workspace=on_device(torch.zeros(call.workspace.numel(), dtype=torch.uint8)))
    mine._exec = call._exec
    streams.taken()
    mine.run(stream=other)
    assert streams.taken() == [("run", 0x20)]

    # the cache's arrays, and rows that are read back
    for name in ("zeros", "ones"):
        monkeypatch.setattr(torch, name, lambda *a, make=getattr(torch, name), device=None, **kw: make(*a, **kw))
    cache = attn.KvCache(4, 64, 2, 128)
    cache._append = cache._read = lambda *a: streams.log.append(("run", a[-1].value)) or 0
    memory = {t.data_ptr() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)}
    slots = on_device(torch.zeros(40, dtype=torch.int32))
    streams.taken()
    cache.append(q, q, slots, stream=other)
    assert kept(streams.taken(), 0x20) == [("wait", 0x20, 0x10), ("run", 0x20)]
    cache.read(slots, stream=other)
    assert streams.taken() == [("made", 0x20)] * 2 + [("run", 0x20)]
    cache.read(slots, stream=streams.home)
    assert streams.taken() == [("made", 0x10)] * 2 + [("run", 0x10)]
    table, context = on_device(torch.zeros(1, 4, dtype=torch.int32)), on_device(torch.zeros(1, dtype=torch.int32))
    tree = attn.TreeAttention(q[:1], cache, table, context, starts[0], 1, 200)
    tree._exec = call._exec
    memory |= {tree.out.data_ptr()}
    streams.taken()
    tree.run(stream=other)
    assert kept(streams.taken(), 0x20) == [("wait", 0x20, 0x10), ("run", 0x20)]


def test_results_whose_rows_lie_on_one_another_are_refused(attn):
    """Rows that are read may repeat (a stride of 0); rows that are written would race"""
    L, ok = attn.lib(), attn.abq_gemm
    for stride in (0, 8, 120):
        flat = {"row_stride": stride}
        assert prompt(attn, q=flat, k=flat, v=flat)[0] == ok.ABQ_OK and tree(attn, q=flat)[0] == ok.ABQ_OK, stride
        assert prompt(attn, out=flat)[0] == ok.ABQ_ERR_INVALID_ARG and tree(attn, out=flat)[0] == ok.ABQ_ERR_INVALID_ARG, stride
        for k, v in ((flat, {}), ({}, flat)):
            args = [ctypes.byref(cache_desc(attn)), ctypes.byref(rows(attn, **k)), ctypes.byref(rows(attn, **v)), 0, 5 * A, None]
            assert L.abq_kv_read(*args) == ok.ABQ_ERR_INVALID_ARG, stride
        # heads outermost, and a single row whose stride says nothing
        assert prompt(attn, out={"row_stride": 128, "head_stride": 12 * 128})[0] == ok.ABQ_OK
        one = {"rows": 1, "row_stride": stride}
        assert prompt(attn, q=one, k=one, v=one, out=one)[0] == ok.ABQ_OK, stride


def test_memory_of_the_host_is_refused(attn):
    """The binding hands out addresses that the kernels read and write: what is not on the device, or not in one piece, never gets there"""
    torch = attn.torch

    class Fake(torch.Tensor):  # a CPU tensor that says it is on the device: no launch is made
        is_cuda = True
    on_device = lambda t: t.as_subclass(Fake)  # noqa: E731
    with pytest.raises(ValueError):
        attn.KvCache(4, 64, 2, 128, device="cpu")
    q, k = on_device(torch.zeros(40, 2, 128).half()), on_device(torch.zeros(1500, 2, 128).half())
    starts = [on_device(torch.tensor([0, n], dtype=torch.int32)) for n in (40, 1500)]
    for workspace in (torch.zeros(1 << 20, dtype=torch.uint8), on_device(torch.zeros(1 << 14, 64, dtype=torch.uint8))[:, :32]):
        with pytest.raises(ValueError):
            attn.PromptAttention(q, k, k, *starts, 40, 1500, out=torch.empty_like(q), workspace=workspace)
