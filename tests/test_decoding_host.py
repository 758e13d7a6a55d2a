"""Host side of rotary positions, pages of sequences and attention to chosen pages: structures, sizes, refusals.  No GPU."""
import ctypes
import os
import subprocess

import pytest

pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_attention_host import A, BAD_ROWS, StreamsOfHand, cache_desc, rows  # noqa: E402


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def ref(x):
    return None if x is None else ctypes.byref(x)


def test_structures_match_the_header(attn, tmp_path):
    src = '#include "abq_attention.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu %zu %zu %zu", sizeof(abq_rotary), ' \
          'offsetof(abq_rotary, axis), sizeof(abq_kv_pages), offsetof(abq_kv_pages, refs), sizeof(abq_kv_bounds), sizeof(abq_sparse_state), ' \
          'offsetof(abq_sparse_state, count));return 0;}'
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-x", "c", "-I" + os.path.join(ROOT, "include"), "-o", exe, "-"], input=src.encode(), check=True)
    want = [int(x) for x in subprocess.check_output([exe]).split()]
    assert want == [ctypes.sizeof(attn.RotaryDesc), attn.RotaryDesc.axis.offset, ctypes.sizeof(attn.KvPagesDesc), attn.KvPagesDesc.refs.offset,
                    ctypes.sizeof(attn.KvBoundsDesc), ctypes.sizeof(attn.SparseState), attn.SparseState.count.offset]


def rotary(attn, **kw):
    d = dict(rotary_dim=128, axes=1, interleaved=0, turns=7 * A, axis=None)
    d.update(kw)
    return attn.RotaryDesc(*d.values())


BAD_ROTARY = [{"rotary_dim": 0}, {"rotary_dim": -16}, {"rotary_dim": 24}, {"rotary_dim": 144}, {"axes": 0}, {"axes": 9}, {"turns": None}, {"turns": 7 * A + 4}]


def test_turning_is_refused(attn):
    L, ok = attn.lib(), attn.abq_gemm

    def apply(r={}, q={}, q_out={}, k={}, k_out={}, heads=2, kv_heads=2, dim=128, dtype=0, positions=6 * A, stride=12):
        args = [None if x is None else rows(attn, **dict({"data": (8 + 4 * i) * A}, **x)) for i, x in enumerate((q, q_out, k, k_out))]
        return L.abq_rotary_apply(ref(None if r is None else rotary(attn, **r)), ref(args[0]), ref(args[1]), heads, ref(args[2]), ref(args[3]), kv_heads, dim, dtype,
                                  positions, stride, None)

    for r in BAD_ROTARY + [None]:
        assert apply(r=r) == ok.ABQ_ERR_INVALID_ARG, r
    for bad in BAD_ROWS:
        assert apply(q_out=bad) == ok.ABQ_ERR_INVALID_ARG and apply(k=bad) == ok.ABQ_ERR_INVALID_ARG and apply(k_out=bad) == ok.ABQ_ERR_INVALID_ARG, bad
    for kw in ({"q": None}, {"q_out": None}, {"k_out": None}, {"heads": 0}, {"kv_heads": 0}, {"dtype": 2}, {"positions": None}, {"dim": 0}, {"dim": -16}, {"stride": -1},
               {"r": {"axes": 2}, "stride": 11}, {"q_out": {"row_stride": 0}}, {"q_out": {"row_stride": 120}}):
        assert apply(**kw) == ok.ABQ_ERR_INVALID_ARG, kw
    same = {"data": 8 * A}
    assert apply(q=same, q_out=dict(same, row_stride=512)) == ok.ABQ_ERR_INVALID_ARG and apply(q=same, q_out=dict(same, head_stride=1536)) == ok.ABQ_ERR_INVALID_ARG
    for dim in (8, 72, 272):
        assert apply(dim=dim) == ok.ABQ_ERR_UNSUPPORTED
    many = {"rows": 1 << 31}
    assert apply(q=many, q_out=many, k=many, k_out=many, stride=1 << 31) == ok.ABQ_ERR_TOO_LARGE
    wide = {"head_stride": 128, "row_stride": 1 << 40}
    assert apply(q=wide, q_out=wide, heads=1 << 30) == ok.ABQ_ERR_TOO_LARGE
    none = {"rows": 0, "data": None}
    assert apply(q=none, q_out=none, k=none, k_out=none, positions=None) == ok.ABQ_OK  # nothing to do: no launch

    def append(c={}, r={}, q={}, q_out={}, k={}, k_out={}, v={}, heads=2, dtype=0, positions=6 * A, stride=12, slots=5 * A):
        args = [None if x is None else rows(attn, **dict({"data": (8 + 4 * i) * A}, **x)) for i, x in enumerate((q, q_out, k, k_out, v))]
        return L.abq_kv_append_rotary(ref(cache_desc(attn, **c)), ref(None if r is None else rotary(attn, **r)), ref(args[0]), ref(args[1]), heads, ref(args[2]), ref(args[3]),
                                      ref(args[4]), dtype, positions, stride, slots, None)

    for r in BAD_ROTARY + [None]:
        assert append(r=r) == ok.ABQ_ERR_INVALID_ARG, r
    assert append(c={"head_dim": 64}) == ok.ABQ_ERR_INVALID_ARG  # (more elements turn than there are)
    for c in ({"bits": 3}, {"head_dim": 80}):
        assert append(c=c) == ok.ABQ_ERR_UNSUPPORTED, c
    for bad in BAD_ROWS:
        for name in ("q", "q_out", "k_out", "v"):
            assert append(**{name: bad}) == ok.ABQ_ERR_INVALID_ARG, (name, bad)
    for kw in ({"c": {"k_codes": None}}, {"q": None}, {"q_out": None}, {"k": None}, {"v": None}, {"heads": 0}, {"dtype": -1}, {"slots": None}, {"positions": None},
               {"v": {"data": 12 * A}}, {"v": {"data": 20 * A}}):
        assert append(**kw) == ok.ABQ_ERR_INVALID_ARG, kw
    assert append(**{n: many for n in ("q", "q_out", "k", "k_out", "v")}, stride=1 << 31) == ok.ABQ_ERR_TOO_LARGE
    assert append(**{n: none for n in ("q", "q_out", "k", "k_out", "v")}, slots=None, positions=None) == ok.ABQ_OK


def pages(attn, **kw):
    d = dict(seqs=3, max_pages=8, page_size=16, num_pages=20, table=A, lengths=2 * A, refs=3 * A)
    d.update(kw)
    return attn.KvPagesDesc(*d.values())


def test_calls_on_pages_are_refused(attn):
    L, ok = attn.lib(), attn.abq_gemm

    def calls(**kw):
        p = ref(pages(attn, **kw))
        return {L.abq_kv_pages_fork(p, A, None), L.abq_kv_pages_extend(p, A, A, 5, A, A, A, None), L.abq_kv_pages_compact(p, A, None)}

    for kw in ({"seqs": 0}, {"max_pages": 0}, {"num_pages": 0}, {"page_size": 8}, {"page_size": 48}, {"page_size": 8192}, {"num_pages": 1 << 27}, {"table": None},
               {"lengths": None}, {"refs": None}, {"seqs": -1}):
        assert calls(**kw) == {ok.ABQ_ERR_INVALID_ARG}, kw
    for kw in ({"seqs": 8193}, {"max_pages": 1 << 27}, {"max_pages": (1 << 22) - 2}):
        assert calls(**kw) == {ok.ABQ_ERR_TOO_LARGE}, kw
    p = ref(pages(attn))
    assert L.abq_kv_pages_fork(None, A, None) == L.abq_kv_pages_fork(p, None, None) == L.abq_kv_pages_compact(p, None, None) == ok.ABQ_ERR_INVALID_ARG
    good = [A, A, 5, A, A, A]
    for i in (0, 1, 3, 4, 5):
        assert L.abq_kv_pages_extend(p, *[None if j == i else x for j, x in enumerate(good)], None) == ok.ABQ_ERR_INVALID_ARG
    assert L.abq_kv_pages_extend(p, A, A, -1, A, A, A, None) == ok.ABQ_ERR_INVALID_ARG
    assert L.abq_kv_pages_extend(p, A, A, 1 << 31, A, A, A, None) == ok.ABQ_ERR_TOO_LARGE
    assert L.abq_kv_pages_compact(ref(pages(attn, seqs=8192, max_pages=1 << 21)), A, None) == ok.ABQ_ERR_TOO_LARGE
    assert L.abq_kv_pages_compact(ref(pages(attn, num_pages=1)), None, None) == ok.ABQ_OK  # nothing can move: no launch

    def copy(c={}, bounds=None, pairs=A, count=3):
        return L.abq_kv_copy_pages(ref(cache_desc(attn, **c)), ref(bounds), pairs, count, None)
    assert copy(c={"bits": 5}) == ok.ABQ_ERR_UNSUPPORTED
    for kw in ({"c": {"k_codes": None}}, {"pairs": None}, {"count": -1}, {"bounds": attn.KvBoundsDesc(None, A)}, {"bounds": attn.KvBoundsDesc(A, None)},
               {"bounds": attn.KvBoundsDesc(A + 8, A)}, {"bounds": attn.KvBoundsDesc(A, A + 2)}):
        assert copy(**kw) == ok.ABQ_ERR_INVALID_ARG, kw
    assert copy(count=1 << 24) == ok.ABQ_ERR_TOO_LARGE and copy(count=0, pairs=None) == ok.ABQ_OK


def test_bounds_and_the_choice_are_refused(attn):
    L, ok = attn.lib(), attn.abq_gemm
    for kw, codes, scales in [({}, 10 * 2 * 256, 10 * 2 * 4), ({"head_dim": 64, "kv_heads": 7, "bits": 4}, 10 * 7 * 128, 10 * 7 * 4), ({"bits": 5}, 0, 0), ({"page_size": 20}, 0, 0),
                              ({"num_pages": 1 << 24, "kv_heads": 40}, (1 << 24) * 40 * 256, (1 << 24) * 40 * 4)]:
        d = cache_desc(attn, **kw)
        assert (L.abq_kv_bound_codes_bytes(ref(d)), L.abq_kv_bound_scales_bytes(ref(d))) == (codes, scales), kw
    assert L.abq_kv_bound_codes_bytes(None) == L.abq_kv_bound_scales_bytes(None) == 0
    good = attn.KvBoundsDesc(A, A)
    bad_bounds = [None, attn.KvBoundsDesc(None, A), attn.KvBoundsDesc(A, None), attn.KvBoundsDesc(A + 4, A), attn.KvBoundsDesc(A, A + 1)]

    def bound(c={}, bounds=good, slots=A, count=3):
        return L.abq_kv_bound(ref(cache_desc(attn, **c)), ref(bounds), slots, count, None)

    def choose(c={}, bounds=good, q={}, dtype=0, heads=2, table=A, max_pages=4, context=A, q_starts=A, seqs=2, max_q=3, max_context=100, first=1, last=1, count=3, blocks=A, workspace=None,
               bytes=0):
        return L.abq_attn_choose(ref(cache_desc(attn, **c)), ref(bounds), ref(None if q is None else rows(attn, **q)), dtype, heads, table, max_pages, context, q_starts, seqs,
                                 max_q, max_context, first, last, count, blocks, workspace, bytes, None)

    for b in bad_bounds:
        assert bound(bounds=b) == ok.ABQ_ERR_INVALID_ARG and choose(bounds=b) == ok.ABQ_ERR_INVALID_ARG
    for call in (bound, choose):
        assert call(c={"head_dim": 96}) == ok.ABQ_ERR_UNSUPPORTED and call(c={"k_scales": None}) == ok.ABQ_ERR_INVALID_ARG
    assert bound(slots=None) == bound(count=-1) == ok.ABQ_ERR_INVALID_ARG and bound(count=1 << 40) == ok.ABQ_ERR_TOO_LARGE and bound(count=0, slots=None) == ok.ABQ_OK
    for kw in [{"q": b} for b in BAD_ROWS if "rows" not in b] + [{"q": {"rows": -1}}, {"q": None}, {"dtype": 3}, {"heads": 0}, {"heads": 3}, {"table": None}, {"max_pages": 0},
                                                                 {"context": None}, {"q_starts": None}, {"seqs": 0}, {"max_q": 0}, {"first": -1}, {"last": -1}, {"count": 0},
                                                                 {"first": 2, "last": 2}, {"blocks": None}, {"first": 2 ** 31 - 1, "last": 2 ** 31 - 1}, {"max_context": -1},
                                                                 {"bytes": 8}, {"workspace": A + 2, "bytes": 8}]:
        assert choose(**kw) == ok.ABQ_ERR_INVALID_ARG, kw
    for kw in ({"max_pages": 32769}, {"count": 32769}, {"seqs": 1 << 22, "max_q": 64}, {"max_pages": 32768, "c": {"page_size": 4096, "num_pages": (1 << 19) - 1}, "seqs": 2 ** 31 - 1,
                                                                                     "max_q": 2 ** 31 - 1}):
        assert choose(**kw) == ok.ABQ_ERR_TOO_LARGE, kw
    assert choose(q={"rows": 0}, blocks=None) == ok.ABQ_OK
    need = lambda *a, **c: L.abq_attn_choose_workspace_bytes(ref(cache_desc(attn, **c)), *a)  # noqa: E731
    assert need(2000, 1, 1, 1500 * 64) == 2000 * 2 * 4 and need(2000, 1, 1, 100) == need(100, 1, 1, 10 ** 6) == need(2000, 999, 1, 10 ** 6) == 0
    assert need(2000, 999, 2, 10 ** 6) == 999 * 2 * 2 * 2000 * 4 and need(32768, 1 << 20, 64, 10 ** 6) == 0
    assert need(0, 1, 1, 10 ** 6) == need(32769, 1, 1, 10 ** 6) == need(2000, 1, 1, 10 ** 6, bits=3) == need(2000, 2 ** 31 - 1, 2 ** 31 - 1, 10 ** 6) == 0


def sparse(attn, cache={}, q={}, out={}, dtype=0, heads=2, page_table=A, max_pages=4, context=A, q_starts=A, mask=A, blocks=A, count=3, seqs=2, max_q=10, max_context=100, scale=0.1):
    st = attn.SparseState()
    return attn.lib().abq_attn_sparse_init(ref(cache_desc(attn, **cache)), ref(rows(attn, **q)), ref(rows(attn, **out)), dtype, heads, page_table, max_pages, context, q_starts,
                                           mask, blocks, count, seqs, max_q, max_context, scale, ref(st)), st


def test_attention_to_chosen_pages_is_refused(attn):
    L, ok = attn.lib(), attn.abq_gemm
    for kw in [{"dtype": 2}, {"heads": 3}, {"q_starts": None}, {"seqs": 0}, {"max_q": 0}, {"scale": 0.0}, {"page_table": None}, {"context": None}, {"max_context": -1},
               {"blocks": None}, {"count": 0}, {"cache": {"k_codes": None}}] + [{"out": b} for b in BAD_ROWS] + [{"q": b} for b in BAD_ROWS]:
        s, st = sparse(attn, **kw)
        assert s == ok.ABQ_ERR_INVALID_ARG and L.abq_attn_sparse_exec(ref(st), None) == ok.ABQ_ERR_NOT_INITIALIZED, kw
        assert L.abq_attn_sparse_workspace_bytes(ref(st)) == 0 and L.abq_attn_sparse_set_workspace(ref(st), A, 100) == ok.ABQ_ERR_NOT_INITIALIZED
    assert sparse(attn, cache={"bits": 2})[0] == ok.ABQ_ERR_UNSUPPORTED
    for kw in ({"max_q": 65}, {"count": 32769}, {"seqs": 1 << 20, "max_q": 64}):
        assert sparse(attn, **kw)[0] == ok.ABQ_ERR_TOO_LARGE, kw
    assert L.abq_attn_sparse_exec(None, None) == L.abq_attn_sparse_set_workspace(None, A, 1) == ok.ABQ_ERR_INVALID_ARG and L.abq_attn_sparse_workspace_bytes(None) == 0
    s, st = sparse(attn, count=3000, max_pages=4000, max_q=1, max_context=200000)
    assert s == ok.ABQ_OK and st.attn.parts == 1
    need = L.abq_attn_sparse_workspace_bytes(ref(st))
    assert need > 0 and L.abq_attn_sparse_set_workspace(ref(st), A + 4, need) == ok.ABQ_ERR_INVALID_ARG
    assert L.abq_attn_sparse_set_workspace(ref(st), A, need) == ok.ABQ_OK and st.attn.parts > 1 and need == st.attn.parts * 12 * 2 * 130 * 4
    # the state inside is not one of the other calls'
    assert L.abq_attn_exec(ref(st.attn), None) == L.abq_attn_set_workspace(ref(st.attn), A, need) == ok.ABQ_ERR_NOT_INITIALIZED
    assert L.abq_attn_workspace_bytes(ref(st.attn)) == 0
    s, st = sparse(attn, q={"rows": 0}, out={"rows": 0})
    assert s == ok.ABQ_OK and L.abq_attn_sparse_exec(ref(st), None) == ok.ABQ_OK
    # a short context is not split, whatever the list's length
    s, st = sparse(attn, count=3000, max_pages=4000, max_q=1, max_context=100)
    assert s == ok.ABQ_OK and L.abq_attn_sparse_workspace_bytes(ref(st)) == 0


def test_the_binding_refuses(attn):
    torch = attn.torch

    class Fake(torch.Tensor):  # a CPU tensor that says it is on the device: no launch is made
        is_cuda = True
    fake = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype).as_subclass(Fake)  # noqa: E731
    i32 = torch.int32
    for call in (lambda: attn.Rotary([0.1] * 8, device="cpu"), lambda: attn.PageTable(4, 16, 2, 3, device="cpu"), lambda: attn.KvCache(4, 16, 2, 64, device="cpu", bounds=True)):
        with pytest.raises(ValueError):
            call()
    for kw in ({"turns": [0.1] * 7}, {"turns": []}, {"turns": [[0.1] * 8]}, {"turns": [0.1] * 8, "axis": [0] * 7}, {"turns": [0.1] * 8, "axis": [-1] * 8},
               {"turns": [0.1] * 8, "axis": [2] * 8, "axes": 2}):
        with pytest.raises(ValueError):
            attn.Rotary(**kw)
    with pytest.raises(ValueError):
        attn.Rotary.of_base(128, sections=(10, 10))
    with pytest.raises(ValueError):
        attn.PageTable(4, 16, 0, 3)
    # without a device no object can be made: their checks are seen on ones put together by hand
    r = attn.Rotary.__new__(attn.Rotary)
    r.axes, r._memory = 3, attn._Memory.__new__(attn._Memory)
    for positions in (fake(3, 5), fake(2, 5, dtype=i32), fake(3, 4, dtype=i32), torch.zeros(3, 5, dtype=i32), fake(5, 3, dtype=i32).T, fake(5, dtype=i32)):
        with pytest.raises(ValueError):
            r._positions(positions, 5)
    assert r._positions(fake(3, 9, dtype=i32)[:, :5], 5)[1] == 9
    cache = attn.KvCache.__new__(attn.KvCache)
    cache._row, cache.bounds, cache._bounds = (2, 64), None, None
    cache.desc = cache_desc(attn, head_dim=64)
    k = fake(5, 2, 64)
    for q, kk, v, q_out, k_out in ((fake(4, 4, 64), k, k, None, None), (fake(5, 4, 128), k, k, None, None), (fake(5, 4, 64, dtype=torch.bfloat16), k, k, None, None),
                                   (None, k, fake(5, 3, 64), None, None), (None, fake(5, 2, 128), fake(5, 2, 128), None, None), (k, k, k, fake(5, 3, 64), None),
                                   (k, k, k, k, fake(4, 2, 64)), (None, k, k, k, None)):
        with pytest.raises(ValueError):
            cache.append_rotated(r, q, kk, v, None, None, q_out=q_out, k_out=k_out)
    for pairs in (fake(6, dtype=i32), fake(3, 3, dtype=i32)):
        with pytest.raises(ValueError):
            cache.copy_pages(pairs)
    with pytest.raises(ValueError):
        cache.bound(fake(3, dtype=i32))
    q, ints = fake(3, 4, 64), lambda *shape: fake(*shape, dtype=i32)  # noqa: E731
    with pytest.raises(ValueError):  # no bounds
        attn.SparseAttention(q, cache, ints(2, 9), ints(2), ints(3), 2, 100, 4)
    for kw in ({"count": 0}, {"count": 2, "first": 2}, {"count": 3, "last": -1}, {"count": 4, "blocks": ints(3, 2, 3)}, {"count": 4, "blocks": torch.zeros(3, 2, 4, dtype=i32)},
               {"count": 4, "out": fake(3, 4, 128)}):
        with pytest.raises(ValueError):
            attn.SparseAttention(q, cache, ints(2, 9), ints(2), ints(3), 2, 100, **dict({"blocks": ints(3, 2, 4)}, **kw))


def test_memory_of_the_objects_is_safe_on_other_streams(attn, monkeypatch):
    torch = attn.torch
    streams = StreamsOfHand(torch, monkeypatch)
    for name in ("zeros", "full"):
        monkeypatch.setattr(torch, name, lambda *a, make=getattr(torch, name), device=None, **kw: make(*a, **kw))
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    table = attn.PageTable(8, 16, 2, 3)
    table._fork = table._extend = lambda *a: streams.log.append(("run", a[-1].value)) or 0
    other, parents = streams.Stream(streams, 0x20), torch.zeros(2, dtype=torch.int32)
    streams.taken()
    table.fork(parents, stream=streams.home)
    assert streams.taken() == [("run", 0x10)]
    table.fork(parents, stream=other)
    log = streams.taken()
    assert {e[1] for e in log if e[0] == "keep"} == {t.data_ptr() for t in (table.table, table.lengths, table.refs)}
    assert [e for e in log if e[0] != "keep"] == [("wait", 0x20, 0x10), ("run", 0x20)]
    table.fork(parents, stream=0x20)
    assert streams.taken() == [("run", 0x20)]
    given = table.extend(parents, 5, stream=other)
    assert streams.taken() == [("made", 0x20), ("run", 0x20)]
    assert [tuple(t.shape) for t in (given.slots, given.starts, given.granted, given.copies)] == [(5,), (3,), (2,), (2, 2)]
    assert [t.data_ptr() for t in (given.slots, given.starts, given.granted, given.copies)] == list(given.at)
    assert table.extend(parents, 5, out=given, stream=other) is given
    with pytest.raises(ValueError):
        table.extend(parents, 6, out=given, stream=other)


def test_tensors_on_another_device_are_refused(attn, monkeypatch):
    """Every call's tensors are on the device that its stream is of; with one device nothing is looked up"""
    torch = attn.torch

    class Fake(torch.Tensor):  # a CPU tensor that says it is on a device: no launch is made
        is_cuda, on = True, 0

        def get_device(self):
            return self.on

    def fake(on, *shape, dtype=torch.int32):
        t = torch.zeros(shape, dtype=dtype).as_subclass(Fake)
        t.on = on
        return t
    StreamsOfHand(torch, monkeypatch)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    half = torch.float16

    def objects(on):
        r, t, c = (kind.__new__(kind) for kind in (attn.Rotary, attn.PageTable, attn.KvCache))
        r.turns, r.axes, t.table, t.desc = fake(on, 8, dtype=torch.float64), 1, fake(on, 2, 3), attn.KvPagesDesc(2, 3, 16, 8, None, None, None)
        c.k_codes, c.desc, c._row, c.bounds = fake(on, 1), cache_desc(attn, head_dim=64), (2, 64), True
        return r, t, c

    def calls(r, t, c, x, stream):
        """x: what each call's tensors are made by"""
        rows = lambda: x(5, 2, 64, dtype=half)  # noqa: E731
        return (lambda: r.apply(rows(), rows(), x(5), stream=stream), lambda: t.fork(x(2), stream=stream), lambda: t.extend(x(2), 4, stream=stream),
                lambda: t.compact(x(4, 2), stream=stream), lambda: c.copy_pages(x(3, 2), stream=stream), lambda: c.bound(x(3), stream=stream),
                lambda: c.append_rotated(r, rows(), rows(), rows(), x(5), x(5), q_out=rows(), stream=stream),
                lambda: attn.SparseAttention(rows(), c, x(2, 9), x(2), x(3), 2, 100, 4, out=rows(), blocks=x(5, 2, 4)))
    on_second = type("Stream", (), {"device_index": 1, "cuda_stream": 0x30})()
    for many, objects_on, x_on, stream in ((True, 1, 0, None), (True, 0, 1, None), (True, 1, 1, None), (True, 0, 0, on_second), (True, 0, 1, on_second)):
        monkeypatch.setattr(attn, "_many_devices", many)
        made = calls(*objects(objects_on), lambda *shape, **kw: fake(x_on, *shape, **kw), stream)
        for call in made[:-1] if stream else made:
            with pytest.raises(ValueError, match="another device"):
                call()
    call = attn.SparseAttention.__new__(attn.SparseAttention)
    call.out, call._choose = fake(1, 3), True
    with pytest.raises(ValueError, match="another device"):
        call.run()
    for stream, tensors in ((None, [fake(0, 1), None, fake(0, 1)]), (on_second, [fake(1, 1)]), (0x30, [fake(1, 1), fake(0, 1)])):
        attn._together(stream, *tensors)
    monkeypatch.setattr(attn, "_many_devices", False)
    attn._together(None, fake(1, 1))


def test_launches_stay_within_the_threads_that_hip_counts(attn, tmp_path):
    """Grid times workgroup of every launch below 2^32, and within what a launch may hold of LDS, at the largest sizes that are taken"""
    from decoding_launch_probe import launches
    calls = [("rotary", 2 ** 31 - 16, 8, 0, 128), ("rotary", 1 << 24, 32, 8, 128), ("rotary", 7, 1 << 20, 4, 64), ("rotary", 1 << 23, 8, 2, 256),
             ("append", 2 ** 20, 32, 8, 128), ("append", 2 ** 22, 64, 8, 64), ("append", 3, 1 << 14, 512, 128),
             ("fork", 8192, (1 << 22) - 3), ("fork", 4096, 1000), ("fork", 1, 1), ("extend", 8192, 100, 2 ** 31 - 16), ("extend", 5, 100, 4096), ("compact", 8192, 1 << 20),
             ("copy", 8, 1 << 20), ("copy", 512, (1 << 24) - 1), ("bound", 8, 2 ** 34), ("bound", 65536, 1024), ("bound", 65536, 1023), ("bound", 8, 2 ** 27), ("bound", 8, 2 ** 27 - 64), ("bound", 64, 1 << 20),
             ("choose", 8, 1 << 16, 8, 32768, 1 << 19), ("choose", 8, 1, 1, 32768, 1 << 19), ("choose", 32, 2000, 64, 500, 1 << 14), ("choose", 32, 300, 64, 1000, 16000),
             ("sparse", 8, 100000, 8, 32768, 1 << 19), ("sparse", 64, 8, 64, 300, 1 << 19), ("sparse", 8, 1, 1, 32768, 1 << 19)]
    refused = {("rotary", 2 ** 31 - 16, 8, 0, 128), ("compact", 8192, 1 << 20), ("bound", 8, 2 ** 34), ("bound", 65536, 1024), ("bound", 8, 2 ** 27), ("choose", 8, 1 << 16, 8, 32768, 1 << 19)}
    for call, r in zip(calls, launches(tmp_path, calls)):
        assert r["status"] == (attn.abq_gemm.ABQ_ERR_TOO_LARGE if call in refused else 0) and bool(r["launches"]) == (call not in refused), (call, r)
        for made in r["launches"]:
            assert made["grid"][0] * made["block"][0] < 2 ** 32 and made["grid"][1:] == made["block"][1:] == [1, 1], (call, made)
            assert made["lds"] <= 128 << 10, (call, made)
