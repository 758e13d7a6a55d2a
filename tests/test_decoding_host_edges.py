"""Calls around the quantised cache at the edges of what is documented: nothing to do, one page, the caller's own tensors.  No GPU."""
import pytest

pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from test_decoding_host import ref, rotary, sparse  # noqa: E402
from test_attention_host import A, StreamsOfHand, cache_desc, rows  # noqa: E402


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def test_attention_to_chosen_pages_without_drafts(attn):
    """No rows: there is nothing to list pages for, and an empty tensor has no address"""
    L, ok = attn.lib(), attn.abq_gemm
    none = {"rows": 0, "data": None}
    s, st = sparse(attn, q=none, out=none, blocks=None)
    assert s == ok.ABQ_OK and L.abq_attn_sparse_exec(ref(st), None) == ok.ABQ_OK
    assert L.abq_attn_sparse_workspace_bytes(ref(st)) == 0 and L.abq_attn_sparse_set_workspace(ref(st), None, 0) == ok.ABQ_OK
    for kw in ({"count": 0}, {"blocks": None}, {"blocks": None, "q": {"rows": 0}}):
        assert sparse(attn, **kw)[0] == ok.ABQ_ERR_INVALID_ARG, kw
    assert sparse(attn, blocks=A)[0] == ok.ABQ_OK


def on_no_device(torch):
    class Fake(torch.Tensor):  # a CPU tensor that says it is on the device: no launch is made
        is_cuda = True
    return lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype).as_subclass(Fake)


def test_one_chosen_page(attn, monkeypatch):
    """Unless it is said otherwise one page from either end is chosen in any case, as far as there is room for it, the last one first"""
    torch = attn.torch
    StreamsOfHand(torch, monkeypatch)
    monkeypatch.setattr(attn, "_rows", lambda t: attn.Rows(t.data_ptr(), t.shape[0], t.stride(0), t.stride(1)))
    fake = on_no_device(torch)
    cache = attn.KvCache.__new__(attn.KvCache)
    cache.desc, cache._memory = cache_desc(attn, head_dim=64), attn._Memory(())
    cache.bounds, cache._bounds, cache.k_codes = True, None, fake(1)
    full = torch.full
    monkeypatch.setattr(torch, "full", lambda *a, device=None, **kw: full(*a, **kw).as_subclass(type(fake(1))))
    aligned = torch.zeros(2 * 3 * 4 * 64 + 64, dtype=torch.float16).as_subclass(type(fake(1)))
    at = -aligned.data_ptr() // 2 % 8
    q, out = (aligned[at + i * 768:at + (i + 1) * 768].view(3, 4, 64) for i in range(2))

    def forced(**kw):
        call = attn.SparseAttention(q, cache, fake(2, 9), fake(2), fake(3), 2, 100, out=out, workspace=fake(0), **kw)
        return call._chosen[-6:-4], call.blocks.shape
    assert forced(count=1) == ((0, 1), (3, 2, 1)) and forced(count=2) == ((1, 1), (3, 2, 2)) and forced(count=9) == ((1, 1), (3, 2, 9))
    assert forced(count=1, first=1)[0] == (1, 0) and forced(count=1, first=0, last=0)[0] == (0, 0) and forced(count=3, first=0)[0] == (0, 1)
    assert forced(count=3, first=3)[0] == (3, 0) and forced(count=3, last=2)[0] == (1, 2) and forced(count=3, last=3)[0] == (0, 3)
    for kw in ({"count": 1, "first": 1, "last": 1}, {"count": 2, "first": 3}, {"count": 2, "last": 3}, {"count": 3, "last": -1}, {"count": 3, "first": -1}, {"count": 0}):
        with pytest.raises(ValueError):
            forced(**kw)


def test_angles_are_the_objects_own(attn, monkeypatch):
    """Angles and axes that are on the device already, in the type that is wanted, are copied as all others are"""
    torch = attn.torch
    StreamsOfHand(torch, monkeypatch)
    moved = torch.Tensor.to

    def to(t, *a, copy=False, **kw):  # (what is here is on the device already)
        if a == ("cuda",) or str(kw.get("device")) == "cuda":
            a, kw = (), {k: v for k, v in kw.items() if k != "device"}
            return t.clone() if copy else moved(t, **kw) if kw else t
        return moved(t, *a, copy=copy, **kw)
    monkeypatch.setattr(torch.Tensor, "to", to)
    turns, axis = torch.arange(8, dtype=torch.float64), torch.tensor([0, 1] * 4, dtype=torch.int32)
    for given in (turns, turns.numpy(), torch.stack([turns, turns], 1)[:, 0]):
        r = attn.Rotary(given, axis)
        before = r.turns.clone(), r.axis.clone()
        given *= 2
        axis.mul_(0)
        assert torch.equal(r.turns, before[0]) and torch.equal(r.axis, before[1]) and r.turns.is_contiguous()
        assert (r.desc.turns, r.desc.axis) == (r.turns.data_ptr(), r.axis.data_ptr()) and r.desc.rotary_dim == 16
        given /= 2
        axis.copy_(before[1])


def test_turned_rows_that_lie_on_other_rows_are_refused(attn):
    """q_out on k, k_out on q, or both results on one place: waves would read what others have written"""
    L, ok = attn.lib(), attn.abq_gemm
    none = dict.fromkeys(("q", "q_out", "k", "k_out", "v"))
    at = {"q": 8 * A, "q_out": 12 * A, "k": 16 * A, "k_out": 20 * A, "v": 24 * A}

    def calls(count=12, **places):
        r = {n: ref(None if p is None else rows(attn, data=p, rows=count)) for n, p in dict(at, **places).items()}
        angles = ref(rotary(attn))
        apply = L.abq_rotary_apply(angles, r["q"], r["q_out"], 2, r["k"], r["k_out"], 2, 128, 0, 6 * A, 12, None) if places.get("q", A) else None
        return apply, L.abq_kv_append_rotary(ref(cache_desc(attn)), angles, r["q"], r["q_out"], 2, r["k"], r["k_out"], r["v"], 0, 6 * A, 12, 5 * A, None)
    bad = ok.ABQ_ERR_INVALID_ARG
    for places in ({"q_out": 16 * A}, {"k_out": 8 * A}, {"q_out": 20 * A}, {"q_out": 8 * A, "k_out": 8 * A}, {"q_out": 16 * A, "k_out": 8 * A}, {"q": 16 * A, "q_out": 16 * A}):
        assert calls(**places) == (bad, bad), places
    assert calls(q_out=16 * A, k_out=None)[1] == calls(q=None, q_out=None, k_out=24 * A)[1] == bad
    empty = dict.fromkeys(none, 8 * A)  # no rows: nothing lies on anything
    assert calls(count=0, **empty) == (ok.ABQ_OK, ok.ABQ_OK)


def test_rows_may_be_turned_in_place(attn, tmp_path):
    from decoding_launch_probe import launches
    for r in launches(tmp_path, [("rotary", 5, 4, 4, 128), ("rotary", 5, 4, 0, 128), ("append", 5, 4, 4, 128)]):
        assert r["status"] == 0 and len(r["launches"]) == 1
