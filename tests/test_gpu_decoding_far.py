"""Rotary positions, pages and attention to chosen pages where offsets are beyond 32 bits, tables are large, and launches need more LDS than
they get unasked."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import check, load_abq_attention  # noqa: E402
from decoding_reference import Pages, sparse_reference, turned  # noqa: E402
from test_gpu_attention import starts  # noqa: E402
from test_gpu_pages import ints, same  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def test_rows_far_apart(attn):
    """Rows whose distance in bytes is beyond 32 bits, and in elements too"""
    gen = torch.Generator().manual_seed(1)
    rotary = attn.Rotary.of_base(128)
    memory = torch.empty(3 * 2200000000, dtype=torch.float16, device="cuda")
    x = torch.randn(3, 2, 128, generator=gen).half()
    far = torch.as_strided(memory, (3, 2, 128), (2200000000, 136, 1))
    far.copy_(x)
    at = torch.tensor([[7, 100, 5000]], dtype=torch.int32)
    want, allowed = turned(x, at, rotary.turns.cpu(), torch.zeros(64, dtype=torch.int64), False)
    got, _ = rotary.apply(far, None, at.cuda())
    assert ((got.cpu().double() - want).abs() <= allowed).all()
    rotary.apply(far, None, at.cuda(), out=(far, None))
    assert torch.equal(far, got)


def test_a_cache_of_many_gigabytes(attn):
    """Pages at both ends of a cache whose halves are 6.5 GB each: written, bounded, chosen, read and copied like any"""
    gen = torch.Generator().manual_seed(2)
    pages, size, kv, dim, heads = 25000, 64, 32, 128, 32
    far, near = (attn.KvCache(n, size, kv, dim, bounds=True) for n in (pages, 40))
    order = torch.randperm(18, generator=gen) * 1388 + 1390  # (up to 24986)
    tokens, context = 18 * size - 20, 18 * size - 21
    k, v = (torch.randn(tokens, kv, dim, generator=gen).half().cuda() for _ in range(2))
    at = torch.arange(tokens)
    rotary = attn.Rotary.of_base(dim)
    positions = at.to(torch.int32).cuda()
    tables = []
    for cache, names in ((far, order), (near, torch.arange(18))):
        slots = (names[at // size] * size + at % size).to(torch.int32).cuda()
        cache.append_rotated(rotary, None, k, v, positions, slots)
        cache.bound(slots)
        tables.append((names.to(torch.int32)[None].cuda(), slots))
    for a, b in zip(far.read(tables[0][1]), near.read(tables[1][1])):
        assert torch.equal(a, b)
    q = torch.randn(1, heads, dim, generator=gen).half().cuda()
    results = []
    for cache, (table, _) in zip((far, near), tables):
        call = attn.SparseAttention(q, cache, table, ints([context]), starts([1]), 1, context, 5)
        results.append((call.run().clone(), call.blocks.clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    want, allowed = sparse_reference(q, near, tables[1][0].cpu().numpy(), [context], [1], None, dim ** -0.5, results[1][1].tolist())
    check(results[1][0].cpu(), want, allowed, "chosen")
    # moved to other far pages, bounds and all
    new = order + 3
    far.copy_pages(torch.stack([order, new], 1).to(torch.int32).cuda())
    moved = attn.SparseAttention(q, far, new.to(torch.int32)[None].cuda(), ints([context]), starts([1]), 1, context, 5)
    assert torch.equal(moved.run(), results[0][0]) and torch.equal(moved.blocks, results[0][1])


def test_the_largest_tables(attn):
    rng = np.random.default_rng(5)
    pages, want = attn.PageTable(30000, 16, 8192, 6), Pages(30000, 16, 8192, 6)
    for step in range(4):
        counts = rng.integers(-9, 40, 8192).tolist()
        rows = sum(max(c, 0) for c in counts)
        got, (slots, starts_, granted, copies) = pages.extend(ints(counts), rows), want.extend(counts, rows)
        assert got.slots.tolist() == slots and got.starts.tolist() == starts_ and got.granted.tolist() == granted and got.copies.tolist() == copies
        parents = rng.integers(0, 8192, 8192).tolist()
        pages.fork(ints(parents))
        want.fork(parents)
        same(pages, want, step)
    assert pages.compact().tolist() == want.compact()
    same(pages, want, "compact")


def test_many_pages_taken_away_at_once(attn):
    pages, want = attn.PageTable(4000, 16, 70, 700), Pages(4000, 16, 70, 700)
    for counts in ([900] * 60 + [0] * 10, [-899] * 30 + [-20] * 30 + [5] * 10, [2000] * 5 + [-3] * 65, [-2 ** 31] * 70):
        rows = sum(max(c, 0) for c in counts)  # (the first in two launches, the others in one)
        got, (slots, _, granted, copies) = pages.extend(ints(counts), rows), want.extend(counts, rows)
        assert got.slots.tolist() == slots and got.granted.tolist() == granted and got.copies.tolist() == copies
        same(pages, want, counts[0])
    pages.extend(ints([900] * 60 + [0] * 10), 54000), want.extend([900] * 60 + [0] * 10, 54000)
    pages.extend(ints([-500] * 20 + [700] * 20 + [0] * 30), 14000), want.extend([-500] * 20 + [700] * 20 + [0] * 30, 14000)
    same(pages, want, "two launches")


def test_counts_that_are_not_aligned(attn):
    """refs from an address that is no multiple of 16"""
    pages, want = attn.PageTable(50, 16, 4, 20), Pages(50, 16, 4, 20)
    memory = torch.zeros(51, dtype=torch.int32, device="cuda")
    pages.refs = memory[1:]
    pages.desc.refs = pages.refs.data_ptr()
    for counts in ([100, 3, 0, 17], [5, 5, 300, 5], [-60, 1, -299, 40]):
        rows = sum(max(c, 0) for c in counts)
        got, (slots, _, granted, _) = pages.extend(ints(counts), rows), want.extend(counts, rows)
        assert got.slots.tolist() == slots and got.granted.tolist() == granted
        same(pages, want, counts)
    assert memory[0] == 0


def test_the_largest_choice_in_a_graph(attn):
    gen = torch.Generator().manual_seed(3)
    columns, size = 32768, 16
    cache = attn.KvCache(600, size, 1, 64, bits=4, bounds=True)
    cache.bound_codes.copy_(torch.randint(-127, 128, cache.bound_codes.shape, generator=gen))
    cache.bound_scales.copy_(torch.rand(cache.bound_scales.shape, generator=gen))
    cache.k_codes.random_(0, 256), cache.v_codes.random_(0, 256)
    table = torch.randint(0, 600, (1, columns), generator=gen).to(torch.int32).cuda()
    q, context = torch.randn(2, 3, 64, generator=gen).half().cuda(), ints([columns * size - 40])
    for max_context in (columns * size, 0):  # scores in a launch of their own, and not
        call = attn.SparseAttention(q, cache, table, context, starts([2]), 2, max_context, 200)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.run()
        for i in range(3):
            q.copy_(torch.randn(q.shape, generator=gen))
            context.copy_(ints([columns * size - 40 - 70000 * i]))
            want = call.run().clone(), call.blocks.clone()
            call.out.zero_(), call.blocks.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(call.out, want[0]) and torch.equal(call.blocks, want[1]) and (call.blocks >= 0).all()
