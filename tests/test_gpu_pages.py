"""Tables of pages on the device, through the C ABI, against the rules followed sequence by sequence, and what the pages hold."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from decoding_reference import Pages  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def same(pages, want, what):
    assert pages.table.tolist() == want.table(), what
    assert pages.lengths.tolist() == want.lengths, what
    assert pages.refs.tolist() == want.refs, what


@pytest.mark.parametrize("num_pages,size,seqs,most,steps", [(40, 16, 5, 9, 40), (7, 32, 3, 4, 40), (1, 16, 1, 1, 10), (300, 16, 70, 30, 25), (5000, 16, 1100, 8, 8),
                                                            (9000, 64, 20, 600, 10), (12, 4096, 3, 5, 20)])
def test_tables_follow_the_rules(attn, num_pages, size, seqs, most, steps):
    rng = np.random.default_rng(num_pages + seqs)
    pages, want = attn.PageTable(num_pages, size, seqs, most), Pages(num_pages, size, seqs, most)
    for step in range(steps):
        kind = rng.choice(["extend", "extend", "one", "fork", "compact"])
        if kind in ("extend", "one"):
            if kind == "one":
                counts = [1] * seqs
            else:
                counts = (rng.integers(-2, 3, seqs) * rng.integers(0, max(2, num_pages * size // seqs // 2), seqs) // 2).tolist()
            rows = max(0, sum(max(c, 0) for c in counts) + int(rng.integers(-3, 4)))
            got = pages.extend(ints(counts), rows)
            slots, starts, granted, copies = want.extend(counts, rows)
            assert got.slots.tolist() == slots and got.starts.tolist() == starts, (step, counts)
            assert got.granted.tolist() == granted and got.copies.tolist() == copies, (step, counts)
        elif kind == "fork":
            parents = rng.integers(-1, seqs + 1, seqs) if rng.random() < 0.3 else np.where(rng.random(seqs) < 0.5, np.arange(seqs), rng.integers(0, seqs, seqs))
            pages.fork(ints(parents.tolist()))
            want.fork(parents.tolist())
        else:
            assert pages.compact().tolist() == want.compact(), step
            live = [p for p, n in enumerate(want.refs) if n]
            assert live == list(range(len(live)))
        same(pages, want, (step, kind))


def test_a_sequence_that_gets_only_some_of_its_pages_gives_them_back(attn):
    pages, want = attn.PageTable(10, 16, 4, 10), Pages(10, 16, 4, 10)
    for counts in ([20, 16 * 6, 0, 0], [100, 5, 16, 1], [0, 0, 0, 1], [1, 1, 1, 1]):  # (the second: four pages too few by three)
        got = pages.extend(ints(counts), sum(counts))
        slots, starts, granted, copies = want.extend(counts, sum(counts))
        assert (got.slots.tolist(), got.granted.tolist()) == (slots, granted)
        same(pages, want, counts)
    # the same for one whose first page would be a copy
    pages, want = attn.PageTable(4, 16, 2, 4), Pages(4, 16, 2, 4)
    for t in (pages, want):
        t.extend(ints([20, 0]) if t is pages else [20, 0], 20)
        t.fork(ints([0, 0]) if t is pages else [0, 0])
    got, (slots, _, granted, copies) = pages.extend(ints([0, 60]), 60), want.extend([0, 60], 60)
    assert granted == [0, 0] and (got.slots.tolist(), got.granted.tolist(), got.copies.tolist()) == (slots, granted, copies)
    same(pages, want, "copy")
    got, (slots, _, granted, copies) = pages.extend(ints([3, 28]), 31), want.extend([3, 28], 31)
    assert granted == [3, 0] and (got.slots.tolist(), got.granted.tolist(), got.copies.tolist()) == (slots, granted, copies)
    same(pages, want, "one of two")


def test_counts_and_lengths_of_any_size(attn):
    top = 2 ** 31 - 1
    pages, want = attn.PageTable(6, 16, 3, 5), Pages(6, 16, 3, 5)
    for counts in ([17, 33, 2], [top, -top - 1, 5], [-1, top, top], [-7, 1, top]):
        got = pages.extend(ints(counts), 40)
        slots, starts, granted, copies = want.extend(counts, 40) if sum(max(c, 0) for c in counts) < 1000 else (None,) + short(want, counts)
        assert got.starts.tolist() == [min(x, top) for x in starts] and got.granted.tolist() == granted and got.copies.tolist() == copies
        same(pages, want, counts)


def short(want, counts):
    """want.extend without the slots of tokens that are too many to be there"""
    cut = [min(c, 10000) for c in counts]
    _, _, granted, copies = want.extend(cut, 0)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + max(c, 0))
    return starts, granted, copies


def test_whatever_the_arrays_hold_the_calls_keep_to_them(attn):
    """Entries, counts and lengths that no call leaves: nothing outside the arrays is read or written"""
    gen = torch.Generator().manual_seed(1)
    guard = [torch.full((n + 64,), 77, dtype=torch.int32, device="cuda") for n in (30, 5, 20)]
    pages = attn.PageTable(20, 16, 5, 6)
    inner = [g[32:-32] for g in guard]
    pages.desc.table, pages.desc.lengths, pages.desc.refs = (t.data_ptr() for t in inner)
    wild = lambda n: torch.randint(-2 ** 31, 2 ** 31, (n,), generator=gen, dtype=torch.int64).to(torch.int32)  # noqa: E731
    for i in range(6):
        for t, n in zip(inner, (30, 5, 20)):
            t.copy_(wild(n) if i % 2 else wild(n) % 40 - 5)
        pages.extend(wild(5).cuda(), 50)
        pages.fork((wild(5) % 9).cuda())
        pages.compact()
        torch.cuda.synchronize()
        assert all((g[:32] == 77).all() and (g[-32:] == 77).all() for g in guard)


@pytest.mark.parametrize("bits,symmetric,dim,kv,size", [(8, True, 128, 2, 16), (4, False, 64, 3, 32), (8, False, 64, 1, 64), (4, True, 128, 5, 16)])
def test_sequences_keep_their_tokens(attn, bits, symmetric, dim, kv, size):
    """Forked, extended, cut and moved, every sequence reads back what it was given: rows whose numbers the cache holds exactly"""
    rng, gen = np.random.default_rng(size + dim), torch.Generator().manual_seed(dim)
    seqs, most, pool = 6, 8, 26
    pages = attn.PageTable(pool, size, seqs, most)
    layers = [attn.KvCache(pool, size, kv, dim, bits=bits, symmetric=symmetric, bounds=i == 0) for i in range(2)]
    held = [[] for _ in range(seqs)]
    for step in range(30):
        kind = rng.choice(["extend", "extend", "extend", "fork", "compact"])
        if kind == "fork":
            parents = np.where(rng.random(seqs) < 0.4, np.arange(seqs), rng.integers(-1, seqs, seqs)).tolist()
            pages.fork(ints(parents))
            held = [list(held[p]) if p >= 0 else [] for p in parents]
        elif kind == "compact":
            moves = pages.compact()
            for layer in layers:
                layer.copy_pages(moves)
        else:
            counts = [int(rng.choice([1, 1, 3, size, -2, -size, 2 * size + 1])) for _ in range(seqs)]
            rows = sum(max(c, 0) for c in counts)
            given = pages.extend(ints(counts), rows)
            new = torch.randn(rows, kv, dim, generator=gen).half().cuda()
            for layer in layers:
                layer.copy_pages(given.copies)
                layer.append(new, -new, given.slots)
            at = 0
            for s, (c, g) in enumerate(zip(counts, given.granted.tolist())):
                held[s] = held[s][:len(held[s]) + g] if g < 0 else held[s] + list(new[at:at + g])
                at += max(c, 0)
        table, lengths = pages.table.cpu(), pages.lengths.tolist()
        assert lengths == [len(h) for h in held], step
        for s in range(seqs):
            if not held[s]:
                continue
            t = torch.arange(lengths[s])
            slots = (table[s][t // size] * size + t % size).to(torch.int32).cuda()
            want = torch.stack(held[s])
            fresh = attn.KvCache(lengths[s] // size + 1, size, kv, dim, bits=bits, symmetric=symmetric)
            flat = t.to(torch.int32).cuda()
            fresh.append(want, -want, flat)
            for layer in layers:
                for a, b in zip(layer.read(slots), fresh.read(flat)):
                    assert torch.equal(a, b), (step, kind, s)


def test_copied_pages_are_whole_and_others_untouched(attn):
    cache = attn.KvCache(9, 16, 3, 64, bits=4, symmetric=False, bounds=True)
    parts = [(t, t.view(9, -1)) for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.bound_codes, cache.bound_scales)]
    for t, _ in parts:
        t.copy_(torch.randint(-100, 100, t.shape).to(t.dtype)) if t.dtype != torch.float32 else t.copy_(torch.rand(t.shape))
    before = [v.clone() for _, v in parts]
    pairs = [(1, 7), (-1, -1), (3, 3), (2, 8), (0, 9), (-5, 4), (2, 5), (100, 6), (6, -1)]
    cache.copy_pages(ints(pairs))
    for (_, v), old in zip(parts, before):
        want = old.clone()
        for a, b in ((1, 7), (2, 8), (2, 5)):
            want[b] = old[a]
        assert torch.equal(v, want)
    cache.copy_pages(torch.empty((0, 2), dtype=torch.int32, device="cuda"))


def test_a_captured_step_follows_the_tables(attn):
    rng = np.random.default_rng(4)
    pages, want = attn.PageTable(60, 16, 8, 12), Pages(60, 16, 8, 12)
    pages.extend(ints([30] * 8), 240)
    want.extend([30] * 8, 240)
    parents, counts = ints(list(range(8))), ints([1] * 8)
    out = pages.extend(ints([0] * 8), 16)
    moves = pages.compact()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.fork(parents)
        pages.extend(counts, 16, out=out)
        pages.compact(out=moves)
    same(pages, want, "captured, not run")
    for _ in range(6):
        p, c = rng.integers(0, 8, 8).tolist(), rng.integers(-3, 3, 8).tolist()
        parents.copy_(ints(p))
        counts.copy_(ints(c))
        graph.replay()
        torch.cuda.synchronize()
        want.fork(p)
        slots, starts, granted, copies = want.extend(c, 16)
        expected = want.compact()
        assert out.slots.tolist() == slots and out.starts.tolist() == starts and out.granted.tolist() == granted and out.copies.tolist() == copies
        assert moves.tolist() == expected
        same(pages, want, "replayed")
