"""Bounds of pages over their whole life: prompts that complete many pages in one call, and pages that are forked, copied, cut, filled again and
moved; and the choices that a program's steps make by them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from decoding_reference import bounds_of  # noqa: E402
from test_gpu_paged_decoding import example  # noqa: E402, F401
from test_gpu_sparse_attention import ints, keys_held, wanted  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def bounds_are(cache, pages, what):
    """The bounds of these pages are those of the keys that the cache holds there"""
    codes, scale = bounds_of(keys_held(cache))
    assert np.array_equal(cache.bound_codes.cpu().numpy()[pages], codes[pages]), what
    assert np.array_equal(cache.bound_scales.cpu().numpy()[pages], scale[pages]), what


def complete(table, lengths, size):
    """The pages of every sequence that are full, each once"""
    return sorted({int(p) for row, n in zip(table, lengths) for p in row[:n // size]})


@pytest.mark.parametrize("bits,symmetric", [(8, True), (4, False)])
@pytest.mark.parametrize("dim,kv,size,tokens", [(128, 5, 16, 1025), (64, 9, 16, 3 * 1024 + 7), (128, 1, 32, 1031), (64, 6, 32, 2047), (128, 7, 64, 1100), (64, 3, 64, 64 * 64), (128, 2, 512, 2 * 512 + 3)])
def test_prompts_that_complete_many_pages(attn, bits, symmetric, dim, kv, size, tokens):
    """More than 1024 slots: a workgroup looks through many of them, whose number need not divide theirs"""
    gen = torch.Generator().manual_seed(tokens + dim)
    pages = tokens // size + 9
    cache = attn.KvCache(pages, size, kv, dim, bits=bits, symmetric=symmetric, bounds=True)
    order, at = torch.randperm(pages, generator=gen), torch.arange(tokens)
    slots = (order[at // size] * size + at % size).to(torch.int32)
    k = (torch.randn(tokens, kv, dim, generator=gen) + torch.randn(1, kv, dim, generator=gen)).half().cuda()
    cache.append(k, k, slots.cuda())
    full = order[:tokens // size].numpy()
    rest = order[tokens // size:].numpy()
    outside = torch.tensor([-1, pages * size + size - 1, 2 ** 31 - 1], dtype=torch.int32)
    for given in (slots, slots[torch.randperm(tokens, generator=gen)], torch.cat([outside, slots])):
        cache.bound_codes.fill_(99)
        cache.bound_scales.fill_(-3)
        cache.bound(given.cuda())
        bounds_are(cache, full, (size, len(given)))
        assert (cache.bound_codes.cpu().numpy()[rest] == 99).all() and (cache.bound_scales.cpu().numpy()[rest] == -3).all()


@pytest.mark.parametrize("bits,symmetric,dim,kv,size", [(8, True, 128, 2, 16), (4, False, 64, 3, 32), (8, False, 64, 5, 16)])
def test_bounds_follow_their_pages(attn, bits, symmetric, dim, kv, size):
    """Behind every step the bounds of all complete pages are those of their keys, in every layer"""
    rng, gen = np.random.default_rng(size + dim), torch.Generator().manual_seed(dim)
    seqs, most, pool = 6, 8, 30
    pages = attn.PageTable(pool, size, seqs, most)
    layers = [attn.KvCache(pool, size, kv, dim, bits=bits, symmetric=symmetric, bounds=True) for _ in range(2)]
    seen = 0
    for step in range(40):
        kind = rng.choice(["extend", "extend", "extend", "fork", "compact"])
        if kind == "fork":
            pages.fork(ints(np.where(rng.random(seqs) < 0.5, np.arange(seqs), rng.integers(-1, seqs, seqs)).tolist()))
        elif kind == "compact":
            moves = pages.compact()
            for layer in layers:
                layer.copy_pages(moves)
        else:
            counts = [int(rng.choice([1, 3, size, size - 1, -2, -size, size + 1])) for _ in range(seqs)]
            rows = sum(max(c, 0) for c in counts)
            given = pages.extend(ints(counts), rows)
            for i, layer in enumerate(layers):
                new = torch.randn(rows, kv, dim, generator=gen).half().cuda() * (i + 1)
                layer.copy_pages(given.copies)
                layer.append(new, new, given.slots)
                layer.bound(given.slots)
        full = complete(pages.table.tolist(), pages.lengths.tolist(), size)
        seen += len(full)
        for layer in layers:
            bounds_are(layer, full, (step, kind))
    assert seen > 200


def test_bounds_at_the_end_of_a_large_cache(attn):
    """Pages whose codes begin beyond 2^32 bytes"""
    gen = torch.Generator().manual_seed(2)
    pages, size, kv, dim = 18000, 64, 32, 128  # 4.7 GB of keys
    cache = attn.KvCache(pages, size, kv, dim, bounds=True)
    order = torch.arange(17) * 37 + 17000
    at = torch.arange(17 * size)
    slots = (order[at // size] * size + at % size).to(torch.int32).cuda()
    k = torch.randn(17 * size, kv, dim, generator=gen).half().cuda()
    cache.append(k, k, slots)
    cache.bound(slots)
    near = attn.KvCache(17, size, kv, dim, bounds=True)
    near.append(k, k, torch.arange(17 * size, dtype=torch.int32).cuda())
    codes, scale = bounds_of(keys_held(near))
    assert np.array_equal(cache.bound_codes[order.cuda()].cpu().numpy(), codes) and np.array_equal(cache.bound_scales[order.cuda()].cpu().numpy(), scale)


@pytest.mark.parametrize("captured", [False, True])
def test_a_programs_steps_choose_by_what_the_cache_holds(example, captured):  # noqa: F811
    """The example's steps, forked on the way: bounds of all complete pages, and every step's choice by them, from the cache's contents"""
    gen, rng = torch.Generator(device="cuda").manual_seed(5), np.random.default_rng(5)
    hidden, heads, kv_heads, page, sequences, lengths = 512, 8, 2, 16, 5, [90, 0, 47, 16, 31]
    layer = example.DecoderAttention(hidden, heads, kv_heads, pages=1, page_size=16)
    decoder = example.PagedDecoder(layer, sequences, max_pages=9, num_pages=50, page_size=page, chosen=3)
    decoder.prompts(torch.randn(sum(lengths), hidden, generator=gen, device="cuda").half(), lengths)
    x = torch.zeros(sequences, hidden, dtype=torch.float16, device="cuda")
    parents = torch.arange(sequences, dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph()
    if captured:
        side = torch.cuda.Stream()
        before = [t.clone() for t in (decoder.pages.table, decoder.pages.lengths, decoder.pages.refs)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decoder.step(x)
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip((decoder.pages.table, decoder.pages.lengths, decoder.pages.refs), before):
            t.copy_(old)
        with torch.cuda.graph(graph):
            decoder.fork(parents)
            decoder.step(x)
    chosen = 0
    for i in range(36):
        parents.copy_(torch.from_numpy((rng.integers(0, sequences, sequences) if i % 4 == 0 else np.arange(sequences)).astype(np.int32)))
        x.copy_(torch.randn(sequences, hidden, generator=gen, device="cuda"))
        if captured:
            graph.replay()
        else:
            decoder.fork(parents)
            decoder.step(x)
        torch.cuda.synchronize()
        table, context = decoder.pages.table.cpu(), decoder.context.tolist()
        bounds_are(decoder.cache, complete(table.tolist(), context, page), i)
        blocks = decoder.call.blocks
        want = wanted(decoder.cache, decoder.q, table, context, [1] * sequences, 1, 1, 1, 3, torch.full_like(blocks, -1))
        assert np.array_equal(blocks.cpu().numpy(), want), i
        chosen += sum(c // page > 3 for c in context)
    assert chosen > 30
