"""Bounds of pages, the choice of pages by them, and attention to chosen pages, through the C ABI, against the formulas."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import cache_contents, check, load_abq_attention  # noqa: E402
from decoding_reference import bounds_of, choice, sparse_reference  # noqa: E402
from test_gpu_attention import filled_cache, random_tree, starts  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def keys_held(cache):
    """[pages, kv heads, page size, dim]: the keys as the cache holds them, in fp32"""
    codes, _, (scale, zero), _ = cache_contents(cache)
    keys = (codes.astype(np.float32) - zero[..., None]) * scale[..., None]
    return keys.reshape(cache.desc.num_pages, cache.desc.page_size, cache.desc.kv_heads, -1).swapaxes(1, 2)


def with_bounds(attn, cache, table, context):
    """The same cache with the bounds of its complete pages"""
    d = cache.desc
    bound = attn.KvCache(d.num_pages, d.page_size, d.kv_heads, d.head_dim, bits=d.bits, symmetric=bool(d.symmetric), bounds=True)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        getattr(bound, name).copy_(getattr(cache, name))
    slots = [int(table[s, p]) * d.page_size + d.page_size - 1 for s, c in enumerate(context) for p in range(c // d.page_size)]
    if slots:
        bound.bound(ints(slots))
    return bound


# ---------------------------------------------------------------------------------------------- bounds

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dim,kv,size", [(128, 1, 16), (128, 5, 64), (64, 3, 32), (64, 9, 16), (128, 2, 256)])
def test_bounds_of_complete_pages(attn, bits, symmetric, dim, kv, size):
    gen = torch.Generator().manual_seed(bits + dim + size)
    pages = 7
    cache = attn.KvCache(pages, size, kv, dim, bits=bits, symmetric=symmetric, bounds=True)
    tokens = 4 * size + 5
    order = torch.randperm(pages, generator=gen)
    at = torch.arange(tokens)
    slots = (order[at // size] * size + at % size).to(torch.int32)
    k = torch.randn(tokens, kv, dim, generator=gen) * torch.exp(torch.randn(tokens, 1, 1, generator=gen)) + torch.randn(1, kv, dim, generator=gen)
    k[0], k[size] = 0, 5
    k = k.half().cuda()
    cache.append(k, k, slots.cuda())
    cache.bound_codes.fill_(99)
    cache.bound_scales.fill_(-3)
    given = torch.cat([slots[torch.randperm(tokens, generator=gen)], torch.tensor([-1, -size, pages * size + size - 1, 2 ** 31 - 1], dtype=torch.int32)])
    cache.bound(given.cuda())
    codes, scale = bounds_of(keys_held(cache))
    full = order[:4].numpy()
    assert np.array_equal(cache.bound_codes.cpu().numpy()[full], codes[full])
    assert np.array_equal(cache.bound_scales.cpu().numpy()[full], scale[full])
    rest = order[4:].numpy()
    assert (cache.bound_codes.cpu().numpy()[rest] == 99).all() and (cache.bound_scales.cpu().numpy()[rest] == -3).all()
    cache.bound(torch.empty(0, dtype=torch.int32, device="cuda"))
    # a page's tokens that arrive one by one: the last one brings the bounds
    single = attn.KvCache(pages, size, kv, dim, bits=bits, symmetric=symmetric, bounds=True)
    for i in range(size):
        assert not single.bound_scales.any()
        single.append(k[i:i + 1], k[i:i + 1], slots[i:i + 1].cuda())
        single.bound(slots[i:i + 1].cuda())
    assert torch.equal(single.bound_codes[order[0]], cache.bound_codes[order[0]]) and torch.equal(single.bound_scales[order[0]], cache.bound_scales[order[0]])


# ---------------------------------------------------------------------------------------------- choice

def chosen(attn, cache, q, table, context, lens, max_q, first, last, count, out, max_context=1 << 20, workspace=True):
    need = attn.lib().abq_attn_choose_workspace_bytes(ctypes.byref(cache.desc), table.shape[1], context.numel(), max_q, max_context) if workspace else 0
    scores = torch.full((need // 4 + 1,), -1, dtype=torch.int32, device="cuda")
    attn._check(attn.lib().abq_attn_choose(ctypes.byref(cache.desc), cache._bounds, ctypes.byref(attn._rows(q)), attn._dtype(q), q.shape[1], table.data_ptr(),
                                           table.shape[1], context.data_ptr(), lens.data_ptr(), context.numel(), max_q, max_context, first, last, count,
                                           out.data_ptr(), scores.data_ptr() if need else None, need, attn.abq_gemm._stream_ptr(None)), "abq_attn_choose")


def wanted(cache, q, table, context, lens, max_q, first, last, count, out):
    codes, scales = cache.bound_codes.cpu().numpy().astype(np.int64), cache.bound_scales.cpu().numpy()
    d, want, row = cache.desc, out.cpu().numpy().copy(), 0
    group = q.shape[1] // d.kv_heads
    for s, n in enumerate(lens):
        full = min(max(context[s], 0) // d.page_size, table.shape[1])
        for i in range(n):
            for h in range(d.kv_heads):
                if i < max_q:
                    want[row, h] = choice(q[row, h * group:(h + 1) * group].cpu(), codes[:, h], scales[:, h], table[s].tolist(), d.num_pages, full, first, last, count)
            row += 1
    return want


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,kv,size,columns,context,lens,first,last,count", [
    (128, 4, 4, 16, 20, [300], [1], 1, 1, 5), (64, 8, 2, 64, 9, [64 * 9, 64 * 4 + 1, 63], [1, 2, 3], 0, 0, 3), (128, 16, 1, 32, 40, [1200, 0, 31, 32], [3, 1, 0, 1], 2, 3, 7),
    (64, 40, 2, 16, 200, [3199, 16 * 300], [2, 1], 1, 0, 64), (128, 17, 1, 16, 700, [16 * 700], [5], 0, 2, 33), (128, 6, 3, 16, 1500, [23000, 8], [1, 64], 1, 4, 1000),
    (64, 2, 2, 16, 30, [480], [1], 5, 4, 9), (64, 1, 1, 16, 3, [48], [1], 0, 0, 1),
])
def test_the_choice(attn, dtype, dim, heads, kv, size, columns, context, lens, first, last, count):
    gen = torch.Generator().manual_seed(dim + heads + columns)
    pages = columns + 11
    cache = attn.KvCache(pages, size, kv, dim, bounds=True)
    cache.bound_codes.copy_(torch.randint(-127, 128, cache.bound_codes.shape, generator=gen))
    cache.bound_scales.copy_(torch.rand(cache.bound_scales.shape, generator=gen) * 0.3)
    # pages of the same bounds, and places outside the cache
    cache.bound_codes[1::3], cache.bound_scales[1::3] = cache.bound_codes[1], cache.bound_scales[1]
    table = torch.randint(0, pages, (len(context), columns), generator=gen).to(torch.int32)
    table[:, ::13] = torch.tensor([-1, pages, 2 ** 31 - 1, -7]).repeat(columns)[:table[:, ::13].shape[1]].to(torch.int32)
    rows = sum(lens) + 2
    q = torch.randn(rows, heads, dim, generator=gen).to(dtype)
    q[0, 0] = 0
    if rows > 4:
        q[1, -1, 3], q[2, 0, 5] = float("inf"), 1e-30
    max_q = max(1, max(lens) - 1)
    args = (q.cuda(), table.cuda(), ints(context), starts(lens), max_q, first, last, count)
    out = torch.full((rows, kv, count), 55, dtype=torch.int32, device="cuda")
    want = wanted(cache, q, table, context, lens, max_q, first, last, count, out)
    for kw in ({}, {"max_context": 0}, {"workspace": False}):
        got = out.clone()
        chosen(attn, cache, *args, got, **kw)
        assert np.array_equal(got.cpu().numpy(), want), kw


def test_the_choice_among_many_pages(attn):
    """As many as a workgroup keeps the scores of"""
    gen = torch.Generator().manual_seed(2)
    for columns, count, context in ((32768, 100, 32768 * 16), (32768, 32767, 32768 * 16), (20000, 1, 16 * 19999 + 3), (4097, 4096, 4097 * 16)):
        cache = attn.KvCache(500, 16, 1, 64, bits=4, bounds=True)
        cache.bound_codes.copy_(torch.randint(-127, 128, cache.bound_codes.shape, generator=gen))
        cache.bound_scales.copy_(torch.rand(cache.bound_scales.shape, generator=gen))
        table = torch.randint(0, 500, (1, columns), generator=gen).to(torch.int32)
        q = torch.randn(1, 3, 64, generator=gen).half()
        out = torch.full((1, 1, count), 55, dtype=torch.int32, device="cuda")
        want = wanted(cache, q, table, [context], [1], 1, 0, 1, count, out)
        for workspace in (True, False):
            got = out.clone()
            chosen(attn, cache, q.cuda(), table.cuda(), ints([context]), starts([1]), 1, 0, 1, count, got, workspace=workspace)
            assert np.array_equal(got.cpu().numpy(), want), (columns, workspace)


def test_the_bounds_promise_at_least_the_scores(attn):
    """A page's bound is not below the largest product of the query with one of its keys, but for the roundings to 8 bits: half a step of
    each factor's row, times the other's sum"""
    gen = torch.Generator().manual_seed(7)
    cache, table = filled_cache(attn, gen, [640], [0], 1, 128, 64, 8, True, torch.float16)
    cache = with_bounds(attn, cache, table, [640])
    q = torch.randn(128, generator=gen).half().float().numpy()
    keys = keys_held(cache)[table[0, :10].cpu().numpy(), 0].astype(np.float64)
    codes, scale = cache.bound_codes.cpu().numpy()[:, 0].astype(np.float64), cache.bound_scales.cpu().numpy()[:, 0]
    step = np.abs(q).max() / 127
    c = np.rint(q / step)
    for p, page in enumerate(table[0, :10].tolist()):
        bound = (np.maximum(c, 0) @ codes[page, 0] + np.minimum(c, 0) @ codes[page, 1]) * step * scale[page]
        slack = 0.5 * scale[page] * np.abs(c * step).sum() + 0.5 * step * np.abs(keys[p]).max(0).sum()
        assert (keys[p] @ q).max() <= bound + slack * 1.001


# ---------------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,size,context,lens,count", [
    (2, 2, 16, [0], [1], 3), (4, 1, 16, [15, 16, 17], [1, 1, 1], 1), (3, 3, 64, [31, 320, 200], [1, 2, 3], 2), (8, 2, 32, [100, 0, 5], [9, 12, 1], 2),
    (6, 2, 16, [127], [64], 4), (40, 2, 16, [300, 7], [5, 7], 6), (2, 1, 32, [333, 50], [0, 33], 4),
])
def test_chosen_pages(attn, bits, symmetric, dim, dtype, heads, kv_heads, size, context, lens, count):
    gen, rng = torch.Generator().manual_seed(bits * dim + sum(context)), np.random.default_rng(sum(lens) + size)
    cache, table = filled_cache(attn, gen, context, lens, kv_heads, dim, size, bits, symmetric, dtype)
    cache = with_bounds(attn, cache, table, context)
    q = (2 * torch.randn(sum(lens), heads, dim, generator=gen)).to(dtype).cuda()
    for mask in (None, random_tree(rng, lens)):
        call = attn.SparseAttention(q, cache, table, ints(context), starts(lens), max(lens), max(context), count, first=min(1, count - 1), last=1, mask=None if mask is None else mask.cuda())
        got = call.run()
        want = wanted(cache, q, table, context, lens, 64, min(1, count - 1), 1, count, torch.full_like(call.blocks, -1))
        assert np.array_equal(call.blocks.cpu().numpy(), want)
        check(got.cpu(), *sparse_reference(q, cache, table.cpu().numpy(), context, lens, mask, dim ** -0.5, want.tolist()), (heads, kv_heads))
    # lists of the caller's own: any order, entries that name no complete page, one of them more than once
    full = max(1, max(context) // size)
    blocks = torch.from_numpy(rng.integers(-2, full + 2, (sum(lens), kv_heads, 7)).astype(np.int32))
    got = attn.SparseAttention(q, cache, table, ints(context), starts(lens), max(lens), max(context), 7, blocks=blocks.cuda()).run()
    check(got.cpu(), *sparse_reference(q, cache, table.cpu().numpy(), context, lens, None, dim ** -0.5, blocks.tolist()), "lists")


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("bits,symmetric,dim,dtype,size", [(8, True, 128, torch.float16, 64), (4, False, 128, torch.bfloat16, 16), (8, False, 64, torch.bfloat16, 128)])
def test_long_contexts(attn, split, bits, symmetric, dim, dtype, size):
    gen = torch.Generator().manual_seed(17)
    context, lens, heads, kv = [9000, 4111], [1, 3], 8, 2
    cache, table = filled_cache(attn, gen, context, lens, kv, dim, size, bits, symmetric, dtype)
    cache = with_bounds(attn, cache, table, context)
    q = torch.randn(sum(lens), heads, dim, generator=gen).to(dtype).cuda()
    count = 3000 // size
    call = attn.SparseAttention(q, cache, table, ints(context), starts(lens), 3, 9000, count, first=2, last=2, workspace=None if split else torch.empty(0, device="cuda"))
    assert (call.state.attn.parts > 1) == split
    got = call.run()
    want = wanted(cache, q, table, context, lens, 3, 2, 2, count, torch.full_like(call.blocks, -1))
    assert np.array_equal(call.blocks.cpu().numpy(), want)
    check(got.cpu(), *sparse_reference(q, cache, table.cpu().numpy(), context, lens, None, dim ** -0.5, want.tolist()), "long")


def test_all_pages_chosen_is_attention_to_all(attn):
    gen = torch.Generator().manual_seed(3)
    context, lens = [500, 64], [4, 1]
    cache, table = filled_cache(attn, gen, context, lens, 2, 128, 32, 8, True, torch.float16)
    cache = with_bounds(attn, cache, table, context)
    q = torch.randn(5, 6, 128, generator=gen).half().cuda()
    tree = attn.TreeAttention(q, cache, table, ints(context), starts(lens), 4, 500).run()
    got = attn.SparseAttention(q, cache, table, ints(context), starts(lens), 4, 500, 16).run()
    blocks = [[[p for p in range(c // 32)]] * 2 for c, n in zip(context, lens) for _ in range(n)]
    want, allowed = sparse_reference(q, cache, table.cpu().numpy(), context, lens, None, 128 ** -0.5, blocks)
    check(got.cpu(), want, allowed, "chosen")
    check(tree.cpu(), want, allowed, "all")


def test_what_is_not_chosen_never_reaches_the_result(attn):
    """Pages that are not listed may hold anything"""
    gen = torch.Generator().manual_seed(9)
    context, lens = [200], [2]
    cache, table = filled_cache(attn, gen, context, lens, 2, 64, 16, 8, True, torch.float16)
    q = torch.randn(2, 2, 64, generator=gen).half().cuda()
    blocks = ints([[[1, 5], [2, -1]], [[0, 11], [7, 3]]])
    clean = attn.SparseAttention(q, cache, table, ints(context), starts(lens), 2, 200, 2, blocks=blocks).run()
    size = 16 * 64
    for page in (4, 6, 8, 9, 10):
        at = int(table[0, page])
        cache.k_scales.view(-1, 2, 16)[at] = float("nan")
        cache.v_scales.view(-1, 2, 16)[at] = float("inf")
        cache.k_codes.view(-1, 2, size)[at] = 255
    assert torch.equal(attn.SparseAttention(q, cache, table, ints(context), starts(lens), 2, 200, 2, blocks=blocks).run(), clean)


def test_rows_beyond_what_is_dealt_with_stay(attn):
    gen = torch.Generator().manual_seed(10)
    context, lens = [100, 40], [3, 1]
    cache, table = filled_cache(attn, gen, context, lens, 2, 64, 16, 8, True, torch.float16)
    cache = with_bounds(attn, cache, table, context)
    q = torch.randn(6, 4, 64, generator=gen).half().cuda()  # two rows behind the last sequence
    out = torch.full_like(q, 9)
    call = attn.SparseAttention(q, cache, table, ints(context), starts(lens), 2, 100, 3, out=out)
    call.run()
    assert (out[2] == 9).all() and (out[4:] == 9).all() and not (out[[0, 1, 3]] == 9).all(-1).any()
    assert (call.blocks[2] == -1).all() and (call.blocks[4:] == -1).all() and (call.blocks[0] >= 0).all()


def test_on_another_stream_and_in_a_graph(attn):
    gen = torch.Generator().manual_seed(15)
    context, lens, size = [900, 47], [2, 1], 16
    cache, table = filled_cache(attn, gen, context, lens, 2, 128, size, 8, True, torch.float16)
    cache = with_bounds(attn, cache, table, context)
    q = torch.randn(3, 4, 128, generator=gen).half().cuda()
    k = torch.randn(3, 2, 128, generator=gen).half().cuda()
    at = torch.cat([torch.arange(c, c + n) for c, n in zip(context, lens)])
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(lens))
    slots = (table.cpu()[seq, at // size] * size + at % size).to(torch.int32).cuda()
    ctx = ints(context)
    call = attn.SparseAttention(q, cache, table, ctx, starts(lens), 2, 900, 55)
    assert call.state.attn.parts > 1

    def step(stream=None):
        cache.append(k, k, slots, stream=stream)
        cache.bound(slots, stream=stream)
        call.run(stream=stream)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    want = call.out.clone(), call.blocks.clone()
    torch.cuda.synchronize()
    step(stream)
    stream.synchronize()
    assert torch.equal(call.out, want[0]) and torch.equal(call.blocks, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen).half())
        k.copy_(torch.randn(k.shape, generator=gen).half())
        ctx.copy_(ints([900 - 200 * i, 47 - i]))
        step()
        eager = call.out.clone(), call.blocks.clone()
        call.out.zero_(), call.blocks.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(call.out, eager[0]) and torch.equal(call.blocks, eager[1])
