"""Attention of whole prompts and of drafts on the quantised cache, through the C ABI, against the formulas in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import attend, cache_contents, check, load_abq_attention  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def starts(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


# ---------------------------------------------------------------------------------------------- whole prompts

def prompt_reference(q, k, v, q_lens, k_lens, scale):
    out, allowed = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group, a, b = q.shape[1] // k.shape[1], 0, 0
    for n, m in zip(q_lens, k_lens):
        visible = torch.arange(m)[None, :] <= m - n + torch.arange(n)[:, None]
        for h in range(q.shape[1]):
            out[a:a + n, h], allowed[a:a + n, h] = attend(q[a:a + n, h].cpu(), k[b:b + m, h // group].cpu(), v[b:b + m, h // group].cpu(), visible, scale, q.dtype)
        a, b = a + n, b + m
    return out, allowed


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], [1]), ([2], [2]), ([31], [31]), ([33, 1, 64], [33, 1, 64]), ([63, 65, 128], [63, 65, 128]), ([129, 0, 255], [129, 0, 255]), ([300], [300]),
    ([7, 40], [500, 130]), ([1, 1, 1], [64, 65, 1000]), ([130], [129]), ([50, 5, 3], [20, 0, 3]), ([260], [700]),
])
def test_prompts(attn, dtype, dim, q_lens, k_lens):
    gen = torch.Generator().manual_seed(sum(q_lens) + dim)
    for heads, kv_heads in [(3, 3), (4, 1)] if sum(k_lens) < 600 else [(6, 2)]:
        q = (2 * torch.randn(sum(q_lens), heads, dim, generator=gen)).to(dtype).cuda()
        k, v = ((torch.randn(sum(k_lens), kv_heads, dim, generator=gen) + 0.2).to(dtype).cuda() for _ in range(2))
        scale = 0.7 * dim ** -0.5
        out = torch.full_like(q, 77)
        got = attn.PromptAttention(q, k, v, starts(q_lens), starts(k_lens), max(q_lens), max(k_lens), scale=scale, out=out).run()
        check(got.cpu(), *prompt_reference(q, k, v, q_lens, k_lens, scale), (heads, kv_heads))
        if q_lens == k_lens:
            again = attn.PromptAttention(q, k, v, starts(q_lens), max_q=max(q_lens), scale=scale).run()
            assert torch.equal(again, got)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("heads,kv_heads,q_lens,k_lens", [(8, 8, [1100], [1100]), (2, 1, [1, 17], [4000, 2500]), (4, 2, [513, 200, 1], [513, 900, 3000])])
def test_longer_prompts(attn, workspace, heads, kv_heads, q_lens, k_lens):
    gen = torch.Generator().manual_seed(5)
    for dtype, dim in [(torch.bfloat16, 128), (torch.float16, 64)]:
        q = (3 * torch.randn(sum(q_lens), heads, dim, generator=gen)).to(dtype).cuda()
        k, v = (torch.randn(sum(k_lens), kv_heads, dim, generator=gen).to(dtype).cuda() for _ in range(2))
        call = attn.PromptAttention(q, k, v, starts(q_lens), starts(k_lens), max(q_lens), max(k_lens),
                                    workspace=None if workspace else torch.empty(0, device="cuda"))
        check(call.run().cpu(), *prompt_reference(q, k, v, q_lens, k_lens, dim ** -0.5), (dtype, dim))


def test_prompt_rows_are_slices(attn):
    gen = torch.Generator().manual_seed(6)
    lens, heads, kv_heads, dim = [45, 99], 4, 2, 128
    fused = torch.randn(sum(lens) + 2, (heads + 2 * kv_heads) * dim, generator=gen).half().cuda()[1:-1]
    q, k, v = (x.unflatten(1, (-1, dim)) for x in fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    into = torch.full((heads, sum(lens) + 2, dim + 8), 5.0, dtype=torch.float16, device="cuda")
    out = into[:, 1:-1, :dim].transpose(0, 1)
    attn.PromptAttention(q, k, v, starts(lens), max_q=max(lens), out=out).run()
    check(out.cpu(), *prompt_reference(q, k, v, lens, lens, dim ** -0.5), "slices")
    assert (into[:, 0] == 5).all() and (into[:, -1] == 5).all() and (into[:, :, dim:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_a_prompts_query_does_not_see_never_reaches_it(attn, dtype, dim, bad):
    """Keys and values that are not finite: queries in front of them, and the sequences beside them, are as without them"""
    gen = torch.Generator().manual_seed(8)
    lens, heads = [70, 200, 3], 2
    q = torch.randn(sum(lens), heads, dim, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(sum(lens), heads, dim, generator=gen).to(dtype).cuda() for _ in range(2))
    clean = attn.PromptAttention(q, k, v, starts(lens), max_q=max(lens)).run().clone()
    k2, v2 = k.clone(), v.clone()
    first = {0: 66, 1: 70 + 97, 2: 270 + 1}  # the first bad token of each sequence
    for s, at in first.items():
        v2[at, 0, 3] = bad
        k2[at, 1, dim - 1] = bad
    v2[70 + 150, 0, dim - 2] = bad
    got = attn.PromptAttention(q, k2, v2, starts(lens), max_q=max(lens)).run()
    want, allowed = prompt_reference(q, k, v, lens, lens, dim ** -0.5)
    sound = torch.ones(sum(lens), dtype=torch.bool)
    for (a, n), at in zip(((0, 70), (70, 200), (270, 3)), first.values()):
        sound[at:a + n] = False
    check(got.cpu()[sound], want[sound], allowed[sound], "in front of them")
    assert torch.isfinite(clean).all()
    # a bad value reaches its own element of the queries that see it, and no other element
    for at, end in ((66, 70), (70 + 97, 270), (271, 273)):
        assert not torch.isfinite(got[at:end, 0, 3]).any()
    other = torch.ones(dim, dtype=torch.bool)
    other[[3, dim - 2]] = False
    check(got.cpu()[:, 0, other], want[:, 0, other], allowed[:, 0, other], "other elements")


def test_prompt_offsets_that_make_no_sense_stay_inside_the_tensors(attn):
    q = torch.randn(20, 2, 64).half().cuda()
    for bad in ([0, 30, 20], [-5, 4, 20], [0, 12, 6]):
        out = attn.PromptAttention(q, q, q, torch.tensor(bad, dtype=torch.int32).cuda(), max_q=20).run()
        torch.cuda.synchronize()
        assert out.shape == q.shape


# ---------------------------------------------------------------------------------------------- drafts on the cache

def tree_reference(q, cache, table, context, lens, mask, scale):
    kc, vc, (ks, kz), (vs, vz) = cache_contents(cache)
    size, pages, group = cache.desc.page_size, cache.desc.num_pages, q.shape[1] // cache.desc.kv_heads
    half = 2 ** (cache.desc.bits - 1)
    out, allowed = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    a = 0
    for s, n in enumerate(lens):
        m = min(max(context[s], 0) + n, table.shape[1] * size)
        at = np.arange(m)
        page = table[s].cpu().numpy()[at // size]
        there = (page >= 0) & (page < pages)
        slot = np.where(there, page, 0) * size + at % size
        visible = torch.zeros((n, m), dtype=torch.bool)
        for i in range(n):
            bits = (1 << (i + 1)) - 1 if mask is None else int(mask[a + i]) % (1 << 64)
            visible[i] = torch.tensor([bool(there[t]) and (t < context[s] or bool(bits >> (t - context[s]) & 1)) for t in range(m)], dtype=torch.bool)
        for h in range(q.shape[1]):
            g = h // group
            k, v = ((c[slot, g] - z[slot, g, None].astype(np.float64)) * w[slot, g, None].astype(np.float64) for c, z, w in ((kc, kz, ks), (vc, vz, vs)))
            # the second product is of codes less half their range, and of zero points likewise
            spread = (np.abs(vc[slot, g] - half) * 2.0 ** -8 + np.abs(vz[slot, g, None] - half) * 2.0 ** -8 + np.abs(vc[slot, g] - vz[slot, g, None])) * vs[slot, g, None]
            top = vs[slot, g].max() / max(1e-30, vs[slot, g].min()) if m else 1.0
            k_spread = torch.from_numpy((np.abs(kc[slot, g] - half) + np.abs(kz[slot, g, None] - half)) * ks[slot, g, None].astype(np.float64))
            rows = q[a:a + n, h].cpu()
            out[a:a + n, h], some = attend(rows, torch.from_numpy(k), torch.from_numpy(v), visible, scale, q.dtype, torch.from_numpy(spread), top)
            # scores are taken from codes and zero points apart: errors of fp32 sums of that size
            if m:
                more = (rows.double().abs() @ k_spread.T * scale).amax(-1, keepdim=True) * (q.shape[2] + 8) * 2.0 ** -23
                some = some + more * (torch.from_numpy(spread).amax(0)[None, :])
            allowed[a:a + n, h] = some
        a += n
    return out, allowed


def filled_cache(attn, gen, context, lens, kv_heads, dim, size, bits, symmetric, dtype, extra_pages=2):
    """A cache that holds the sequences' tokens on pages in any order, garbage everywhere else"""
    need = [max(1, (c + n + size - 1) // size) for c, n in zip(context, lens)]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        for i in range(n):
            table[s, i] = order.pop()
    cache = attn.KvCache(pages, size, kv_heads, dim, bits=bits, symmetric=symmetric)
    cache.k_codes.random_(0, 256)
    cache.v_codes.random_(0, 256)
    cache.k_scales.fill_(float("nan"))
    cache.v_scales.fill_(float("nan"))
    for s, (c, n) in enumerate(zip(context, lens)):
        if c + n == 0:
            continue
        at = torch.arange(c + n)
        slots = table[s][at // size] * size + at % size
        level = torch.exp(torch.randn(c + n, 1, 1, generator=gen))
        k = torch.randn(c + n, kv_heads, dim, generator=gen) + 0.3
        v = torch.randn(c + n, kv_heads, dim, generator=gen) * level + 0.1 * level
        cache.append(k.to(dtype).cuda(), v.to(dtype).cuda(), slots.to(torch.int32).cuda())
    return cache, table.cuda()


def random_tree(rng, lens):
    masks = []
    for n in lens:
        seen = []
        for i in range(n):
            parent = int(rng.integers(-1, i)) if i else -1
            seen.append((1 << i) | (seen[parent] if parent >= 0 else 0))
        masks += seen
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,size,context,lens", [
    (2, 2, 16, [0], [1]), (4, 1, 16, [15, 16, 17], [1, 1, 1]), (3, 3, 64, [31, 32, 200], [1, 2, 3]), (8, 2, 32, [100, 0, 5], [9, 12, 1]),
    (6, 2, 16, [127], [64]), (16, 1, 128, [300, 7], [5, 7]), (2, 1, 32, [33, 50], [0, 33]),
])
def test_drafts(attn, bits, symmetric, dim, dtype, heads, kv_heads, size, context, lens):
    gen, rng = torch.Generator().manual_seed(bits * dim + sum(context)), np.random.default_rng(sum(lens) + size)
    cache, table = filled_cache(attn, gen, context, lens, kv_heads, dim, size, bits, symmetric, dtype)
    q = (2 * torch.randn(sum(lens), heads, dim, generator=gen)).to(dtype).cuda()
    ctx = torch.tensor(context, dtype=torch.int32).cuda()
    for mask in (None, random_tree(rng, lens)):
        call = attn.TreeAttention(q, cache, table, ctx, starts(lens), max(lens), max(context), mask=None if mask is None else mask.cuda(), out=torch.full_like(q, 77))
        check(call.run().cpu(), *tree_reference(q, cache, table, context, lens, mask, dim ** -0.5), (mask is None))


@pytest.mark.parametrize("bits,symmetric,dim,dtype", [(8, True, 128, torch.float16), (4, False, 128, torch.bfloat16), (8, False, 64, torch.bfloat16), (4, True, 64, torch.float16)])
@pytest.mark.parametrize("split", [True, False])
def test_long_contexts(attn, bits, symmetric, dim, dtype, split):
    gen, rng = torch.Generator().manual_seed(dim), np.random.default_rng(dim)
    context, lens = [3000, 1, 777, 1500], [1, 3, 40, 17]
    cache, table = filled_cache(attn, gen, context, lens, 2, dim, 64, bits, symmetric, dtype)
    q = (2 * torch.randn(sum(lens), 4, dim, generator=gen)).to(dtype).cuda()
    mask = random_tree(rng, lens)
    call = attn.TreeAttention(q, cache, table, torch.tensor(context, dtype=torch.int32).cuda(), starts(lens), 40, 3000, mask=mask.cuda(),
                              workspace=None if split else torch.empty(0, device="cuda"))
    assert (call.workspace_bytes > 0) and (call.state.parts > 1) == split
    want = tree_reference(q, cache, table, context, lens, mask, dim ** -0.5)
    check(call.run().cpu(), *want, split)
    if split:  # a workspace for fewer parts: the split goes by what there is
        small = torch.empty(call.workspace_bytes // call.state.parts * 2, dtype=torch.uint8, device="cuda")
        fewer = attn.TreeAttention(q, cache, table, torch.tensor(context, dtype=torch.int32).cuda(), starts(lens), 40, 3000, mask=mask.cuda(), workspace=small)
        assert fewer.state.parts == 2
        check(fewer.run().cpu(), *want, "two parts")


def test_drafts_that_see_nothing_or_little(attn):
    gen = torch.Generator().manual_seed(3)
    context, lens = [0, 40], [5, 6]
    cache, table = filled_cache(attn, gen, context, lens, 2, 128, 16, 8, True, torch.float16)
    q = torch.randn(sum(lens), 4, 128, generator=gen).half().cuda()
    mask = torch.tensor([0, 1, 0, 6, 16, 0, 32, 1, 0, 0, -1], dtype=torch.int64)  # (bits beyond the drafts stand for nothing)
    got = attn.TreeAttention(q, cache, table, torch.tensor(context, dtype=torch.int32).cuda(), starts(lens), 6, 40, mask=mask.cuda()).run()
    check(got.cpu(), *tree_reference(q, cache, table, context, lens, mask, 128 ** -0.5), "masks")
    assert (got[0] == 0).all() and (got[2] == 0).all()


def test_pages_outside_the_cache_and_lengths_beyond_the_table_are_not_seen(attn):
    gen = torch.Generator().manual_seed(12)
    context, lens = [100, 60], [2, 1]
    cache, table = filled_cache(attn, gen, context, lens, 2, 64, 16, 8, False, torch.float16)
    table[0, 2], table[0, 4], table[1, 0] = -3, cache.desc.num_pages, 1 << 30
    q = torch.randn(sum(lens), 2, 64, generator=gen).half().cuda()
    for max_context in (1, 100, 5000):  # it only guides the split
        got = attn.TreeAttention(q, cache, table, torch.tensor(context, dtype=torch.int32).cuda(), starts(lens), 2, max_context).run()
        check(got.cpu(), *tree_reference(q, cache, table, context, lens, None, 64 ** -0.5), max_context)
    wild = torch.tensor([-9, 2 ** 31 - 1], dtype=torch.int32).cuda()
    got = attn.TreeAttention(q, cache, table.clamp(0, cache.desc.num_pages - 1), wild, starts(lens), 2, 100).run()
    torch.cuda.synchronize()
    assert got.shape == q.shape


def test_values_of_very_different_scales(attn):
    """Value scales from 1e-5 to hundreds in one sequence: weights are held relative to what they weigh"""
    gen = torch.Generator().manual_seed(13)
    for level in (1e-4, 1.0, 300.0):
        cache = attn.KvCache(8, 16, 1, 128)
        slots = torch.arange(100, dtype=torch.int32).cuda()
        k = torch.randn(100, 1, 128, generator=gen).half()
        v = (torch.randn(100, 1, 128, generator=gen) * level).half()
        cache.append(k.cuda(), v.cuda(), slots)
        table, q = torch.arange(8, dtype=torch.int32).cuda()[None], torch.randn(1, 3, 128, generator=gen).half().cuda()
        got = attn.TreeAttention(q, cache, table, torch.tensor([99], dtype=torch.int32).cuda(), starts([1]), 1, 99).run()
        check(got.cpu(), *tree_reference(q, cache, table, [99], [1], None, 128 ** -0.5), level)


def test_queries_of_any_size_in_bf16(attn):
    gen = torch.Generator().manual_seed(14)
    cache, table = filled_cache(attn, gen, [70], [4], 1, 128, 16, 8, True, torch.bfloat16)
    q = torch.randn(4, 2, 128, generator=gen)
    q[0] *= 1e-20
    q[1] *= 1e20
    q[2, 0] = 0
    q = q.to(torch.bfloat16).cuda()
    for scale in (128 ** -0.5, 1e-20):
        got = attn.TreeAttention(q, cache, table, torch.tensor([70], dtype=torch.int32).cuda(), starts([4]), 4, 70, scale=scale).run()
        want, allowed = tree_reference(q, cache, table, [70], [4], None, scale)
        some = [0, 2, 3] if scale > 1e-10 else [0, 1, 2, 3]  # (with huge scores one token takes all: its weight is 1, which one it is a matter of bits)
        check(got.cpu()[some], want[some], allowed[some], scale)
        assert torch.isfinite(got).all()


def test_both_on_another_stream_and_in_a_graph(attn):
    gen = torch.Generator().manual_seed(15)
    context, lens = [900, 30], [3, 1]
    cache, table = filled_cache(attn, gen, context, lens, 2, 128, 16, 8, True, torch.float16)
    q = torch.randn(sum(lens), 4, 128, generator=gen).half().cuda()
    k = torch.randn(sum(lens), 2, 128, generator=gen).half().cuda()
    ctx = torch.tensor(context, dtype=torch.int32).cuda()
    at = torch.cat([torch.arange(c, c + n) for c, n in zip(context, lens)])
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(lens))
    slots = (table.cpu()[seq, at // 16] * 16 + at % 16).to(torch.int32).cuda()
    tree = attn.TreeAttention(q, cache, table, ctx, starts(lens), 3, 900)
    prompt = attn.PromptAttention(q, k, k, starts(lens), max_q=3)
    assert tree.state.parts > 1

    def step(stream=None):
        cache.append(k, k, slots, stream=stream)
        tree.run(stream=stream)
        prompt.run(stream=stream)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    want = tree.out.clone(), prompt.out.clone()
    torch.cuda.synchronize()
    step(stream)
    stream.synchronize()
    assert torch.equal(tree.out, want[0]) and torch.equal(prompt.out, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen).half())
        k.copy_(torch.randn(k.shape, generator=gen).half())
        ctx.copy_(torch.tensor([900 - 200 * i, 30 - i], dtype=torch.int32))
        step()
        eager = tree.out.clone(), prompt.out.clone()
        tree.out.zero_(), prompt.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tree.out, eager[0]) and torch.equal(prompt.out, eager[1])
