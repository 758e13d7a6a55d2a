"""Attention in blocks of 128 queries, values that are not finite in every kind of block, bounds on queries, and offsets that point
anywhere, through the C ABI."""
import pytest

torch = pytest.importorskip("torch")

from attention_reference import check, load_abq_attention  # noqa: E402
from test_gpu_attention import filled_cache, prompt_reference, starts, tree_reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def some_heads(heads, kv_heads):
    """The first and the last head of every key head"""
    group = heads // kv_heads
    return [h for g in range(kv_heads) for h in (g * group, g * group + group - 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_lens,k_lens", [
    (64, 2, [1, 300, 129, 64, 31, 0, 128, 200], [1, 300, 129, 64, 31, 0, 128, 200]),
    (512, 2, [7, 100], [500, 131]), (171, 3, [384], [384]), (64, 4, [130, 1, 60, 256], [129, 700, 3, 321]),
])
def test_prompts_in_blocks_of_128(attn, dtype, dim, heads, kv_heads, q_lens, k_lens):
    gen = torch.Generator().manual_seed(31)
    q = (2 * torch.randn(sum(q_lens), heads, dim, generator=gen)).to(dtype).cuda()
    k, v = ((torch.randn(sum(k_lens), kv_heads, dim, generator=gen) + 0.2).to(dtype).cuda() for _ in range(2))
    call = attn.PromptAttention(q, k, v, starts(q_lens), starts(k_lens), max(q_lens), max(k_lens), out=torch.full_like(q, 77))
    assert call.state.block_rows == 128 and call.state.parts == 1
    got, some = call.run().clone(), some_heads(heads, kv_heads)
    check(got[:, some].cpu(), *prompt_reference(q[:, some], k, v, q_lens, k_lens, dim ** -0.5), (heads, kv_heads))
    for _ in range(3):
        assert torch.equal(call.run(), got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads,lens,ahead,block,split", [(128, [70, 200, 3], 0, 128, False), (2, [70, 130], 3000, 64, True)])
def test_values_that_are_not_finite_stay_where_they_are_seen(attn, dtype, dim, bad, heads, lens, ahead, block, split):
    """In blocks of 128 queries, and where the keys are split over workgroups: a value that is not finite reaches its own element of
    the queries that see it, and nothing else"""
    gen = torch.Generator().manual_seed(32)
    k_lens = [ahead + n for n in lens]
    q = torch.randn(sum(lens), heads, dim, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(sum(k_lens), 2, dim, generator=gen).to(dtype).cuda() for _ in range(2))
    v2, k2 = v.clone(), k.clone()
    seen_from = torch.zeros(sum(lens), 2, dtype=torch.bool)  # which queries see a bad value of element 3, dim - 2
    a = b = 0
    for n in lens:
        for j, (place, element) in enumerate(((n * 2 // 3, 3), (n * 3 // 4, dim - 2))):  # (places among the sequence's last tokens)
            v2[b + ahead + place, 0, element] = bad
            seen_from[a + place:a + n, j] = True
        k2[b + ahead + n * 2 // 3, 1, dim - 1] = bad
        a, b = a + n, b + ahead + n
    call = attn.PromptAttention(q, k2, v2, starts(lens), starts(k_lens), max(lens), max(k_lens))
    assert call.state.block_rows == block and (call.state.parts > 1) == split
    got = call.run().cpu()
    some = some_heads(heads, 2)
    want, allowed = prompt_reference(q[:, some], k, v, lens, k_lens, dim ** -0.5)
    got = got[:, some]
    for j, element in enumerate((3, dim - 2)):
        seen = seen_from[:, j]
        assert not torch.isfinite(got[seen][:, :2, element]).any()
        check(got[~seen][:, :2, element], want[~seen][:, :2, element], allowed[~seen][:, :2, element], element)
    other = torch.ones(dim, dtype=torch.bool)
    other[[3, dim - 2]] = False
    check(got[:, :2, other], want[:, :2, other], allowed[:, :2, other], "other elements")
    before = ~seen_from[:, 0]  # a bad key reaches the queries that see it
    check(got[before][:, 2:], want[before][:, 2:], allowed[before][:, 2:], "in front of the keys")


@pytest.mark.parametrize("heads,dim,block,split", [(2, 128, 64, False), (2, 64, 64, True), (256, 64, 128, False)])
def test_queries_beyond_the_bound_are_left_alone(attn, heads, dim, block, split):
    gen = torch.Generator().manual_seed(33)
    lens, most = [100, 70, 190], 70
    k_lens = [n + (1000 if split else 5) for n in lens]
    q = torch.randn(sum(lens), heads, dim, generator=gen).half().cuda()
    k, v = (torch.randn(sum(k_lens), 2, dim, generator=gen).half().cuda() for _ in range(2))
    call = attn.PromptAttention(q, k, v, starts(lens), starts(k_lens), most, max(k_lens), out=torch.full_like(q, 77))
    assert call.state.block_rows == block and (call.state.parts > 1) == split
    some = some_heads(heads, 2)
    got = call.run()[:, some].cpu()
    want, allowed = prompt_reference(q[:, some], k, v, lens, k_lens, dim ** -0.5)
    inside = torch.cat([torch.arange(n) < most for n in lens])
    check(got[inside], want[inside], allowed[inside], "inside")
    assert (got[~inside] == 77).all()


@pytest.mark.parametrize("context,split", [(40, False), (2000, True)])
@pytest.mark.parametrize("heads,most", [(4, 3), (8, 5)])
def test_drafts_beyond_the_bound_are_left_alone(attn, heads, most, context, split):
    """They stand in the cache all the same, and a draft that names one sees it"""
    gen = torch.Generator().manual_seed(34)
    lens, contexts = [9, 2, 30], [context, context // 2, 7]
    cache, table = filled_cache(attn, gen, contexts, lens, 1, 128, 16, 8, True, torch.float16)
    q = torch.randn(sum(lens), heads, 128, generator=gen).half().cuda()
    mask = torch.full((sum(lens),), 0x2AAAAAAA | 1, dtype=torch.int64)
    call = attn.TreeAttention(q, cache, table, torch.tensor(contexts, dtype=torch.int32).cuda(), starts(lens), most, max(contexts), mask=mask.cuda(),
                              out=torch.full_like(q, 77))
    assert (call.state.parts > 1) == split
    got = call.run().cpu()
    want, allowed = tree_reference(q, cache, table, contexts, lens, mask, 128 ** -0.5)
    inside = torch.cat([torch.arange(n) < most for n in lens])
    check(got[inside], want[inside], allowed[inside], "inside")
    assert (got[~inside] == 77).all()


@pytest.mark.parametrize("heads", [2, 256])
def test_offsets_that_make_no_sense_touch_nothing_else(attn, heads):
    """Starts that fall, are negative or lie beyond the rows: what stands around the tensors stays"""
    gen = torch.Generator().manual_seed(35)
    dim, rows, edge = 64, 40, 9
    around = [torch.full((rows + 2 * edge, h + 2, dim), 5.0).half().cuda() for h in (heads, 2, 2, heads)]
    q, k, v, out = (t[edge:-edge, 1:-1] for t in around)
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=gen))
    cache, table = filled_cache(attn, gen, [20, 3], [4, 4], 2, dim, 16, 8, True, torch.float16)
    for bad in ([0, 60, 40], [-5, 4, 40], [0, 24, 6], [2 ** 31 - 1, -2 ** 31, 40], [30, 10, 2 ** 31 - 1]):
        at = torch.tensor(bad, dtype=torch.int32).cuda()
        attn.PromptAttention(q, k, v, at, max_q=rows, out=out).run()
        attn.PromptAttention(q, k, v, at, starts([20, 20]), rows, rows, out=out).run()
        attn.TreeAttention(q, cache, table, torch.tensor([20, 3], dtype=torch.int32).cuda(), at, 30, 20, out=out).run()
        torch.cuda.synchronize()
    for t, inner in zip(around, (q, k, v, out)):
        edges = torch.ones(t.shape, dtype=torch.bool, device="cuda")
        edges[edge:-edge, 1:-1] = False
        assert (t[edges] == 5).all()
