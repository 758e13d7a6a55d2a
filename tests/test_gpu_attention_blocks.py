"""Attention in every kind of block of queries: bounds on queries that a block reaches beyond, through the C ABI."""
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
