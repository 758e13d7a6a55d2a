"""Attention on a stream that is busy, with memory that the binding made on another one."""
import pytest

torch = pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from test_gpu_attention import filled_cache, starts  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def busy(stream):
    """Some milliseconds of work"""
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x = torch.eye(4096, device="cuda")
        for _ in range(10):
            x = x @ x


def fill_what_is_free(sizes):
    """Tensors of the current stream that take the blocks that were given back there, filled at once"""
    return [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]


def test_a_workspace_outlives_its_object_on_another_stream(attn):
    gen = torch.Generator().manual_seed(41)
    q = torch.randn(3, 4, 128, generator=gen).half().cuda()
    k, v = (torch.randn(3000, 2, 128, generator=gen).half().cuda() for _ in range(2))
    at = [starts([3]), starts([3000])]
    keep = attn.PromptAttention(q, k, v, *at, 3, 3000)
    want, need = keep.run().clone(), keep.workspace_bytes
    cache, table = filled_cache(attn, gen, [2000], [3], 2, 128, 64, 8, True, torch.float16)
    context = torch.tensor([2000], dtype=torch.int32).cuda()
    tree = attn.TreeAttention(q, cache, table, context, at[0], 3, 2000)
    tree_want, tree_need = tree.run().clone(), tree.workspace_bytes
    assert keep.state.parts > 1 and tree.state.parts > 1
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for how in (stream, stream.cuda_stream, None):
        busy(stream)
        with torch.cuda.stream(stream if how is None else None):
            got = attn.PromptAttention(q, k, v, *at, 3, 3000).run(stream=how)
            tree_got = attn.TreeAttention(q, cache, table, context, at[0], 3, 2000).run(stream=how)
        filled = fill_what_is_free([need, tree_need])
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(tree_got, tree_want), how
        assert all((t == 255).all() for t in filled), how


def test_a_cache_that_was_just_made_is_written_on_another_stream(attn):
    """Its zeros come before what is written, whichever stream is slower"""
    gen = torch.Generator().manual_seed(42)
    k = torch.randn(100, 2, 128, generator=gen).half().cuda()
    slots = torch.arange(100, dtype=torch.int32).cuda()
    first = attn.KvCache(2, 64, 2, 128)
    first.append(k, k, slots)
    want = [t.clone() for t in first.read(slots)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    busy(torch.cuda.current_stream())
    cache = attn.KvCache(2, 64, 2, 128)
    cache.append(k, k, slots, stream=stream)
    got = cache.read(slots, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
