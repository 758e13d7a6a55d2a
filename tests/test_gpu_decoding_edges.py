"""Calls around the quantised cache at the edges of what is documented, on the device: no drafts, one page, angles that are there already."""
import pytest

torch = pytest.importorskip("torch")

from attention_reference import check, load_abq_attention  # noqa: E402
from decoding_reference import sparse_reference  # noqa: E402
from test_gpu_attention import filled_cache, starts  # noqa: E402
from test_gpu_sparse_attention import ints, with_bounds  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def test_no_drafts(attn):
    cache = attn.KvCache(4, 16, 2, 64, bounds=True)
    q = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    for blocks in (None, torch.empty(0, 2, 3, dtype=torch.int32, device="cuda")):
        call = attn.SparseAttention(q, cache, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints([40, 0]), starts([0, 0]), 1, 40, 3, blocks=blocks)
        assert call.run().shape == (0, 4, 64)


def test_one_page(attn):
    """The last complete page, where nothing else is said"""
    gen = torch.Generator().manual_seed(21)
    context, lens = [90, 5, 16], [2, 1, 1]
    cache, table = filled_cache(attn, gen, context, lens, 2, 64, 16, 8, True, torch.float16)
    cache = with_bounds(attn, cache, table, context)
    q = torch.randn(4, 4, 64, generator=gen).half().cuda()
    call = attn.SparseAttention(q, cache, table, ints(context), starts(lens), 2, 90, 1)
    got, blocks = call.run(), call.blocks.tolist()
    assert blocks == [[[4], [4]]] * 2 + [[[-1], [-1]], [[0], [0]]]
    check(got.cpu(), *sparse_reference(q, cache, table.cpu().numpy(), context, lens, None, 64 ** -0.5, blocks), "one page")


def test_angles_on_the_device_are_copied(attn):
    turns, axis = torch.rand(8, dtype=torch.float64, device="cuda"), ints([0, 1] * 4)
    rotary = attn.Rotary(turns, axis)
    x, at = torch.randn(5, 2, 32, device="cuda").half(), torch.arange(10, dtype=torch.int32, device="cuda").view(2, 5)
    want = rotary.apply(x, None, at)[0].clone()
    turns.zero_(), axis.zero_()
    assert torch.equal(rotary.apply(x, None, at)[0], want) and not torch.equal(want, x)
