"""Attention of drafts and to chosen pages where a wave's later tokens outweigh its earlier ones by more than it lets pass without
rescaling: what came before keeps its share, at any level of the scores"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import check, load_abq_attention  # noqa: E402
from decoding_reference import sparse_reference  # noqa: E402
from test_gpu_attention import starts, tree_reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("level", [2.0 ** -7, 1.0, 300.0])
@pytest.mark.parametrize("group", [1, 18])
def test_earlier_tokens_keep_their_share(attn, dtype, level, group):
    gen = torch.Generator().manual_seed(6)
    heads, dim, tokens, size = 60, 64, 3 * 256, 64
    # the first third of the tokens lies some powers of two below the second in every head, and that below one token in the last: all three
    # parts of a wave's have about the same weight together.  Scores, and the values' level, begin anywhere.
    jump = 5.5 + torch.rand(heads, generator=gen)
    base = (torch.rand(heads, generator=gen) - 0.5) * 40
    score = torch.empty(tokens, heads)
    score[:256], score[256:512], score[512:] = base - jump, base, base - 30
    score[512::32] = base + 5.1
    k = torch.zeros(tokens, heads, dim)
    k[:, :, 0] = score * 0.6931 / 4
    v = torch.randn(tokens, heads, dim, generator=gen) * 0.1
    v[:256] += 1
    v[256:512] -= 1
    q = torch.zeros(1, heads * group, dim)
    q[:, :, 0] = 4
    cache = attn.KvCache(tokens // size + 1, size, heads, dim, bounds=True)
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    cache.append(k.to(dtype).cuda(), (v * level).to(dtype).cuda(), slots)
    q = q.to(dtype).cuda()
    table = torch.arange(tokens // size + 1, dtype=torch.int32)[None].cuda()
    context = torch.tensor([tokens - 1], dtype=torch.int32).cuda()
    none = torch.empty(0, device="cuda")
    got = attn.TreeAttention(q, cache, table, context, starts([1]), 1, tokens, scale=1.0, workspace=none).run()
    check(got.cpu(), *tree_reference(q, cache, table, [tokens - 1], [1], None, 1.0), "drafts")
    blocks = torch.arange(tokens // size - 1, dtype=torch.int32).repeat(1, heads, 1).contiguous()
    got = attn.SparseAttention(q, cache, table, context, starts([1]), 1, tokens, blocks.shape[2], scale=1.0, workspace=none, blocks=blocks.cuda()).run()
    check(got.cpu(), *sparse_reference(q, cache, table.cpu().numpy(), [tokens - 1], [1], None, 1.0, blocks.tolist()), "chosen")
