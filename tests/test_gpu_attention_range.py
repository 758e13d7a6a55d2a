"""Attention where values, scores and scales come near the ends of their types, through the C ABI: nothing overflows on the way to a
result that the type holds."""
import pytest

torch = pytest.importorskip("torch")

from attention_reference import check, load_abq_attention  # noqa: E402
from test_gpu_attention import prompt_reference, starts  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


@pytest.mark.parametrize("lens,k_lens,heads,block,split", [([70, 1, 200], [70, 1, 200], 2, 64, False), ([40], [1500], 2, 64, True), ([200] * 4, [200] * 4, 64, 128, False)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("top", [1e33, 1e37, 3e38])
def test_values_of_any_size_in_bf16(attn, top, dim, lens, k_lens, heads, block, split):
    """The sums of weights times values stay below the largest value: it is a mean of them"""
    gen = torch.Generator().manual_seed(21)
    q = torch.randn(sum(lens), heads, dim, generator=gen).bfloat16()
    k = torch.randn(sum(k_lens), 2, dim, generator=gen).bfloat16()
    k[:, 1] = 0  # (all weights alike)
    unit = (torch.rand(sum(k_lens), 2, dim, generator=gen) * 2 - 1).sign() * (0.5 + 0.5 * torch.rand(sum(k_lens), 2, dim, generator=gen))
    unit[:, :, 0] = 1  # (a mean as large as they are)
    v = (unit * top).bfloat16()
    call = attn.PromptAttention(q.cuda(), k.cuda(), v.cuda(), starts(lens), starts(k_lens), max(lens), max(k_lens))
    assert call.state.block_rows == block and (call.state.parts > 1) == split
    some = [0, heads // 2 - 1, heads // 2, heads - 1]  # heads of either key head
    got = call.run().cpu()[:, some]
    # the reference on values of ordinary size: a power of two changes no digit
    down = 2.0 ** -100
    want, allowed = prompt_reference(q[:, some], k, (v.double() * down).float(), lens, k_lens, dim ** -0.5)
    check((got.double() * down).float(), want, allowed, top)
