"""Attention where values, scores and scales come near the ends of their types, through the C ABI: nothing overflows on the way to a
result that the type holds."""
import pytest

torch = pytest.importorskip("torch")

from attention_reference import attend, cache_contents, check, load_abq_attention  # noqa: E402
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


def equal_keys(dtype, dim, T, gen):
    """(q row, key row, scale): scores of T in powers of two"""
    q = (1 + torch.rand(dim, generator=gen)).to(dtype)
    k = (1 + torch.rand(dim, generator=gen)).to(dtype)
    scale = T / float(q.double() @ k.double()) / 1.4426950408889634
    return q, k, scale


def mean_bound(v, dtype, u_weight):
    """Mean of the first 1, 2, .. tokens' values, and what may be off it: equal weights are rounded alike (u_weight), their sum in fp32
    is off by 2^-23 a term, and the result is rounded once"""
    count = torch.arange(1, v.shape[0] + 1, dtype=torch.float64)[:, None]
    mean, size = v.double().cumsum(0) / count, v.double().abs().cumsum(0) / count
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    return mean, size * (u_weight + count * 2.0 ** -23) + mean.abs() * u * 1.01 + 2.0 ** -24


# (between them, steps of fp32 at such scores are 1, 2, 4 .. in powers of two)
LEVELS = [2.0 ** e * x for e in (18, 23, 24, 25, 26, 27, 28, 30, 33, 40) for x in (1.13, 1.71)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,tokens,m,split", [(2, 150, 150, False), (2, 150, 1500, True), (256, 150, 150, False), (2, 1, 128, False)])
def test_prompts_whose_scores_are_large_and_equal(attn, dtype, sign, heads, tokens, m, split):
    """Equal scores mean equal weights, whatever their size: every query gets the mean of the values that it sees"""
    gen = torch.Generator().manual_seed(22)
    dim = 64
    v = torch.randn(m, 1, dim, generator=gen).to(dtype)
    want, allowed = mean_bound(v[:, 0], dtype, {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype])
    for T in LEVELS:
        q, k, scale = equal_keys(dtype, dim, T, gen)
        call = attn.PromptAttention((sign * q).expand(tokens, heads, dim).contiguous().cuda(), k.expand(m, 1, dim).contiguous().cuda(), v.cuda(),
                                    starts([tokens]), starts([m]), tokens, m, scale=scale)
        assert (call.state.block_rows, call.state.parts > 1) == (128 if heads > 2 else 64, split)
        got = call.run().cpu()
        for h in (0, heads - 1):
            check(got[:, h], want[m - tokens:], allowed[m - tokens:], (T, h))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("split", [False, True])
def test_prompts_whose_scores_are_large_and_far_apart(attn, dtype, split):
    """One key ahead of the others by a quarter of its score takes all"""
    gen = torch.Generator().manual_seed(23)
    dim, tokens, m, at = 128, 30, 1000, 333
    v = torch.randn(m, 1, dim, generator=gen).to(dtype)
    for T in LEVELS:
        q, k, scale = equal_keys(dtype, dim, T, gen)
        keys = (k * (0.25 + 0.5 * torch.rand(m, 1, 1, generator=gen))).to(dtype)
        keys[at, 0] = k
        call = attn.PromptAttention(q.expand(tokens, 1, dim).contiguous().cuda(), keys.cuda(), v.cuda(), starts([tokens]), starts([m]), tokens, m, scale=scale,
                                    workspace=None if split else torch.empty(0, device="cuda"))
        assert (call.state.parts > 1) == split
        want = v[at].double().expand(tokens, 1, dim)
        u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
        check(call.run().cpu(), want, want.abs() * 2.1 * u + 2.0 ** -24, T)


def tree_of(attn, v, k, bits, symmetric, dtype):
    tokens, _, dim = v.shape
    cache = attn.KvCache((tokens + 63) // 64, 64, 1, dim, bits=bits, symmetric=symmetric)
    cache.append(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.arange(tokens, dtype=torch.int32).cuda())
    _, vc, _, (vs, vz) = cache_contents(cache)
    held = torch.from_numpy((vc[:tokens, 0] - vz[:tokens, 0, None]) * vs[:tokens, 0, None].astype("float64"))
    return cache, torch.arange((tokens + 63) // 64, dtype=torch.int32).cuda()[None], held


@pytest.mark.parametrize("bits,symmetric", [(8, True), (8, False), (4, True), (4, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,tokens", [(3, 70), (3, 1500), (40, 300)])
def test_drafts_whose_scores_are_large_and_equal(attn, bits, symmetric, dtype, heads, tokens):
    gen = torch.Generator().manual_seed(24)
    dim = 128
    v = torch.randn(tokens, 1, dim, generator=gen)
    v[:, :, 0], v[:, :, 1] = 4, -4  # (one range, so one scale and one zero point: then the weights are alike too)
    for T in LEVELS:
        q, k, scale = equal_keys(dtype, dim, T, gen)
        cache, table, held = tree_of(attn, v.clamp(-4, 4), k.expand(tokens, 1, dim), bits, symmetric, dtype)
        mean, allowed = mean_bound(held, dtype, 2.0 ** -11)
        call = attn.TreeAttention(q.expand(1, heads, dim).contiguous().cuda(), cache, table, torch.tensor([tokens - 1], dtype=torch.int32).cuda(), starts([1]), 1,
                                  tokens - 1, scale=scale)
        assert call.state.block_rows == (16 if heads <= 16 else 32) and (call.state.parts > 1 or tokens < 1000)
        check(call.run().cpu()[0], mean[-1].expand(heads, dim), allowed[-1].expand(heads, dim), T)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("size", [1e30, 1e34, 1e35])
def test_bf16_queries_near_the_types_end_on_the_cache(attn, symmetric, size):
    """Scores that fp32 holds, of queries that in units of the keys' codes it does not"""
    gen = torch.Generator().manual_seed(25)
    dim, tokens, at = 128, 100, 41
    v = torch.randn(tokens, 1, dim, generator=gen)
    keys = 0.5 * torch.rand(tokens, 1, dim, generator=gen)
    keys[at] = 0.75 + 0.25 * torch.rand(dim, generator=gen)
    keys[:, :, 0], keys[:, :, 1] = 1, 0.01
    cache, table, held = tree_of(attn, v, keys, 8, symmetric, torch.bfloat16)
    q = (size * (0.5 + 0.5 * torch.rand(1, 2, dim, generator=gen))).bfloat16()
    got = attn.TreeAttention(q.cuda(), cache, table, torch.tensor([tokens - 1], dtype=torch.int32).cuda(), starts([1]), 1, tokens - 1).run()
    want = held[at].expand(1, 2, dim)
    check(got.cpu(), want, want.abs() * 2.0 ** -8 * 1.1 + held.abs().max() * 2.0 ** -18, size)


@pytest.mark.parametrize("bits,symmetric", [(8, True), (8, False), (4, True), (4, False)])
@pytest.mark.parametrize("heads", [3, 20])
def test_value_scales_far_apart_in_one_sequence(attn, bits, symmetric, heads):
    """A token's values lie anywhere between 1e-4 and 300, some are 0, and for one query a token of small values takes nearly all.  Weights
    times value scales are held to 11 bits or to 2^-35 of the largest, whichever is more."""
    gen = torch.Generator().manual_seed(26)
    dim, tokens = 128, 700
    level = torch.exp(torch.rand(tokens, 1, 1, generator=gen) * 14.9 - 9.2)
    v = (torch.randn(tokens, 1, dim, generator=gen) * level).half()
    v[::13] = 0
    k = torch.randn(tokens, 1, dim, generator=gen).half()
    small = int(level[1:].flatten().argmin()) + 1
    v[small] = (torch.randn(1, dim, generator=gen) * 1e-3).half()
    q = torch.randn(1, heads, dim, generator=gen).half()
    q[0, 0] = k[small, 0] * 1.5  # (about 17 ahead of the others' scores)
    cache, table, held = tree_of(attn, v, k, bits, symmetric, torch.float16)
    got = attn.TreeAttention(q.cuda(), cache, table, torch.tensor([tokens - 1], dtype=torch.int32).cuda(), starts([1]), 1, tokens - 1).run().cpu()
    kc, vc, (ks, kz), (vs, vz) = cache_contents(cache)
    half = 2 ** (bits - 1)
    codes = lambda c, z: torch.from_numpy(abs(c[:tokens, 0] - half) * 1.0 + abs(z[:tokens, 0, None] - half) * 1.0)  # noqa: E731
    keys = torch.from_numpy((kc[:tokens, 0] - kz[:tokens, 0, None]) * ks[:tokens, 0, None].astype("float64"))
    scale, seen = dim ** -0.5, torch.ones(1, tokens, dtype=torch.bool)
    step = torch.from_numpy(vs[:tokens, 0].astype("float64"))
    spread = codes(vc, vz) * 2.0 ** -8 * step[:, None] + held.abs()
    for h in range(heads):
        out, allowed = attend(q[0, h][None], keys, held, seen, scale, torch.float16, spread, 0.0)
        p = torch.softmax(q[0, h].double() @ keys.T * scale, 0)
        more = q[0, h].double().abs() @ (codes(kc, kz) * torch.from_numpy(ks[:tokens, 0, None].astype("float64"))).T * scale
        allowed = allowed + 2.0 ** -35 * (p * step).max() * codes(vc, vz).sum(0) + float(more.max()) * (dim + 8) * 2.0 ** -23 * (p @ spread)
        check(got[0, h][None], out, allowed, h)
        assert (allowed < out.abs().max() * 0.05).all()  # (the bound says something)


def held_mean(got, value, u, tokens, what):
    """Every token holds the value: so does every result, but for weights rounded on one side of the quotient (u), the sums' fp32 and
    one rounding"""
    assert torch.isfinite(got).all(), ("not finite", what)
    assert ((got.double() - value).abs() <= abs(value) * (2.02 * u + tokens * 2.0 ** -23)).all(), what


@pytest.mark.parametrize("dtype,u", [(torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,lens,k_lens,split", [(4, [200, 64], [200, 64], False), (256, [200], [200], False), (4, [200], [1500], True)])
def test_means_of_the_types_largest_value_in_prompts(attn, dtype, u, dim, heads, lens, k_lens, split):
    gen = torch.Generator().manual_seed(27)
    largest = torch.finfo(dtype).max
    for spread in (1, 3, 5):  # (a few tokens of about the same weight, many, and one)
        q = (spread * torch.randn(sum(lens), heads, dim, generator=gen)).to(dtype).cuda()
        k = torch.randn(sum(k_lens), 2, dim, generator=gen).to(dtype).cuda()
        v = torch.full((sum(k_lens), 2, dim), largest, dtype=dtype)
        v[:, :, 1::2] *= -1
        v[:, :, 2::4] = 1
        call = attn.PromptAttention(q, k, v.cuda(), starts(lens), starts(k_lens), max(lens), max(k_lens))
        assert (call.state.parts > 1) == split
        got = call.run().cpu()
        for at, value in ((slice(0, None, 4), largest), (slice(1, None, 2), -largest), (slice(2, None, 4), 1.0)):
            held_mean(got[:, :, at], value, u, max(k_lens), (spread, value))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("context,group,drafts,split", [(30, 8, 64, False), (6000, 8, 64, False), (6000, 8, 64, True), (6000, 16, 1, False)])
def test_means_of_the_types_largest_value_in_drafts(attn, bits, symmetric, context, group, drafts, split):
    gen = torch.Generator().manual_seed(28)
    dim, seqs = 128, 2 if drafts > 1 else 40
    size = (context + drafts + 63) // 64
    cache = attn.KvCache(seqs * size, 64, 1, dim, bits=bits, symmetric=symmetric)
    tokens = seqs * size * 64
    k = torch.randn(tokens, 1, dim, generator=gen).half().cuda()
    v = torch.full((tokens, 1, dim), 65504.0).half()
    if symmetric:
        v[:, :, 1::2] *= -1
    else:
        v[:, :, 1::2] = 0  # (a zero point of 0: with one of its own the smallest code would stand for less than the type holds)
    cache.append(k, v.cuda(), torch.arange(tokens, dtype=torch.int32).cuda())
    table = torch.arange(seqs * size, dtype=torch.int32).cuda().view(seqs, size)
    for spread in (1, 4, 6, 8):
        q = (spread * torch.randn(seqs * drafts, group, dim, generator=gen)).half().cuda()
        call = attn.TreeAttention(q, cache, table, torch.full((seqs,), context, dtype=torch.int32).cuda(), starts([drafts] * seqs), drafts, context,
                                  workspace=None if split else torch.empty(0, device="cuda"))
        assert (call.state.parts > 1) == split
        got = call.run().cpu()
        held_mean(got[:, :, 0::2], 65504.0, 2.0 ** -11, context + drafts, spread)
        if symmetric:
            held_mean(got[:, :, 1::2], -65504.0, 2.0 ** -11, context + drafts, -spread)
        else:
            assert (got[:, :, 1::2].abs() <= 65504 * 0.01).all()
