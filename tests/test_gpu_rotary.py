"""Rotary positions, by themselves and on the way into the cache, through the C ABI, against the formulas in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import cache_contents, load_abq_attention, quantise  # noqa: E402
from decoding_reference import turned  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def angles(pairs, axes, base=10000.0):
    i = torch.arange(pairs, dtype=torch.float64)
    return base ** (-i / pairs) / (2 * np.pi), (i * axes / pairs).to(torch.int32)


def places(gen, axes, tokens, far):
    return torch.randint(-3, far, (axes, tokens), generator=gen, dtype=torch.int64).to(torch.int32)


def near(got, want, allowed):
    off = (got.cpu().double() - want).abs()
    assert (off <= allowed).all(), float((off - allowed).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs,axes", [(128, 64, 1), (128, 64, 3), (64, 32, 2), (128, 32, 1), (16, 8, 1), (80, 16, 4), (96, 48, 1), (256, 128, 8), (240, 8, 1)])
def test_turned_rows(attn, dtype, interleaved, dim, pairs, axes):
    gen = torch.Generator().manual_seed(dim + pairs + axes)
    turns, axis = angles(pairs, axes)
    rotary = attn.Rotary(turns, axis, axes, interleaved=interleaved)
    for tokens, heads, kv_heads, far in [(1, 1, 1, 10), (3, 5, 2, 100000), (70, 9, 3, 2 ** 31 - 1)]:
        q, k = (torch.randn(tokens, h, dim, generator=gen).to(dtype).cuda() for h in (heads, kv_heads))
        at = places(gen, axes, tokens, far)
        before = q.clone(), k.clone()
        got = rotary.apply(q, k, at.cuda())
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
        for x, y in zip((q, k), got):
            near(y, *turned(x, at, turns, axis, interleaved))
        again = rotary.apply(q, k, at.cuda(), out=(q, k))  # in place
        assert again[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])
        only = rotary.apply(before[0], None, at.cuda())
        assert only[1] is None and torch.equal(only[0], got[0])


def test_the_usual_angles(attn):
    one, three = attn.Rotary.of_base(128), attn.Rotary.of_base(128, sections=(16, 24, 24))
    turns, _ = angles(64, 1)
    assert torch.allclose(one.turns.cpu(), turns, rtol=1e-14) and one.axes == 1 and three.axes == 3
    assert three.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    x = torch.randn(5, 2, 128).half().cuda()
    at = torch.arange(5, dtype=torch.int32).cuda()
    assert torch.equal(one.apply(x, None, at)[0], three.apply(x, None, at.expand(3, 5).contiguous())[0])


def test_a_row_of_position_zero_and_scores_by_distance(attn):
    """Position 0 leaves a row as it is; products of a query and a key depend on the distance alone"""
    rotary = attn.Rotary.of_base(128)
    x = torch.randn(4, 3, 128).half().cuda()
    x[0, 0, :3] = torch.tensor([65504.0, -65504.0, 6e-8])
    assert torch.equal(rotary.apply(x, None, torch.zeros(4, dtype=torch.int32).cuda())[0], x)
    q, k = torch.randn(1, 1, 128).bfloat16().cuda(), torch.randn(1, 1, 128).bfloat16().cuda()
    scores = []
    for far in (0, 1000, 123456789):
        a, b = (rotary.apply(t, None, torch.tensor([far + p], dtype=torch.int32).cuda())[0].double() for t, p in ((q, 70), (k, 13)))
        scores.append(float((a * b).sum()))
        size = float((a.abs() * b.abs()).sum())
    assert max(scores) - min(scores) <= 2 * size * 2 * 2.0 ** -8 * 1.01  # (each element rounded once, by half a step)


def test_rows_that_are_not_finite_stay_in_their_pairs(attn):
    rotary = attn.Rotary.of_base(64)
    x = torch.randn(3, 2, 128).half().cuda()
    at = torch.tensor([5, 6, 7], dtype=torch.int32).cuda()
    clean = rotary.apply(x, None, at)[0]
    bad = x.clone()
    bad[1, 0, 3], bad[1, 1, 40], bad[2, 0, 100], bad[2, 1, 90] = float("inf"), float("nan"), float("-inf"), float("nan")
    got = rotary.apply(bad, None, at)[0]
    hit = torch.zeros(x.shape, dtype=torch.bool)
    hit[1, 0, [3, 35]] = hit[1, 1, [8, 40]] = True
    hit[2, 0, 100] = hit[2, 1, 90] = True
    hit = hit.cuda()
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()
    assert got[2, 0, 100] == float("-inf")  # (behind what turns: copied)


def test_rows_are_slices_and_nothing_else_is_touched(attn):
    gen = torch.Generator().manual_seed(3)
    heads, kv, dim, tokens = 4, 2, 128, 37
    fused = torch.randn(tokens, (heads + 2 * kv) * dim + 16, generator=gen).half().cuda()
    q, k = (fused[:, a:b].unflatten(1, (-1, dim)) for a, b in ((8, 8 + heads * dim), (8 + heads * dim, 8 + (heads + kv) * dim)))
    into = torch.full((kv, tokens + 2, dim + 8), 5.0, dtype=torch.float16, device="cuda")
    k_out = into[:, 1:-1, :dim].transpose(0, 1)
    turns, axis = angles(64, 1)
    at = places(gen, 1, tokens, 5000)
    want = [turned(x, at, turns, axis, False) for x in (q, k)]
    rest = fused[:, 8 + heads * dim:].clone(), fused[:, :8].clone()
    rotary = attn.Rotary(turns)
    rotary.apply(q, k, at[0].cuda(), out=(q, k_out))
    near(q, *want[0])
    near(k_out, *want[1])
    assert torch.equal(fused[:, 8 + heads * dim:], rest[0]) and torch.equal(fused[:, :8], rest[1])
    assert (into[:, 0] == 5).all() and (into[:, -1] == 5).all() and (into[:, :, dim:] == 5).all()
    wide = torch.randint(0, 100, (3, 50), generator=gen).to(torch.int32).cuda()  # axes apart by more than the tokens
    three = attn.Rotary.of_base(dim, sections=(20, 20, 24))
    assert torch.equal(three.apply(k, None, wide[:, :tokens])[0], three.apply(k, None, wide[:, :tokens].contiguous())[0])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,pairs,interleaved", [(128, 64, False), (128, 64, True), (64, 32, False), (64, 16, True), (128, 16, False)])
def test_the_cache_holds_the_turned_keys(attn, bits, symmetric, dtype, dim, pairs, interleaved):
    """As abq_rotary_apply followed by abq_kv_append: bit for bit"""
    gen = torch.Generator().manual_seed(bits + dim + pairs)
    turns, axis = angles(pairs, 2)
    rotary = attn.Rotary(turns, axis, interleaved=interleaved)
    for tokens, heads, kv, size in [(1, 4, 4, 16), (7, 6, 2, 16), (130, 9, 3, 64)]:
        pages = tokens // size + 3
        q, k, v = (torch.randn(tokens, h, dim, generator=gen).to(dtype).cuda() for h in (heads, kv, kv))
        at = places(gen, 2, tokens, 9000).cuda()
        slots = torch.randperm(pages * size, generator=gen)[:tokens] if tokens < 100 else torch.arange(5, 5 + tokens)
        slots = slots.to(torch.int32)
        if tokens > 5:
            slots[3], slots[5] = -1, pages * size
        slots = slots.cuda()
        one, two = (attn.KvCache(pages, size, kv, dim, bits=bits, symmetric=symmetric) for _ in range(2))
        q_want, k_want = rotary.apply(q, k, at)
        one.append(k_want, v, slots)
        k_out = torch.empty_like(k)
        for keep in (k_out, None):
            q_got, k_got = two.append_rotated(rotary, q, k, v, at, slots, k_out=keep)
            assert torch.equal(q_got, q_want) and (keep is None or torch.equal(k_got, k_want)) and (keep is not None or k_got is None)
            for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
                assert torch.equal(getattr(one, name), getattr(two, name)), (name, tokens)
                getattr(two, name).zero_() if "codes" in name else getattr(two, name).fill_(1)
        two.append_rotated(rotary, None, k, v, at, slots)
        assert torch.equal(one.k_codes, two.k_codes) and torch.equal(one.v_codes, two.v_codes)
        there = (slots.cpu() >= 0) & (slots.cpu() < pages * size)
        got = cache_contents(two)[0][slots.cpu()[there].numpy()]
        assert np.array_equal(got, quantise(k_want.cpu(), bits, symmetric)[0][there.numpy()])


def test_one_at_a_time_is_as_all_at_once(attn):
    """A cache filled token by token holds what one filled by a prompt holds"""
    gen = torch.Generator().manual_seed(12)
    rotary = attn.Rotary.of_base(128)
    k, v = (torch.randn(90, 2, 128, generator=gen).half().cuda() for _ in range(2))
    at, slots = torch.arange(90, dtype=torch.int32).cuda(), torch.arange(90, dtype=torch.int32).cuda()
    whole, single = attn.KvCache(2, 64, 2, 128), attn.KvCache(2, 64, 2, 128)
    whole.append_rotated(rotary, None, k, v, at, slots)
    for i in range(90):
        single.append_rotated(rotary, None, k[i:i + 1], v[i:i + 1], at[i:i + 1], slots[i:i + 1])
    assert torch.equal(whole.k_codes, single.k_codes) and torch.equal(whole.v_codes, single.v_codes) and torch.equal(whole.k_scales, single.k_scales)


def test_no_rows(attn):
    rotary = attn.Rotary.of_base(128)
    none, at = torch.empty((0, 2, 128), dtype=torch.float16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    assert rotary.apply(none, none, at)[0].shape == none.shape
    attn.KvCache(2, 16, 2, 128).append_rotated(rotary, none, none, none, at, at)
