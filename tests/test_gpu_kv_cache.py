"""The quantised key / value cache through the C ABI: codes, scales and zero points against the stated format, bit for bit."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import cache_contents, load_abq_attention, quantise  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def rows_like(gen, tokens, heads, dim, dtype):
    """Rows as they come, and the ones a quantiser trips over: constant, tiny, huge, all of one sign, one element far out"""
    x = torch.randn(tokens, heads, dim, generator=gen) * torch.exp(torch.randn(tokens, heads, 1, generator=gen))
    for i in range(tokens):
        kind = i % 9
        if kind == 1:
            x[i] = 0
        elif kind == 2:
            x[i] = 3.25
        elif kind == 3:
            x[i] *= 1e-6
        elif kind == 4:
            x[i] = x[i].abs() + 50
        elif kind == 5:
            x[i] = -x[i].abs() - 7
        elif kind == 6:
            x[i, :, ::7] *= 900
        elif kind == 7:
            x[i] = torch.round(x[i])
    return x.to(dtype)


def slots_of(kind, tokens, pages, size, rng):
    places = pages * size
    if kind == "scattered":
        return rng.permutation(places)[:tokens].astype(np.int32)
    start = {"aligned": 4 * (size // 8), "shifted": 3}[kind]
    order = rng.permutation(pages)[:(start + tokens + size - 1) // size]
    at = np.arange(start, start + tokens)
    return (order[at // size] * size + at % size).astype(np.int32)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,size", [(128, 3, 16), (64, 5, 64), (128, 1, 32), (64, 2, 16)])
def test_written_codes_are_the_formats(attn, bits, symmetric, dtype, dim, heads, size):
    gen, rng = torch.Generator().manual_seed(bits + dim), np.random.default_rng(size + heads)
    pages = 40
    for tokens, kind in [(1, "scattered"), (3, "aligned"), (4, "aligned"), (5, "shifted"), (70, "shifted"), (131, "aligned"), (129, "scattered")]:
        cache = attn.KvCache(pages, size, heads, dim, bits=bits, symmetric=symmetric)
        for t in (cache.k_codes, cache.v_codes):
            t.fill_(0x5a)
        before = cache_contents(cache)
        k, v = rows_like(gen, tokens, heads, dim, dtype), rows_like(gen, tokens, heads, dim, dtype).flip(0)
        slots = slots_of(kind, tokens, pages, size, rng)
        dropped = rng.random(tokens) < 0.2 if tokens > 4 else np.zeros(tokens, bool)
        given = np.where(dropped, rng.choice([-1, -7, pages * size, 2 ** 31 - 1], tokens), slots).astype(np.int32)
        cache.append(k.cuda(), v.cuda(), torch.from_numpy(given).cuda())
        after = cache_contents(cache)
        keep = np.ones(pages * size, bool)
        keep[slots[~dropped]] = False
        for name, x, codes, scales, old, old_scales in (("k", k, after[0], after[2], before[0], before[2]), ("v", v, after[1], after[3], before[1], before[3])):
            want, scale, zero = quantise(x, bits, symmetric)
            at = slots[~dropped]
            what = (name, tokens, kind)
            assert np.array_equal(scales[0][at], scale[~dropped]), what
            assert np.array_equal(scales[1][at], zero[~dropped]), what
            assert np.array_equal(codes[at], want[~dropped]), what
            assert np.array_equal(codes[keep], old[keep]) and np.array_equal(scales[0][keep], old_scales[0][keep]), what  # nothing else is touched
        # read back: the values the codes stand for, rounded once
        for out_type in (torch.float16, torch.bfloat16):
            back = cache.read(torch.from_numpy(given).cuda(), dtype=out_type)
            for x, got in zip((k, v), back):
                code, scale, zero = quantise(x, bits, symmetric)
                value = (code.astype(np.float32) - zero[..., None]) * scale[..., None]
                want = torch.from_numpy(value).to(out_type)
                want[torch.from_numpy(dropped)] = 0
                assert torch.equal(got.cpu(), want), (tokens, kind, out_type)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_are_slices_of_larger_tensors(attn, dtype):
    gen = torch.Generator().manual_seed(4)
    heads, dim, tokens = 4, 128, 37
    fused = torch.randn(tokens, 3 * heads * dim + 24, generator=gen).to(dtype).cuda()
    k = fused[:, heads * dim + 8: 2 * heads * dim + 8].unflatten(1, (heads, dim))
    v = torch.randn(heads, tokens, dim, generator=gen).to(dtype).cuda().transpose(0, 1)  # heads outermost
    cache = attn.KvCache(5, 16, heads, dim, bits=8)
    slots = torch.arange(11, 11 + tokens, dtype=torch.int32).cuda()
    cache.append(k, v, slots)
    kc, vc, _, _ = cache_contents(cache)
    assert np.array_equal(kc[11:11 + tokens], quantise(k.cpu(), 8, True)[0]) and np.array_equal(vc[11:11 + tokens], quantise(v.cpu(), 8, True)[0])
    into = torch.full((tokens, 2 * heads * dim + 8), 9.0, dtype=dtype, device="cuda")
    out = (into[:, :heads * dim].unflatten(1, (heads, dim)), into[:, heads * dim + 8:].unflatten(1, (heads, dim)))
    cache.read(slots, out=out)
    want = cache.read(slots, dtype=dtype)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert (into[:, heads * dim:heads * dim + 8] == 9).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
def test_rows_that_are_not_finite_leave_finite_scales_and_the_other_rows_alone(attn, bits, symmetric):
    gen = torch.Generator().manual_seed(9)
    k = torch.randn(8, 2, 64, generator=gen).half()
    clean = k.clone()
    k[1, 0, 5], k[2, 1, 0], k[3, 0], k[5, 1, 63] = float("inf"), float("-inf"), float("nan"), float("nan")
    cache = attn.KvCache(2, 16, 2, 64, bits=bits, symmetric=symmetric)
    slots = torch.arange(8, dtype=torch.int32).cuda()
    cache.append(k.cuda(), k.cuda(), slots)
    got = cache_contents(cache)
    want, scale, _ = quantise(clean, bits, symmetric)
    touched = np.zeros((8, 2), bool)
    touched[[1, 2, 3, 5], [0, 1, 0, 1]] = True
    for codes, scales in ((got[0], got[2]), (got[1], got[3])):
        assert np.isfinite(scales[0][:8]).all() and np.isfinite(scales[1][:8]).all() and (scales[0][:8] >= 1e-5).all()
        assert np.array_equal(codes[:8][~touched], want[~touched]) and np.array_equal(scales[0][:8][~touched], scale[~touched])
    assert all(torch.isfinite(x).all() for x in cache.read(slots, dtype=torch.bfloat16))  # (1e4 times a code is beyond fp16)


def test_no_rows_and_another_stream(attn):
    cache = attn.KvCache(4, 16, 2, 128)
    none = torch.empty((0, 2, 128), dtype=torch.float16, device="cuda")
    cache.append(none, none, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert cache.read(torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0, 2, 128)
    stream = torch.cuda.Stream()
    k = torch.randn(5, 2, 128).half().cuda()
    slots = torch.tensor([3, 9, 17, 2, 40], dtype=torch.int32).cuda()
    stream.wait_stream(torch.cuda.current_stream())
    cache.append(k, k, slots, stream=stream)
    stream.synchronize()
    assert np.array_equal(cache_contents(cache)[1][slots.cpu().numpy()], quantise(k.cpu(), 8, True)[0])
