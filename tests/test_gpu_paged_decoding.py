"""examples/paged_decoding.py: tables of pages, rotary positions, cache, bounds and attention to chosen pages run together, eagerly and
captured, each step against the formulas on what the engine's own QKV linear gave"""
import importlib.util
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attention_reference import load_abq_attention, quantise  # noqa: E402
from conftest import ROOT  # noqa: E402
from decoding_reference import sparse_reference, turned  # noqa: E402
from test_gpu_attention import prompt_reference  # noqa: E402
from test_gpu_attention_example import check_output  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    load_abq_attention()
    path = list(sys.path)
    spec = importlib.util.spec_from_file_location("paged_decoding", os.path.join(ROOT, "examples", "paged_decoding.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    sys.path[:] = path
    return module


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("hidden,heads,kv_heads,bits,symmetric,page", [(512, 8, 2, 8, True, 16), (1024, 8, 8, 4, False, 32)])
def test_prompts_and_steps(example, captured, hidden, heads, kv_heads, bits, symmetric, page):
    gen, rng = torch.Generator(device="cuda").manual_seed(1), np.random.default_rng(3)
    layer = example.DecoderAttention(hidden, heads, kv_heads, pages=1, page_size=16, kv_bits=bits, kv_symmetric=symmetric)
    sequences, lengths = 6, [90, 0, 47, 3, 64, 0]
    decoder = example.PagedDecoder(layer, sequences, max_pages=9, num_pages=60, page_size=page, chosen=2)
    scale = layer.dim ** -0.5

    x = torch.randn(sum(lengths), hidden, generator=gen, device="cuda").half()
    y = decoder.prompts(x, lengths)
    q, k, v = layer.project(x)
    at = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths])
    q, k = decoder.rotary.apply(q, k, at.cuda())
    check_output(layer, y, *prompt_reference(q, k, v, lengths, lengths, scale))
    # every sequence's tokens, in order: rows of turned keys and of values
    held = [list(zip(a.cpu(), b.cpu())) for a, b in zip(k.split(lengths), v.split(lengths))]

    x = torch.zeros(sequences, hidden, dtype=torch.float16, device="cuda")
    parents = torch.arange(sequences, dtype=torch.int32).cuda()
    graph, into = torch.cuda.CUDAGraph(), None
    if captured:
        side = torch.cuda.Stream()  # (a first pass outside of the capture)
        before = [t.clone() for t in (decoder.pages.table, decoder.pages.lengths, decoder.pages.refs)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decoder.step(x)
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip((decoder.pages.table, decoder.pages.lengths, decoder.pages.refs), before):
            t.copy_(old)
        with torch.cuda.graph(graph):
            decoder.fork(parents)
            into = decoder.step(x)
    for i in range(40):
        p = rng.integers(0, sequences, sequences) if i % 4 == 0 else np.arange(sequences)
        parents.copy_(torch.from_numpy(p.astype(np.int32)))
        x.copy_(torch.randn(sequences, hidden, generator=gen, device="cuda"))
        held = [list(held[j]) for j in p]
        if captured:
            graph.replay()
            y = into
        else:
            decoder.fork(parents)
            y = decoder.step(x)
        q, k, v = layer.project(x)
        at = torch.tensor([len(h) for h in held], dtype=torch.int32)
        q, k = decoder.rotary.apply(q, k, at.cuda())
        torch.cuda.synchronize()
        assert decoder.context.tolist() == at.tolist() and torch.equal(decoder.q, q)
        for h, a, b in zip(held, k.cpu(), v.cpu()):
            h.append((a, b))
        table = decoder.pages.table.cpu().numpy()
        if i % 13 == 12:  # what the cache holds is what each sequence was given
            for s, h in enumerate(held):
                t = np.arange(len(h))
                slots = torch.from_numpy((table[s][t // page] * page + t % page).astype(np.int32)).cuda()
                for side, got in enumerate(decoder.cache.read(slots, dtype=torch.float16)):
                    code, step, zero = quantise(torch.stack([x[side] for x in h]), bits, symmetric)
                    want = (code.astype(np.float32) - zero[..., None]) * step[..., None]
                    assert torch.equal(got.cpu(), torch.from_numpy(want).half()), (i, s, side)
        if i % 5 == 4:
            want, allowed = sparse_reference(q, decoder.cache, table, at.tolist(), [1] * sequences, None, scale, decoder.call.blocks.tolist())
            check_output(layer, y, want, allowed)
    assert torch.equal(decoder.pages.refs.cpu(), torch.bincount(torch.from_numpy(table[table >= 0]).long(), minlength=60).int())


def test_keys_turned_by_the_layer(example):
    """The example's angles are those of the formula"""
    rotary = example.abq_attention.Rotary.of_base(64)
    x = torch.randn(5, 2, 64).half().cuda()
    at = torch.tensor([[0, 1, 50, 4000, 70000]], dtype=torch.int32)
    pairs = torch.arange(32, dtype=torch.float64)
    want, allowed = turned(x, at, rotary.turns.cpu(), torch.zeros(32, dtype=torch.int64), False)
    assert torch.allclose(rotary.turns.cpu() * 2 * np.pi, 10000.0 ** (-pairs / 32), rtol=1e-14)
    assert ((rotary.apply(x, None, at.cuda())[0].cpu().double() - want).abs() <= allowed).all()


def test_the_program_runs(example):
    off, read, used = example.main(hidden=512, heads=8, kv_heads=4, lengths=(300, 1, 130), answers=3, steps=45, chosen=3)
    assert 0 <= off < 2 and 0 < read <= 1 and 0 < used <= 16 * 9
