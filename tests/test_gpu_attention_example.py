"""examples/decoder_attention.py: linears, cache and attentions of one decoder layer run together, each call against the formulas on
what the engine's own QKV linear gave"""
import importlib.util
import os
import sys

import pytest

torch = pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_gpu_attention import prompt_reference, tree_reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    load_abq_attention()
    path = list(sys.path)
    spec = importlib.util.spec_from_file_location("decoder_attention", os.path.join(ROOT, "examples", "decoder_attention.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    sys.path[:] = path
    return module


def check_output(layer, got, mixed, allowed):
    """got is the output linear of an attention result that may be `allowed` off mixed, rounded to fp16, quantised to 8 bits (half a
    step, a 127th of the row's largest, on either side of the clamp) and multiplied in whole numbers; the product is rounded to fp16"""
    mixed, allowed = mixed.flatten(1), allowed.flatten(1)
    step = (mixed.abs() + allowed).amax(1, keepdim=True) / 127 + 1e-5
    weight = layer.out.value.cpu().double()
    want = mixed @ weight.T
    bound = (allowed + mixed.abs() * 2.0 ** -11 + 0.51 * step) @ weight.abs().T + want.abs() * 2.0 ** -10 + 1e-4
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("hidden,heads,kv_heads,kv_bits,kv_symmetric", [(4096, 32, 8, 8, True), (512, 8, 8, 4, False)])
def test_a_layers_attention_call_by_call(example, hidden, heads, kv_heads, kv_bits, kv_symmetric):
    gen = torch.Generator(device="cuda").manual_seed(1)
    layer = example.DecoderAttention(hidden, heads, kv_heads, pages=30, page_size=16, kv_bits=kv_bits, kv_symmetric=kv_symmetric)
    pages = example.Pages(30, 16, 10 * 16)
    lengths, later, counts = [90, 3], [20, 0], [5, 2]
    for _ in lengths:
        pages.add_sequence()
    scale = layer.dim ** -0.5

    x = torch.randn(sum(lengths), hidden, generator=gen, device="cuda").half()
    q, k, v = layer.project(x)
    y = layer.prompts(x, example.starts(lengths), max(lengths), pages.slots([0, 0], lengths))
    check_output(layer, y, *prompt_reference(q, k, v, lengths, lengths, scale))

    whole = [a + b for a, b in zip(lengths, later)]
    x = torch.randn(sum(later), hidden, generator=gen, device="cuda").half()
    everything = pages.slots([0, 0], whole)
    y = layer.chunk(x, example.starts(later), max(later), pages.slots(lengths, whole), example.starts(whole), max(whole), everything)
    k, v = layer.cache.read(everything)
    check_output(layer, y, *prompt_reference(layer.project(x)[0], k, v, later, whole, scale))

    x = torch.randn(sum(counts), hidden, generator=gen, device="cuda").half()
    mask = example.tree_mask([[-1, 0, 0, 2, -1], [-1, -1]])
    y = layer.drafts(x, example.starts(counts), max(counts), pages.slots(whole, [a + b for a, b in zip(whole, counts)]), pages.table(),
                     torch.tensor(whole, dtype=torch.int32).cuda(), max(whole), mask=mask)
    check_output(layer, y, *tree_reference(layer.project(x)[0], layer.cache, pages.table(), whole, counts, mask.cpu(), scale))


def test_the_program_runs(example):
    off = example.main(hidden=512, heads=8, kv_heads=4, lengths=(65, 1, 300), later=(3, 90, 1))
    assert set(off) == {"prompts", "chunk", "drafts"} and all(0 < x < 1 for x in off.values())
