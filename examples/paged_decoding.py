"""Prompts and decoding steps of several requests on one pool of pages, from a decoder layer's input to what its residual adds.

    python examples/paged_decoding.py               (one MI355X; abq-llm_amd/libabq_gemm.so built)

Which pages hold which sequence's tokens is kept on the device (abq_attention.PageTable), so that a step is the same calls whatever the
lengths are, and can be captured into a graph.  The prompts' tokens get room, are turned by their positions as they are quantised into
the cache, and attend to themselves; then every request goes on in several sequences, as in beam search or when several answers are
drawn.  A step:

    fork      sequences take over what others were (a beam that goes on from another's tokens)
    extend    room for one token more; pages that are shared and written to are copied in the cache
    append    QKV linear, rotary positions, keys and values into the cache, bounds of the pages that are complete now
    attend    every sequence chooses pages by their bounds, and attends to those and to its newest tokens; output linear

Weights and inputs are random.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from decoder_attention import DecoderAttention, abq_attention, starts  # noqa: E402


class PagedDecoder:
    def __init__(self, layer, sequences, max_pages, num_pages, page_size=64, chosen=8):
        d = layer.cache.desc
        self.layer, self.sequences = layer, sequences
        self.rotary = abq_attention.Rotary.of_base(layer.dim)
        self.pages = abq_attention.PageTable(num_pages, page_size, sequences, max_pages)
        self.cache = abq_attention.KvCache(num_pages, page_size, d.kv_heads, d.head_dim, bits=d.bits, symmetric=bool(d.symmetric), bounds=True)
        # what a step reads and writes, for as long as it is run
        self.context = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.one = torch.ones(sequences, dtype=torch.int32, device="cuda")
        self.q = torch.empty((sequences, layer.heads, layer.dim), dtype=torch.float16, device="cuda")
        self.call = abq_attention.SparseAttention(self.q, self.cache, self.pages.table, self.context, starts([1] * sequences), 1, max_pages * page_size, chosen)

    def prompts(self, x, lengths):
        """x [tokens, hidden], sequence s having lengths[s] of them and none before"""
        given = self.pages.extend(torch.tensor(lengths, dtype=torch.int32).cuda(), x.shape[0])
        q, k, v = self.layer.project(x)
        positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
        q, k = self.cache.append_rotated(self.rotary, q, k, v, positions, given.slots, k_out=torch.empty_like(k))
        self.cache.bound(given.slots)
        return self.layer.out(abq_attention.PromptAttention(q, k, v, given.starts, max_q=max(lengths)).run().flatten(1))

    def fork(self, parents):
        self.pages.fork(parents)

    def step(self, x):
        """One token more for every sequence: x [sequences, hidden]"""
        self.context.copy_(self.pages.lengths)
        given = self.pages.extend(self.one, self.sequences)
        self.cache.copy_pages(given.copies)
        q, k, v = self.layer.project(x)
        self.cache.append_rotated(self.rotary, q, k, v, self.context, given.slots, q_out=self.q)
        self.cache.bound(given.slots)
        return self.layer.out(self.call.run().flatten(1))


def main(hidden=4096, heads=32, kv_heads=8, lengths=(700, 33, 256), answers=2, steps=70, chosen=6, seed=0):
    """Runs prompts and steps, some of them behind a fork; returns how far the last step is from attention to all tokens (relative, 2-norm), the
    share of the pages that it read, and how many pages are in use"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    layer = DecoderAttention(hidden, heads, kv_heads, pages=1, page_size=64, seed=seed)
    sequences = len(lengths) * answers
    decoder = PagedDecoder(layer, sequences, max_pages=16, num_pages=16 * sequences, chosen=chosen)
    # each request's prompt once; the further answers take over its pages
    first = [n if i == 0 else 0 for n in lengths for i in range(answers)]
    decoder.prompts(torch.randn(sum(lengths), hidden, generator=gen, device="cuda").half(), first)
    decoder.fork(torch.tensor([s - s % answers for s in range(sequences)], dtype=torch.int32).cuda())
    for i in range(steps):
        if i % 20 == 19:  # the first answer goes on from the last one's tokens
            decoder.fork(torch.tensor([s + answers - 1 if s % answers == 0 else s for s in range(sequences)], dtype=torch.int32).cuda())
        y = decoder.step(torch.randn(sequences, hidden, generator=gen, device="cuda").half())
    everything = abq_attention.TreeAttention(decoder.q, decoder.cache, decoder.pages.table, decoder.context, starts([1] * sequences), 1, 16 * 64).run()
    whole = layer.out(everything.flatten(1)).float()
    complete = (decoder.context // 64).clamp(min=1)
    read = (decoder.call.blocks >= 0).sum(-1).float().mean(1) / complete
    return float((y.float() - whole).norm() / whole.norm()), float(read.mean()), int((decoder.pages.refs > 0).sum())


if __name__ == "__main__":
    print("%.3f off attention to all tokens, reading %.0f %% of the complete pages, with %d pages in use" % (lambda a, b, c: (a, 100 * b, c))(*main()))
