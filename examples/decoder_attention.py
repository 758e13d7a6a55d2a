"""The attention half of a decoder layer on the engine, from the layer's input to what its residual adds.

    python examples/decoder_attention.py            (one MI355X; abq-llm_amd/libabq_gemm.so built)

The QKV and output linears run on packed low-bit weights with activations quantised per token (abq_gemm.py); between them keys and
values are quantised into a paged cache as they are written, prompts attend to themselves, and drafted tokens attend to the cache
through a tree mask (abq_attention.py).  Three requests of different lengths share one batch:

    prompts   QKV linear -> cache.append -> PromptAttention -> output linear
    chunk     the same for further tokens of a prompt, on what the cache holds of the earlier ones (cache.read)
    drafts    QKV linear -> cache.append behind the context -> TreeAttention -> output linear

Weights and inputs are random.  Rotary embedding, which a model applies to q and k behind the QKV linear, is left out.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "abq-llm_amd"))
import abq_attention  # noqa: E402
import abq_gemm  # noqa: E402


class Linear:
    """y = x W^T on packed weight codes with a scale per output channel; activations are quantised to 8 bits per token."""

    def __init__(self, rows, cols, bits, gen):
        weight = torch.randn(rows, cols, generator=gen, device="cuda") * cols ** -0.5
        top = 2 ** (bits - 1) - 1
        self.scale = (weight.abs().amax(1) / top).float()
        codes = torch.round(weight / self.scale[:, None]).clamp(-top - 1, top).to(torch.int32)
        self.value = codes.float() * self.scale[:, None]  # what the codes stand for (to check against)
        self.records = abq_gemm.relayout_planes(abq_gemm.pack_i32(codes, bits))

    def __call__(self, x):
        planes, scale, _, _ = abq_gemm.quant_pack_f16(x, 8, symmetric=True, tiled=True)
        return abq_gemm.Gemm(planes, self.records, True, x_tiled=True, w_tiled=True, out_kind=abq_gemm.OUT_F16_SCALED, x_scale=scale,
                             w_scale=self.scale).run()


class DecoderAttention:
    def __init__(self, hidden, heads, kv_heads, pages, page_size=64, w_bits=4, kv_bits=8, kv_symmetric=True, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        self.qkv = Linear((heads + 2 * kv_heads) * self.dim, hidden, w_bits, gen)
        self.out = Linear(hidden, heads * self.dim, w_bits, gen)
        self.cache = abq_attention.KvCache(pages, page_size, kv_heads, self.dim, bits=kv_bits, symmetric=kv_symmetric)

    def project(self, x):
        """q [tokens, heads, dim], k and v [tokens, kv heads, dim]: slices of one result"""
        q, k, v = self.qkv(x).split([self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim], 1)
        return tuple(t.unflatten(1, (-1, self.dim)) for t in (q, k, v))

    def prompts(self, x, starts, longest, slots):
        q, k, v = self.project(x)
        self.cache.append(k, v, slots)
        return self.out(abq_attention.PromptAttention(q, k, v, starts, max_q=longest).run().flatten(1))

    def chunk(self, x, q_starts, longest_q, slots, k_starts, longest_k, all_slots):
        """Further tokens (slots) of sequences whose tokens, these included, stand at all_slots"""
        q, k, v = self.project(x)
        self.cache.append(k, v, slots)
        k, v = self.cache.read(all_slots, dtype=q.dtype)
        return self.out(abq_attention.PromptAttention(q, k, v, q_starts, k_starts, longest_q, longest_k).run().flatten(1))

    def drafts(self, x, starts, most, slots, table, context, longest, mask=None):
        q, k, v = self.project(x)
        self.cache.append(k, v, slots)
        return self.out(abq_attention.TreeAttention(q, self.cache, table, context, starts, most, longest, mask=mask).run().flatten(1))


class Pages:
    """Which pages of the cache hold which sequence's tokens"""

    def __init__(self, pages, page_size, longest):
        self.free, self.size, self.each = list(range(pages))[::-1], page_size, (longest + page_size - 1) // page_size
        self.of = []

    def add_sequence(self):
        self.of.append([self.free.pop() for _ in range(self.each)])

    def slots(self, first, last):
        """int32 slots of the tokens first[i] .. last[i] - 1 of every sequence"""
        flat = [pages[t // self.size] * self.size + t % self.size for pages, a, b in zip(self.of, first, last) for t in range(a, b)]
        return torch.tensor(flat, dtype=torch.int32).cuda()

    def table(self):
        return torch.tensor(self.of, dtype=torch.int32).cuda()


def starts(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()


def tree_mask(parents):
    """Bits of every draft's ancestors and its own, for parents[s][i] (-1: a child of the context)"""
    masks = []
    for tree in parents:
        seen = []
        for i, parent in enumerate(tree):
            seen.append((1 << i) | (seen[parent] if parent >= 0 else 0))
        masks += seen
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()


def main(hidden=4096, heads=32, kv_heads=8, lengths=(700, 33, 256), later=(64, 0, 31), seed=0):
    """Runs the three kinds of call and returns how far each is from the same layer on plain tensors (relative, 2-norm)"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths, later = list(lengths), list(later)
    layer = DecoderAttention(hidden, heads, kv_heads, pages=3 * 16, seed=seed)
    pages = Pages(3 * 16, 64, 16 * 64)
    for _ in lengths:
        pages.add_sequence()
    parents = [[-1, 0, 0, 1, 1, 2], [-1], [-1, 0, 1, -1]]
    counts = [len(p) for p in parents]
    whole = [a + b for a, b in zip(lengths, later)]
    x = [torch.randn(sum(n), hidden, generator=gen, device="cuda").half() for n in (lengths, later, counts)]

    y = [layer.prompts(x[0], starts(lengths), max(lengths), pages.slots([0] * 3, lengths)),
         layer.chunk(x[1], starts(later), max(later), pages.slots(lengths, whole), starts(whole), max(whole), pages.slots([0] * 3, whole)),
         layer.drafts(x[2], starts(counts), max(counts), pages.slots(whole, [a + b for a, b in zip(whole, counts)]), pages.table(),
                      torch.tensor(whole, dtype=torch.int32).cuda(), max(whole), mask=tree_mask(parents))]

    # the same on plain tensors in 32 bits, nothing quantised but the weights
    off, at = [], [0, 0, 0]
    q, k, v = zip(*[[t.unflatten(1, (-1, layer.dim)) for t in (part.float() @ layer.qkv.value.T).split(
        [heads * layer.dim, kv_heads * layer.dim, kv_heads * layer.dim], 1)] for part in x])
    want = [torch.empty(t.shape[0], heads * layer.dim, device="cuda") for t in x]
    for s in range(3):
        spans = [slice(at[i], at[i] + n[s]) for i, n in enumerate((lengths, later, counts))]
        keys, values = (torch.cat([t[i][spans[i]] for i in range(3)]).repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        total = keys.shape[0]
        sees = torch.ones(total, total, dtype=torch.bool, device="cuda").tril()
        for i, m in enumerate(tree_mask([parents[s]]).tolist()):
            sees[whole[s] + i, whole[s]:] = torch.tensor([bool(m >> j & 1) for j in range(counts[s])], device="cuda")
        rows = torch.cat([q[i][spans[i]] for i in range(3)])
        score = torch.einsum("ihd,jhd->hij", rows, keys) * layer.dim ** -0.5
        mixed = torch.einsum("hij,jhd->ihd", torch.softmax(score.masked_fill(~sees, float("-inf")), -1), values).flatten(1)
        for i, part in enumerate(mixed.split([lengths[s], later[s], counts[s]])):
            want[i][spans[i]] = part
            at[i] += part.shape[0]
    for got, plain in zip(y, want):
        plain = plain @ layer.out.value.T
        off.append(float((got.float() - plain).norm() / plain.norm()))
    return dict(zip(("prompts", "chunk", "drafts"), off))


if __name__ == "__main__":
    for what, off in main().items():
        print("%-8s %.4f off the same layer without quantised activations and cache" % (what, off))
