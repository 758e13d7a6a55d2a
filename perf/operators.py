"""Attention on a quantised key / value cache, as a program that serves a model with the engine's linears runs it.

Three kinds of pass, each through the public binding (abq-llm_amd/abq_attention.py) where `own` is set, and otherwise in the
operators' plain form, elementary torch operations in 32 bits:

  cache    new keys and values [tokens, kv heads, head dim] quantised per token and head as they are written into a paged cache
           of 8- or 4-bit codes, and the last tokens of every sequence read back in the type of the activations.
  prompt   causal attention of whole prompts: packed sequences of different lengths, grouped heads, queries, keys and values as
           slices of one fused QKV result; with a prefix, the queries are the last tokens of a longer sequence.
  tree     attention of each sequence's drafted tokens over its quantised cache: every draft sees the context and those drafts that
           its mask names (its ancestors in the tree); one draft per sequence is ordinary decoding.

Lengths are rules of a case's numbers, values come from the seed.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _binding():
    # (the package directory's name is no Python identifier: the binding is loaded by its path)
    if "abq_attention" not in sys.modules:
        path = os.path.join(os.getcwd(), "abq-llm_amd", "abq_attention.py")
        spec = importlib.util.spec_from_file_location("abq_attention", path)
        module = importlib.util.module_from_spec(spec)
        sys.modules["abq_attention"] = module
        spec.loader.exec_module(module)
    return sys.modules["abq_attention"]


# ------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token for each of sixteen sequences written during decoding: a call of a few microseconds
        {"name": "cache_decode_16", "kind": "cache", "seqs": 16, "append": 1, "read": 1, "ragged": False, "page": 64,
         "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # a chunk of a prompt on the 13B heads, written as 4-bit codes with zero points; the prefix is read back with it
        {"name": "cache_chunk_777", "kind": "cache", "seqs": 1, "append": 777, "read": 3001, "ragged": False, "page": 16,
         "kv_heads": 40, "dim": 128, "bits": 4, "symmetric": False, "type": "bf16"},
        # sixteen prompts of 1024 tokens, the prefill of the benchmark's layer
        {"name": "cache_16x1024", "kind": "cache", "seqs": 16, "append": 1024, "read": 1024, "ragged": False, "page": 64,
         "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # a short question
        {"name": "prompt_47", "kind": "prompt", "seqs": 1, "longest": 47, "prefix": 0, "ragged": False, "heads": 32, "kv_heads": 32,
         "dim": 128, "type": "fp16"},
        # one prompt of 1024 tokens on the 7B heads
        {"name": "prompt_1024", "kind": "prompt", "seqs": 1, "longest": 1024, "prefix": 0, "ragged": False, "heads": 32, "kv_heads": 32,
         "dim": 128, "type": "fp16"},
        # a batch of prompts as they come, from a few tokens to 2047, four query heads to a key head
        {"name": "prompt_ragged_13", "kind": "prompt", "seqs": 13, "longest": 2047, "prefix": 0, "ragged": True, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16"},
        # the next chunk of a long conversation, heads of 64
        {"name": "prompt_prefix_7000", "kind": "prompt", "seqs": 1, "longest": 333, "prefix": 7000, "ragged": False, "heads": 24, "kv_heads": 8,
         "dim": 64, "type": "fp16"},
        # one long document
        {"name": "prompt_16384", "kind": "prompt", "seqs": 1, "longest": 16384, "prefix": 0, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16"},
        # one token of one user, a thousand tokens behind it
        {"name": "tree_1_token", "kind": "tree", "seqs": 1, "drafts": 1, "context": 1000, "ragged": False, "page": 64, "heads": 32,
         "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # the benchmark's batch of sixteen sequences of 1024 tokens, one token each
        {"name": "tree_16x1024", "kind": "tree", "seqs": 16, "drafts": 1, "context": 1024, "ragged": False, "page": 64, "heads": 32,
         "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # a tree of 27 drafts behind a long context, grouped heads, 4-bit codes with zero points
        {"name": "tree_27_drafts", "kind": "tree", "seqs": 3, "drafts": 27, "context": 5500, "ragged": False, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "bits": 4, "symmetric": False, "type": "bf16"},
        # many users with contexts of any length up to 16384, five drafts each
        {"name": "tree_48_ragged", "kind": "tree", "seqs": 48, "drafts": 5, "context": 16384, "ragged": True, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
    ]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["cache", "prompt", "prompt", "tree", "tree"])
        kv_heads, group = rng.choice([(32, 1), (40, 1), (8, 4), (8, 8), (4, 7), (1, 16), (12, 1), (5, 3)])
        case = {"kind": kind, "seqs": _size(rng, 1, 64), "ragged": rng.random() < 0.5, "kv_heads": kv_heads,
                "dim": rng.choice([64, 128, 128]), "type": rng.choice(["fp16", "fp16", "bf16"])}
        if kind != "prompt":
            case.update(page=rng.choice([16, 32, 64, 128]), bits=rng.choice([8, 8, 4]), symmetric=rng.random() < 0.5)
        if kind == "cache":
            append = _size(rng, 1, 8192)
            case.update(append=append, read=append + (_size(rng, 1, 8192) if rng.random() < 0.4 else 0))
            if case["seqs"] * case["read"] > 40000:
                continue
        elif kind == "prompt":
            case.update(heads=kv_heads * group, longest=_size(rng, 1, 8192), prefix=_size(rng, 1, 12000) if rng.random() < 0.4 else 0)
            if case["seqs"] * case["heads"] * case["longest"] * (case["longest"] + case["prefix"]) > 3e9:
                continue
        else:
            case.update(heads=kv_heads * group, drafts=1 if rng.random() < 0.4 else _size(rng, 2, 64), context=_size(rng, 1, 32768))
            if case["seqs"] * case["context"] * kv_heads * case["dim"] > 1e9:
                continue
        if _cost(case) <= most:
            return case


def _size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _lengths(case):
    """(tokens before the call, tokens of the call) of every sequence; ragged: the first is the longest, the others anything below"""
    n, rng = case["seqs"], random.Random(case["seqs"] * 7919 + case["kv_heads"])
    spread = [1.0] + [rng.random() ** 1.5 if case["ragged"] else 1.0 for _ in range(n - 1)]
    if case["kind"] == "cache":
        new = [max(1, int(s * case["append"])) for s in spread]
        return [(case["read"] - case["append"], t) for t in new]
    if case["kind"] == "prompt":
        return [(int(s * case["prefix"]), int(s * case["longest"])) for s in spread]
    return [(int(s * case["context"]), 1 + int((case["drafts"] - 1) * math.sqrt(s))) for s in spread]


def work(case):
    lens, dim, kv = _lengths(case), case["dim"], case["kv_heads"]
    new, whole = sum(t for _, t in lens), sum(c + t for c, t in lens)
    if case["kind"] == "prompt":
        pairs = sum(t * c + t * (t + 1) // 2 for c, t in lens)
        return {"bytes": 4.0 * dim * (new * case["heads"] + whole * kv), "flops": 4.0 * dim * case["heads"] * pairs}
    row = dim * case["bits"] / 8 + (4 if case["symmetric"] else 8)  # codes, scale and zero point of a token and head
    if case["kind"] == "cache":
        return {"bytes": 2.0 * kv * (new * (2 * dim + row) + whole * (2 * dim + row)), "flops": 0.0}
    pairs = sum(t * (c + 1) for c, t in lens)
    return {"bytes": 2.0 * kv * whole * row + 4.0 * dim * new * case["heads"], "flops": 4.0 * dim * case["heads"] * pairs}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 8e14)


# ------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _keys_and_values(gen, tokens, case):
    """rows as a model writes them: keys with a few channels far from zero, every token's values at a level of its own"""
    shape = (tokens, case["kv_heads"], case["dim"])
    channel = torch.exp(0.4 * torch.randn((1,) + shape[1:], generator=gen, device="cuda"))
    offset = 1.5 * (torch.rand((1,) + shape[1:], generator=gen, device="cuda") < 0.06)
    k = torch.randn(shape, generator=gen, device="cuda") * channel + offset
    v = torch.randn(shape, generator=gen, device="cuda") * torch.exp(0.5 * torch.randn((tokens, 1, 1), generator=gen, device="cuda"))
    return k.to(_TYPES[case["type"]]), v.to(_TYPES[case["type"]])


def _starts(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()


def _pages(case, gen):
    """(page table [sequences, pages], pages): every sequence's pages lie anywhere in the cache"""
    each = max((c + t + case["page"] - 1) // case["page"] for c, t in _lengths(case))
    order = torch.randperm(case["seqs"] * each + 3, generator=gen, device="cuda")[: case["seqs"] * each]
    return order.to(torch.int32).view(case["seqs"], each), case["seqs"] * each + 3


def _slots(case, table, first, last):
    """The places in the cache of the tokens first[i] .. last[i] - 1 of every sequence, one behind the other"""
    count = torch.tensor([b - a for a, b in zip(first, last)], device="cuda")
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), count)
    ahead = torch.tensor(first, device="cuda") - (count.cumsum(0) - count)
    at = torch.arange(int(count.sum()), device="cuda") + ahead[seq]
    return (table[seq, at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)


def _ancestors(lens, seed):
    """For every draft the bits of the drafts that it sees: its ancestors in a random tree, and itself"""
    rng, masks = random.Random(seed), []
    for _, t in lens:
        seen = []
        for i in range(t):
            parent = rng.randint(max(0, i - 6), i - 1) if i else None
            seen.append((1 << i) | (seen[parent] if i else 0))
        masks += seen
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()


def prepare(case, seed):
    gen, lens, dtype = _gen(seed), _lengths(case), _TYPES[case["type"]]
    new, whole, dim, kv = sum(t for _, t in lens), sum(c + t for c, t in lens), case["dim"], case["kv_heads"]
    state = {"case": case, "scale": dim ** -0.5}
    if case["kind"] == "prompt":
        heads = case["heads"]
        k, v = _keys_and_values(gen, whole, case)
        q = torch.randn((new, heads, dim), generator=gen, device="cuda").to(dtype)
        if new == whole:  # slices of one fused result
            qkv = torch.cat([q.view(new, -1), k.view(new, -1), v.view(new, -1)], 1)
            q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        state.update(q=q, k=k, v=v, q_starts=_starts([t for _, t in lens]), k_starts=_starts([c + t for c, t in lens]),
                     max_q=max(t for _, t in lens), max_k=max(c + t for c, t in lens))
        if own:
            out = torch.empty((new, heads, dim), dtype=dtype, device="cuda")
            state["call"] = _binding().PromptAttention(q, k, v, state["q_starts"], state["k_starts"], state["max_q"], state["max_k"],
                                                       scale=state["scale"], out=out)
        return state
    table, pages = _pages(case, gen)
    slots = _slots(case, table, [0] * len(lens), [c + t for c, t in lens])
    k, v = _keys_and_values(gen, whole, case)
    written = _slots(case, table, [c for c, _ in lens], [c + t for c, t in lens])
    if case["kind"] == "cache":
        at = torch.isin(slots, written)
        state.update(k=k[at], v=v[at], written=written, slots=slots)
    else:
        at = torch.ones_like(slots, dtype=torch.bool)
        state.update(q=torch.randn((new, case["heads"], dim), generator=gen, device="cuda").to(dtype), table=table,
                     context=torch.tensor([c for c, _ in lens], dtype=torch.int32).cuda(), q_starts=_starts([t for _, t in lens]),
                     max_q=max(t for _, t in lens), max_context=max(c for c, _ in lens), mask=_ancestors(lens, seed))
    # the cache as earlier calls left it
    before = ~at if case["kind"] == "cache" else at
    if own:
        binding = _binding()
        cache = binding.KvCache(pages, case["page"], kv, dim, bits=case["bits"], symmetric=case["symmetric"])
        if bool(before.any()):
            cache.append(k[before], v[before], slots[before])
        state["cache"] = cache
        if case["kind"] == "cache":
            state["out"] = (torch.empty((whole, kv, dim), dtype=dtype, device="cuda"), torch.empty((whole, kv, dim), dtype=dtype, device="cuda"))
        else:
            state["call"] = binding.TreeAttention(state["q"], cache, table, state["context"], state["q_starts"], state["max_q"],
                                                  state["max_context"], mask=state["mask"], scale=state["scale"], out=torch.empty_like(state["q"]))
        return state
    codes = torch.zeros((2, pages * case["page"], kv, dim), dtype=torch.int16, device="cuda")
    scales = torch.ones((2, pages * case["page"], kv, 1), device="cuda")
    zeros = torch.zeros((2, pages * case["page"], kv, 1), device="cuda")
    state.update(codes=codes, scales=scales, zeros=zeros)
    if bool(before.any()):
        _write(state, torch.stack([k[before], v[before]]), slots[before])
    return state


# ------------------------------------------------------------------------------------------------- one pass

def _write(state, rows, slots):
    """Quantises rows [2, tokens, heads, dim] per token and head and writes them at their slots"""
    top = 2 ** (state["case"]["bits"] - 1) - 1
    x, at = rows.float(), slots.long()
    if state["case"]["symmetric"]:
        high = x.abs().amax(-1, keepdim=True)
        scale = (high / torch.full_like(high, top)).clamp(1e-5, 1e4)  # (a quotient by a plain number is a product here, not always rounded alike)
        zero = torch.zeros_like(scale)
        code = torch.round(x / scale).clamp(-top - 1, top)
    else:
        low = x.amin(-1, keepdim=True)
        scale = ((x.amax(-1, keepdim=True) - low) / torch.full_like(low, 2 * top + 1)).clamp(1e-5, 1e4)
        zero = torch.round((-low / scale).clamp(-1e4, 1e4))
        code = (torch.round(x / scale) + zero).clamp(0, 2 * top + 1)
    state["codes"][:, at], state["scales"][:, at], state["zeros"][:, at] = code.to(torch.int16), scale, zero


def _values(state, slots):
    """What the cache holds at these slots: keys and values in 32 bits"""
    at = slots.long()
    return (state["codes"][:, at].float() - state["zeros"][:, at]) * state["scales"][:, at]


def _attend(q, k, v, visible, scale):
    """softmax(scale q k^T) v over what is visible; q [seqs, heads, n, dim], k and v [seqs, kv heads, m, dim], visible [seqs, n, m]"""
    seqs, heads, n, dim = q.shape
    kv = k.shape[1]
    s = torch.matmul(q.reshape(seqs, kv, -1, dim), k.transpose(2, 3).contiguous()).mul_(scale)
    s = s.view(seqs, heads, n, -1).masked_fill_(~visible[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.view(seqs, kv, -1, s.shape[-1]), v).view(seqs, heads, n, dim)
    return out / total.masked_fill_(total == 0, 1)


def _padded(starts, longest):
    """(positions [seqs, longest] in the packed rows, which of them are the sequence's own)"""
    at = torch.arange(longest, device="cuda")
    mine = at < (starts[1:] - starts[:-1])[:, None]
    return torch.where(mine, starts[:-1, None] + at, 0).long(), mine


def run(state):
    case = state["case"]
    if own:
        if case["kind"] == "cache":
            state["cache"].append(state["k"], state["v"], state["written"])
            return state["cache"].read(state["slots"], out=state["out"])
        return state["call"].run()
    if case["kind"] == "cache":
        _write(state, torch.stack([state["k"], state["v"]]), state["written"])
        return tuple(_values(state, state["slots"]).to(state["k"].dtype))
    q = state["q"]
    rows, mine = _padded(state["q_starts"], state["max_q"])
    if case["kind"] == "prompt":
        keys, there = _padded(state["k_starts"], state["max_k"])
        k, v = (state[x][keys].float().masked_fill(~there[..., None, None], 0).transpose(1, 2).contiguous() for x in ("k", "v"))
        ahead = (state["k_starts"].diff() - state["q_starts"].diff())[:, None, None]
        place = torch.arange(state["max_k"], device="cuda")
        visible = there[:, None, :] & (place <= ahead + torch.arange(state["max_q"], device="cuda")[:, None])
    else:
        place = torch.arange(state["max_context"] + state["max_q"], device="cuda")
        page = (place // case["page"]).clamp_(max=state["table"].shape[1] - 1)
        k, v = (x.transpose(1, 2).contiguous() for x in _values(state, state["table"][:, page] * case["page"] + place % case["page"]))
        draft = place - state["context"][:, None]  # which draft a place holds, negative in the context
        named = (state["mask"][rows][..., None] >> draft.clamp(0, 63)[:, None, :]) & 1
        drafted = (draft < state["q_starts"].diff()[:, None])[:, None, :] & (named == 1)
        visible = (draft < 0)[:, None, :] | drafted
    out = _attend(q[rows].float().transpose(1, 2), k, v, visible, state["scale"])
    return out.transpose(1, 2)[mine].to(q.dtype)


# ------------------------------------------------------------------------------------------------- the same in 64 bits

def _held(x, bits, symmetric):
    """What a cache of `bits` bits holds of rows x.  The format keeps scales in 32 bits, and the quotient that a code is rounded
    from is one of 32 bits, which decides the ties; everything else is exact"""
    x, held = x.double(), lambda a: a.float().double()
    levels = 2 ** bits - 1
    if symmetric:
        half = (levels - 1) / 2
        step = held((x.abs().amax(-1, keepdim=True) / half).clamp(1e-5, 1e4))
        return held(x / step).round().clamp(-half - 1, half) * step
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = held((held(high - low) / levels).clamp(1e-5, 1e4))
    shift = held(-low / step).clamp(-1e4, 1e4).round()
    return ((held(x / step).round() + shift).clamp(0, levels) - shift) * step


def exact(case, seed):
    gen, lens, dtype, dim, kv = _gen(seed), _lengths(case), _TYPES[case["type"]], case["dim"], case["kv_heads"]
    new, whole = sum(t for _, t in lens), sum(c + t for c, t in lens)
    if case["kind"] == "prompt":
        k, v = _keys_and_values(gen, whole, case)
    else:
        _pages(case, gen)
        k, v = (_held(x, case["bits"], case["symmetric"]) for x in _keys_and_values(gen, whole, case))
    if case["kind"] == "cache":
        return k, v
    q = torch.randn((new, case["heads"], dim), generator=gen, device="cuda").to(dtype).double()
    masks = [m % (1 << 64) for m in _ancestors(lens, seed).tolist()] if case["kind"] == "tree" else None
    out = torch.empty_like(q)
    at_q = at_k = 0
    for c, t in lens:
        see = torch.ones((t, c + t), dtype=torch.bool, device="cuda")
        if masks is None:
            see = see.tril(c)
        else:
            see[:, c:] = torch.tensor([[masks[at_q + i] >> j & 1 for j in range(t)] for i in range(t)], dtype=torch.bool, device="cuda")
        for h in range(case["heads"] if t else 0):
            kh, vh = (x[at_k:at_k + c + t, h * kv // case["heads"]].double() for x in (k, v))
            weight = torch.softmax((q[at_q:at_q + t, h] @ kh.T * dim ** -0.5).masked_fill(~see, -math.inf), -1)
            out[at_q:at_q + t, h] = weight @ vh
        at_q, at_k = at_q + t, at_k + c + t
    return out
