"""What a decoding step needs around the quantised key / value cache, as a program that serves a model with the engine runs it.

Four kinds of pass, each through the public binding (abq-llm_amd/abq_attention.py) where `own` is set, and otherwise in the
operators' plain form, elementary torch operations in 32 bits, or in 64 for angles and for what lies beside a border of a code:

  rotary   queries and keys turned by their positions on one or several axes (time, height, width); with a cache, keys and values are
           quantised into it by the same call, and what it holds of them is read back.
  pages    a step of beam search or of drafts on a shared cache: sequences take over their parents' pages, get room for new tokens, pages
           that they share and write to are copied, and the tokens are taken back.
  compact  a pool of pages whose live ones are moved to its front.
  sparse   new tokens are written into the cache, complete pages get bounds of their keys, each query chooses pages by them, and attends
           to those and to the newest tokens.

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
        # one token for each of sixteen sequences during decoding: a call of a few microseconds
        {"name": "rotary_decode_16", "kind": "rotary", "tokens": 16, "axes": 1, "far": 1000, "turned": 128, "beside": False, "keep": False,
         "cached": True, "page": 64, "heads": 32, "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # a picture between two texts, positions in time, height and width, written as 4-bit codes with zero points
        {"name": "rotary_picture_777", "kind": "rotary", "tokens": 777, "axes": 3, "far": 3000, "turned": 128, "beside": False, "keep": True,
         "cached": True, "page": 16, "heads": 40, "kv_heads": 40, "dim": 128, "bits": 4, "symmetric": False, "type": "bf16"},
        # half of each head turned, neighbouring elements in pairs, far into a long text, and no cache yet
        {"name": "rotary_alone_4096", "kind": "rotary", "tokens": 4096, "axes": 1, "far": 1000000, "turned": 64, "beside": True, "keep": True,
         "cached": False, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # sixteen prompts of 1024 tokens, the prefill of the benchmark's layer; the turned keys are kept for the prompts' own attention
        {"name": "rotary_16x1024", "kind": "rotary", "tokens": 16384, "axes": 1, "far": 1024, "turned": 128, "beside": False, "keep": True,
         "cached": True, "page": 64, "heads": 32, "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # four beams of one request
        {"name": "pages_4_beams", "kind": "pages", "groups": 1, "beams": 4, "length": 1000, "apart": 90, "new": 1, "ragged": False, "page": 64,
         "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True},
        # seven requests whose drafts cross the ends of small pages
        {"name": "pages_7x3_drafts", "kind": "pages", "groups": 7, "beams": 3, "length": 5500, "apart": 301, "new": 27, "ragged": True, "page": 16,
         "kv_heads": 8, "dim": 128, "bits": 4, "symmetric": False},
        # many requests of eight beams each
        {"name": "pages_64x8_beams", "kind": "pages", "groups": 64, "beams": 8, "length": 1500, "apart": 200, "new": 1, "ragged": True, "page": 64,
         "kv_heads": 8, "dim": 128, "bits": 8, "symmetric": True},
        # half of the sequences of a pool have ended, and what is left is moved together
        {"name": "compact_4000", "kind": "compact", "pages": 4000, "seqs": 60, "live": 0.5, "page": 64, "kv_heads": 8, "dim": 128, "bits": 8,
         "symmetric": True},
        # one token of one user, 8000 tokens behind it
        {"name": "sparse_1x8000", "kind": "sparse", "seqs": 1, "drafts": 1, "context": 8000, "written": 1, "ragged": False, "chosen": 16, "first": 1,
         "last": 2, "page": 64, "heads": 32, "kv_heads": 32, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
        # drafts of some users with contexts of any length, small pages, grouped heads, 4-bit codes with zero points
        {"name": "sparse_tree_7x5", "kind": "sparse", "seqs": 7, "drafts": 5, "context": 20000, "written": 5, "ragged": True, "chosen": 100, "first": 2,
         "last": 4, "page": 16, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 4, "symmetric": False, "type": "bf16"},
        # a long document: its last 4000 tokens arrive, and the first token of the answer looks back on all of it
        {"name": "sparse_100000", "kind": "sparse", "seqs": 1, "drafts": 1, "context": 100000, "written": 4000, "ragged": False, "chosen": 64, "first": 1,
         "last": 4, "page": 64, "heads": 24, "kv_heads": 8, "dim": 64, "bits": 8, "symmetric": True, "type": "fp16"},
        # a batch of long conversations, one token each
        {"name": "sparse_16x32768", "kind": "sparse", "seqs": 16, "drafts": 1, "context": 32768, "written": 1, "ragged": False, "chosen": 48, "first": 1,
         "last": 4, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "symmetric": True, "type": "fp16"},
    ]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["rotary", "rotary", "pages", "compact", "sparse", "sparse"])
        kv_heads, group = rng.choice([(32, 1), (40, 1), (8, 4), (8, 8), (4, 7), (1, 16), (12, 1), (5, 3)])
        case = {"kind": kind, "page": rng.choice([16, 32, 64, 128]), "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]),
                "bits": rng.choice([8, 8, 4]), "symmetric": rng.random() < 0.5}
        if kind in ("rotary", "sparse"):
            case.update(heads=kv_heads * group, type=rng.choice(["fp16", "fp16", "bf16"]))
        if kind == "rotary":
            cached = rng.random() < 0.7
            case.update(tokens=_size(rng, 1, 16384), axes=rng.choice([1, 1, 2, 3]), far=_size(rng, 100, 1000000), turned=rng.choice([32, 64, case["dim"]]),
                        beside=rng.random() < 0.3, keep=not cached or rng.random() < 0.5, cached=cached)
        elif kind == "pages":
            case.update(groups=_size(rng, 1, 64), beams=_size(rng, 1, 12), length=_size(rng, 1, 8000), apart=_size(rng, 1, 600), new=_size(rng, 1, 64),
                        ragged=rng.random() < 0.6)
        elif kind == "compact":
            case.update(pages=_size(rng, 50, 8000), seqs=_size(rng, 2, 200), live=rng.choice([0.2, 0.5, 0.8]))
        else:
            drafts = 1 if rng.random() < 0.5 else _size(rng, 2, 64)
            case.update(seqs=_size(rng, 1, 32), drafts=drafts, context=_size(rng, 1, 65536), written=drafts if rng.random() < 0.6 else drafts + _size(rng, 1, 4000),
                        ragged=rng.random() < 0.5, chosen=_size(rng, 4, 128), first=rng.randint(0, 2), last=rng.randint(0, 2))
            if case["seqs"] * case["context"] * kv_heads * case["dim"] > 6e8:
                continue
            if case["seqs"] * drafts * case["heads"] * min(case["context"], case["chosen"] * case["page"]) * case["dim"] > 1.5e9:
                continue
        if kind in ("pages", "compact") and _pool(case)[0] * case["page"] * kv_heads * case["dim"] > 2e9:
            continue
        if _cost(case) <= most:
            return case


def _size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _lengths(case):
    """tokens of every group of beams, or in front of every sequence's drafts; ragged: the first is the longest, the others anything below"""
    n = case["groups"] if case["kind"] == "pages" else case["seqs"]
    longest = case["length"] if case["kind"] == "pages" else case["context"]
    rng = random.Random(n * 7919 + case["kv_heads"])
    return [longest] + [int((rng.random() ** 1.5 if case["ragged"] else 1.0) * longest) for _ in range(n - 1)]


def _row(case):
    """Bytes of a token and head in one of the cache's two halves: codes, scale and zero point"""
    return case["dim"] * case["bits"] / 8 + (4 if case["symmetric"] else 8)


def work(case):
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "rotary":
        # queries in and out, keys in, and out where they are kept; with a cache values in, both written, and read back
        elements = case["heads"] * 2 + kv * (1 + case["keep"]) + (3 * kv if case["cached"] else 0)
        return {"bytes": case["tokens"] * (2.0 * dim * elements + (4 * kv * _row(case) if case["cached"] else 0)),
                "flops": 3.0 * case["tokens"] * case["turned"] * (case["heads"] + kv)}
    if case["kind"] == "pages":
        parents, lens, each = _parents(case, 0), _lengths(case), case["beams"]
        shared = [s for s, p in enumerate(parents) if parents.count(p) > 1 and _beam(case, p, lens[p // each]) % page]
        pages, _ = _pool(case)
        return {"bytes": 4.0 * kv * page * _row(case) * len(shared) + 8.0 * len(parents) * _columns(case) + 4.0 * pages, "flops": 0.0}
    if case["kind"] == "compact":
        alive, owners = _survivors(case), _owners(case)
        count = sum(x in alive for x in owners)
        moved = sum(x in alive for x in owners[count:])
        return {"bytes": 4.0 * kv * page * _row(case) * moved + 12.0 * case["pages"], "flops": 0.0}
    read = scored = 0
    for c in _lengths(case):
        full = c // page
        scored += full
        read += case["drafts"] * (min(full, case["chosen"]) * page + c % page) + case["drafts"]
    new = len(_lengths(case)) * case["written"]
    rows = len(_lengths(case)) * case["drafts"]
    return {"bytes": 2.0 * kv * _row(case) * read + kv * (2.0 * dim + 4) * scored + 4.0 * dim * rows * case["heads"] + 2.0 * kv * new * (2 * dim + _row(case)),
            "flops": 4.0 * dim * case["heads"] * read}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 4e14)


# ------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _keys_and_values(gen, tokens, case):
    """rows as a model writes them: keys with a few channels far from zero, every token's values at a level of its own"""
    shape = (tokens, case["kv_heads"], case["dim"])
    channel = torch.exp(0.4 * torch.randn((1,) + shape[1:], generator=gen, device="cuda"))
    offset = 1.5 * (torch.rand((1,) + shape[1:], generator=gen, device="cuda") < 0.06)
    # a text's keys drift: pages differ in more than noise
    drift = torch.randn((tokens // 50 + 2,) + shape[1:], generator=gen, device="cuda").repeat_interleave(50, 0)[:tokens]
    k = (torch.randn(shape, generator=gen, device="cuda") * 0.8 + drift * 0.6) * channel + offset
    v = torch.randn(shape, generator=gen, device="cuda") * torch.exp(0.5 * torch.randn((tokens, 1, 1), generator=gen, device="cuda"))
    return k.to(_TYPES[case["type"]]), v.to(_TYPES[case["type"]])


# --- rotary

def _turns(case):
    """(revolutions per position, axis) of every pair of elements: neighbouring pairs share an axis, an axis has about as many as the others"""
    pairs = case["turned"] // 2
    i = torch.arange(pairs, dtype=torch.float64)
    return 10000.0 ** (-i / pairs) / (2 * math.pi), (i * case["axes"] / pairs).to(torch.int32)


def _positions(case):
    """[axes, tokens]: texts count on in all axes together, a picture's tokens stand still in time and walk over its rows and columns"""
    n, rng, rows, at = case["tokens"], random.Random(case["tokens"]), [], 0
    start = rng.randint(0, case["far"])
    while len(rows) < n:
        text, wide = rng.randint(1, 200), rng.randint(1, 24)
        rows += [(start + at + i,) * 3 for i in range(text)]
        at += text
        if case["axes"] > 1:
            rows += [(start + at, start + at + i // wide, start + at + i % wide) for i in range(wide * rng.randint(1, 24))]
            at += wide
    return _ints(rows[:n]).T[: case["axes"]].contiguous()


def _prepare_rotary(case, seed):
    gen, n, dim, dtype = _gen(seed), case["tokens"], case["dim"], _TYPES[case["type"]]
    k, v = _keys_and_values(gen, n, case)
    q = torch.randn((n, case["heads"], dim), generator=gen, device="cuda").to(dtype)
    qkv = torch.cat([q.view(n, -1), k.view(n, -1), v.view(n, -1)], 1)  # slices of one fused result
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([x.shape[1] * dim for x in (q, k, v)], 1))
    turns, axis = _turns(case)
    pages = (n + case["page"] - 1) // case["page"] + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = (order[at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)
    state = {"case": case, "q": q, "k": k, "v": v, "turns": turns.cuda(), "axis": axis.cuda(), "positions": _positions(case), "slots": slots}
    empty = lambda *shape: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if own:
        binding = _binding()
        state["rotary"] = binding.Rotary(turns, axis, interleaved=case["beside"])
        state["q_out"], state["k_out"] = empty(n, case["heads"], dim), empty(n, case["kv_heads"], dim) if case["keep"] else None
        if case["cached"]:
            state["cache"] = binding.KvCache(pages, case["page"], case["kv_heads"], dim, bits=case["bits"], symmetric=case["symmetric"])
            state["back"] = (empty(n, case["kv_heads"], dim), empty(n, case["kv_heads"], dim))
    elif case["cached"]:
        state.update(_empty_cache(case, pages))
    return state


# --- pages

def _beam(case, s, length):
    """Tokens of sequence s, of a group whose first beam has `length`"""
    return max(0, length - (s % case["beams"]) * (7 if case["ragged"] else 0))


def _columns(case):
    return (case["length"] + case["new"]) // case["page"] + 2


def _pool(case):
    """(pages of the pool, of each sequence's own)"""
    if case["kind"] == "compact":
        return case["pages"], 0
    lens, page = _lengths(case), case["page"]
    seqs = case["groups"] * case["beams"]
    own_pages = sum(min(x, case["apart"]) // page + 2 for x in lens) * case["beams"]
    return sum(x // page + 1 for x in lens) + own_pages + seqs * (case["new"] // page + 3), seqs


def _parents(case, seed):
    """of every sequence: beams of a group go on from any of them, better ones more often"""
    rng, each = random.Random(seed * 31 + case["groups"]), case["beams"]
    return [g * each + int(rng.random() ** 1.5 * each) for g in range(case["groups"]) for _ in range(each)]


def _prepare_pages(case, seed):
    lens, page, each = _lengths(case), case["page"], case["beams"]
    pages, seqs = _pool(case)
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    table, lengths = [[-1] * _columns(case) for _ in range(seqs)], []
    for g, length in enumerate(lens):
        prefix = [free.pop() for _ in range(max(0, length - case["apart"]) // page)]  # pages that all beams of the group share
        for s in range(g * each, (g + 1) * each):
            mine = _beam(case, s, length)
            used = (mine + page - 1) // page
            table[s][:used] = (prefix + [free.pop() for _ in range(max(0, used - len(prefix)))])[:used]
            lengths.append(mine)
    return _pool_state(case, seed, table, lengths, {"parents": _ints(_parents(case, seed)), "more": _ints([case["new"]] * seqs),
                                                    "less": _ints([-case["new"]] * seqs), "rows": seqs * case["new"]})


def _owners(case):
    """which sequence each page of the pool belongs to"""
    rng = random.Random(case["pages"] * 131 + case["seqs"])
    return [int(rng.random() ** 1.3 * case["seqs"]) for _ in range(case["pages"])]


def _survivors(case):
    rng = random.Random(case["pages"] + 17 * case["seqs"])
    return {s for s in range(case["seqs"]) if rng.random() < case["live"]}


def _prepare_compact(case, seed):
    rng, owners, alive = random.Random(seed), _owners(case), _survivors(case)
    table = [[] for _ in range(case["seqs"])]
    for p, s in enumerate(owners):
        if s in alive:
            table[s].append(p)
    most = max(1, max(len(r) for r in table))
    for r in table:
        rng.shuffle(r)
    lengths = [max(0, len(r) * case["page"] - rng.randint(0, case["page"] - 1)) for r in table]
    state = _pool_state(case, seed, [r + [-1] * (most - len(r)) for r in table], lengths, {})
    state["before"] = (state["table"].clone(), state["refs"].clone())
    return state


def _pool_state(case, seed, table, lengths, more):
    """a table of pages with what a cache holds in them, by its bytes: a page's are the same in either form"""
    gen, (pages, _) = _gen(seed), _pool(case)
    table, lengths = _ints(table), _ints(lengths)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
    codes = case["page"] * case["kv_heads"] * case["dim"] * case["bits"] // 8
    scales = case["page"] * case["kv_heads"] * (1 if case["symmetric"] else 2)
    held = [torch.randint(0, 256, (pages, codes), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
    held += [torch.rand((pages, scales), generator=gen, device="cuda") for _ in range(2)]
    state = {"case": case, **more}
    if own:
        binding = _binding()
        state["pages"] = binding.PageTable(pages, case["page"], table.shape[0], table.shape[1])
        cache = binding.KvCache(pages, case["page"], case["kv_heads"], case["dim"], bits=case["bits"], symmetric=case["symmetric"])
        state["cache"], to = cache, (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)
        for a, b in zip(to, held):
            a.copy_(b.flatten())
        held = [a.view(pages, -1) for a in to]
        for a, b in zip((state["pages"].table, state["pages"].lengths, state["pages"].refs), (table, lengths, refs)):
            a.copy_(b)
        table, lengths, refs = state["pages"].table, state["pages"].lengths, state["pages"].refs
    state.update(table=table, lengths=lengths, refs=refs, held=held)
    return state


# --- sparse

def _ancestors(case, seed):
    """For every draft the bits of the drafts that it sees: its ancestors in a random tree, and itself"""
    rng, masks = random.Random(seed), []
    for _ in range(case["seqs"]):
        seen = []
        for i in range(case["drafts"]):
            seen.append((1 << i) | (seen[rng.randint(max(0, i - 6), i - 1)] if i else 0))
        masks += seen
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()


def _sparse_inputs(case, seed):
    """(q, k, v, lengths, page table, slots of all tokens, which of them the call writes)"""
    gen, page, lens, new = _gen(seed), case["page"], _lengths(case), case["drafts"]
    each = (max(lens) + new + page - 1) // page
    order = torch.randperm(case["seqs"] * each + 3, generator=gen, device="cuda")[: case["seqs"] * each]
    table = order.to(torch.int32).view(case["seqs"], each)
    count = torch.tensor([c + new for c in lens], device="cuda")
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), count)
    at = torch.arange(int(count.sum()), device="cuda") - (count.cumsum(0) - count)[seq]
    slots = (table[seq, at // page] * page + at % page).to(torch.int32)
    fresh = at >= count[seq] - case["written"]
    k, v = _keys_and_values(gen, int(count.sum()), case)
    q = torch.randn((case["seqs"] * new, case["heads"], case["dim"]), generator=gen, device="cuda").to(_TYPES[case["type"]])
    return q, k, v, lens, table, slots, fresh


def _prepare_sparse(case, seed):
    q, k, v, lens, table, slots, fresh = _sparse_inputs(case, seed)
    pages, dim = table.numel() + 3, case["dim"]
    context, starts = _ints(lens), _ints([case["drafts"] * s for s in range(case["seqs"] + 1)])
    mask = _ancestors(case, seed)
    state = {"case": case, "q": q, "k": k[fresh], "v": v[fresh], "written": slots[fresh], "table": table, "context": context, "mask": mask}
    earlier = (k[~fresh], v[~fresh], slots[~fresh])
    if own:
        binding = _binding()
        cache = binding.KvCache(pages, case["page"], case["kv_heads"], dim, bits=case["bits"], symmetric=case["symmetric"], bounds=True)
        if earlier[2].numel():
            cache.append(*earlier)
            cache.bound(earlier[2])
        state["cache"] = cache
        state["call"] = binding.SparseAttention(q, cache, table, context, starts, case["drafts"], max(lens), case["chosen"], first=case["first"],
                                                last=case["last"], mask=mask, scale=dim ** -0.5, out=torch.empty_like(q))
        return state
    state.update(_empty_cache(case, pages))
    state["bound_codes"] = torch.zeros((pages, case["kv_heads"], 2, dim), dtype=torch.int8, device="cuda")
    state["bound_scales"] = torch.zeros((pages, case["kv_heads"]), device="cuda")
    if earlier[2].numel():
        _write(state, torch.stack(earlier[:2]), earlier[2])
        _bound(state, earlier[2])
    return state


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "pages": _prepare_pages, "compact": _prepare_compact, "sparse": _prepare_sparse}[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------------- the plain forms

def _empty_cache(case, pages):
    shape = (2, pages * case["page"], case["kv_heads"])
    return {"codes": torch.zeros(shape + (case["dim"],), dtype=torch.int16, device="cuda"), "scales": torch.ones(shape + (1,), device="cuda"),
            "zeros": torch.zeros(shape + (1,), device="cuda")}


def _codes(x, bits, symmetric):
    """(codes, scale, zero point) of rows x: a quotient by a plain number is a product here, not always rounded alike"""
    top = 2 ** (bits - 1) - 1
    if symmetric:
        high = x.abs().amax(-1, keepdim=True)
        scale = (high / torch.full_like(high, top)).clamp(1e-5, 1e4)
        return torch.round(x / scale).clamp(-top - 1, top), scale, torch.zeros_like(scale)
    low = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - low) / torch.full_like(low, 2 * top + 1)).clamp(1e-5, 1e4)
    zero = torch.round((-low / scale).clamp(-1e4, 1e4))
    return (torch.round(x / scale) + zero).clamp(0, 2 * top + 1), scale, zero


def _write(state, rows, slots):
    """Quantises rows [2, tokens, heads, dim] per token and head and writes them at their slots"""
    code, scale, zero = _codes(rows.float(), state["case"]["bits"], state["case"]["symmetric"])
    at = slots.long()
    state["codes"][:, at], state["scales"][:, at], state["zeros"][:, at] = code.to(torch.int16), scale, zero


def _values(state, slots):
    """What the cache holds at these slots: keys and values in 32 bits"""
    at = slots.long()
    return (state["codes"][:, at].float() - state["zeros"][:, at]) * state["scales"][:, at]


def _turn(state, x):
    """x [tokens, heads, dim] turned by its positions, in 64 bits: a code beside a border goes by the last one"""
    case, pairs = state["case"], state["case"]["turned"] // 2
    turn = state["positions"].double()[state["axis"].long()].T * state["turns"]
    angle = (turn - torch.round(turn)).mul_(2 * math.pi)[:, None]
    cos, sin, y = torch.cos(angle), torch.sin(angle), x.double()
    part = y[..., : 2 * pairs]
    a, b = (part[..., 0::2], part[..., 1::2]) if case["beside"] else (part[..., :pairs], part[..., pairs:])
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([first, second], -1).flatten(2) if case["beside"] else torch.cat([first, second], -1)
    return torch.cat([turned, y[..., 2 * pairs:]], -1).to(x.dtype)


def _run_rotary(state):
    q, k = _turn(state, state["q"]), _turn(state, state["k"])
    out = [q] + ([k] if state["case"]["keep"] else [])
    if state["case"]["cached"]:
        _write(state, torch.stack([k, state["v"]]), state["slots"])
        out += list(_values(state, state["slots"]).to(q.dtype))
    return tuple(out)


def _fork(state, parents):
    """Every sequence takes over its parent's pages"""
    old, new = state["table"], state["table"][parents.long()]
    change = torch.zeros_like(state["refs"])
    for entries, by in ((old, -1), (new, 1)):
        change.index_add_(0, entries.flatten().clamp(min=0).long(), ((entries >= 0).int() * by).flatten())
    state["refs"] += change
    state["lengths"].copy_(state["lengths"][parents.long()])
    old.copy_(new)


def _extend(state, counts, rows):
    """Room for counts[s] tokens more (fewer, where it is negative).  Free pages go to the sequences in order, lowest first; a sequence
    that would write into a page that others hold too gets one of its own, to copy it to."""
    table, lengths, refs, page = state["table"], state["lengths"].long(), state["refs"], state["case"]["page"]
    seqs, columns = table.shape
    counts = counts.long()
    used = lambda n: (n + page - 1) // page  # noqa: E731
    grow, shrink = counts.clamp(min=0), torch.minimum((-counts).clamp(min=0), lengths)
    fits = used(lengths + grow) <= columns
    last = table.gather(1, (lengths // page).clamp(max=columns - 1)[:, None])[:, 0]
    copied = (grow > 0) & (lengths % page > 0) & (refs[last.clamp(min=0).long()] > 1)
    need = (used(lengths + grow) - used(lengths) + copied) * ((grow > 0) & fits)
    ends = need.cumsum(0)
    free = torch.argsort((refs != 0).int(), stable=True)  # the free ones first, in order
    given = (grow > 0) & fits & ((need == 0) | (ends <= (refs == 0).sum()))
    copied = copied & given
    granted = torch.where(given, grow, 0) - shrink
    # the pages: number r of those given out goes to the sequence whose span of them it lies in
    r = torch.arange(free.numel(), device="cuda")
    to = torch.searchsorted(ends, r, right=True).clamp(max=seqs - 1)
    mine = (r < (need * given).sum()) & given[to]
    column = used(lengths)[to] - copied[to].long() + r - (ends - need)[to]
    copies = torch.full((seqs, 2), -1, dtype=torch.int32, device="cuda")
    copies[:, 0] = torch.where(copied, last, -1)
    padded = torch.cat([table, table[:, :1]], 1)  # (a column beyond the last, for what goes nowhere)
    padded[to, torch.where(mine, column, columns)] = free.to(torch.int32)
    table.copy_(padded[:, :columns])
    copies[:, 1] = torch.where(copied, table.gather(1, (lengths // page).clamp(max=columns - 1)[:, None])[:, 0], -1)
    change = torch.zeros_like(refs).index_add_(0, free, mine.int()).index_add_(0, last.clamp(min=0).long(), -copied.int())
    after = lengths + granted
    gone = (torch.arange(columns, device="cuda") >= used(after)[:, None]) & (table >= 0)
    change.index_add_(0, table.clamp(min=0).flatten().long(), -gone.int().flatten())
    refs += change
    table.masked_fill_(gone, -1)
    state["lengths"].copy_(after)
    starts = torch.cat([grow[:1] * 0, grow.cumsum(0)])
    row = torch.arange(rows, device="cuda")
    s = torch.searchsorted(starts[1:], row, right=True).clamp(max=seqs - 1)
    place = (after - granted)[s] + row - starts[s]
    slots = table[s, (place // page).clamp(0, columns - 1)] * page + place % page
    slots = torch.where((row < starts[-1]) & given[s], slots, -1)
    return slots.to(torch.int32), starts.to(torch.int32), granted.to(torch.int32), copies


def _copy_pages(state, pairs):
    pairs = pairs[pairs[:, 0] >= 0].long()
    for a in state["held"]:
        a[pairs[:, 1]] = a[pairs[:, 0]]


def _compact(state):
    """The last live pages move into the first free ones; returns (from, to) of each"""
    live, n = state["refs"] > 0, state["refs"].numel()
    at, count = torch.arange(n, device="cuda"), live.sum()
    hole, mover = ~live & (at < count), live & (at >= count)
    moves = torch.full((n // 2 + 1, 2), -1, dtype=torch.int32, device="cuda")
    for side, which in ((1, hole), (0, mover)):
        moves[torch.where(which, which.cumsum(0) - 1, n // 2), side] = at.to(torch.int32)
    moves = torch.where(torch.arange(n // 2, device="cuda")[:, None] < mover.sum(), moves[:-1], -1)
    new = at.to(torch.int32)
    rank = (mover.cumsum(0) - 1).clamp(0, max(0, n // 2 - 1))
    new = torch.where(mover, moves[rank, 1], new) if n > 1 else new
    table, refs = state["table"], state["refs"].clone()
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], -1))
    state["refs"].zero_().index_add_(0, new.long(), refs)
    return moves


def _run_pages(state):
    _fork(state, state["parents"])
    given = _extend(state, state["more"], state["rows"])
    _copy_pages(state, given[3])
    table = state["table"].clone()  # as the step's attention reads it
    _extend(state, state["less"], 0)
    return (table,) + given + (state["table"], state["lengths"], state["refs"]) + tuple(state["held"])


def _run_compact(state):
    for a, b in zip((state["table"], state["refs"]), state["before"]):
        a.copy_(b)
    moves = _compact(state)
    _copy_pages(state, moves)
    return (moves, state["table"], state["refs"]) + tuple(state["held"])


def _bound(state, slots):
    """Bounds of the keys of every page whose last token is among these: largest and smallest of every channel, in 8 bits with one scale"""
    page = state["case"]["page"]
    pages = slots[slots % page == page - 1].long() // page
    at = (pages[:, None] * page + torch.arange(page, device="cuda")).flatten()
    keys = ((state["codes"][0, at].float() - state["zeros"][0, at]) * state["scales"][0, at]).unflatten(0, (-1, page))
    if pages.numel():
        code, scale, _ = _codes(torch.cat([keys.amax(1), keys.amin(1)], -1), 8, True)
        state["bound_codes"][pages] = code.view(code.shape[:2] + (2, -1)).to(torch.int8)
        state["bound_scales"][pages] = scale[..., 0]


def _select(state):
    """[rows, kv heads, chosen]: the pages that each query's heads of one key head look at, by a bound of their scores, in order; -1 behind them"""
    case, page = state["case"], state["case"]["page"]
    seqs, n, kv = case["seqs"], case["drafts"], case["kv_heads"]
    code, scale, _ = _codes(state["q"].float(), 8, True)
    both = torch.cat([code.clamp(min=0), code.clamp(max=0)], -1).view(seqs, n, kv, -1, 2 * case["dim"])
    columns = state["table"].shape[1]
    pages = state["table"].long().flatten()
    bounds = state["bound_codes"][pages].float().view(seqs, columns, kv, -1).permute(0, 2, 3, 1).contiguous()
    dot = torch.matmul(both.transpose(1, 2).flatten(2, 3), bounds)  # whole numbers below 2^24
    score = (dot.view(seqs, kv, n, -1, columns) * scale.view(seqs, n, kv, -1, 1).transpose(1, 2)).amax(3)
    score = score * state["bound_scales"][pages].view(seqs, columns, kv, 1).permute(0, 2, 3, 1)
    full = (state["context"].long() // page)[:, None, None, None]
    at = torch.arange(columns, device="cuda")
    score = score.masked_fill((at < case["first"]) | (at >= full - case["last"]), math.inf).masked_fill(at >= full, -math.inf)
    chosen = min(case["chosen"], columns)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :chosen]
    best = torch.sort(torch.where(best < full, best, columns), dim=-1)[0]
    best = torch.where(best < columns, best, -1).permute(0, 2, 1, 3).reshape(seqs * n, kv, chosen)
    return torch.nn.functional.pad(best, (0, case["chosen"] - chosen), value=-1).to(torch.int32)


def _run_sparse(state):
    case, page, dim = state["case"], state["case"]["page"], state["case"]["dim"]
    seqs, n, kv = case["seqs"], case["drafts"], case["kv_heads"]
    _write(state, torch.stack([state["k"], state["v"]]), state["written"])
    _bound(state, state["written"])
    blocks = _select(state)
    # places: those of the pages chosen, then from the end of the last complete page to the last draft
    context = state["context"].long().repeat_interleave(n)[:, None, None]
    inside = (blocks.long()[..., None] * page + torch.arange(page, device="cuda")).flatten(2)
    behind = (context // page * page + torch.arange(page + n - 1, device="cuda")).expand(-1, kv, -1)
    place = torch.cat([inside, behind], 2)
    draft = place - context
    named = (state["mask"][:, None, None] >> draft.clamp(0, 63)) & 1
    visible = (place >= 0) & ((draft < 0) | ((draft < n) & (named == 1)))
    table = state["table"].repeat_interleave(n, 0)
    row = torch.arange(seqs * n, device="cuda")[:, None, None]
    at = table[row, (place // page).clamp(0, table.shape[1] - 1)].long() * page + place % page
    head = torch.arange(kv, device="cuda")[:, None]
    k, v = ((state["codes"][i][at, head].float() - state["zeros"][i][at, head]) * state["scales"][i][at, head] for i in range(2))
    q = state["q"].float().view(seqs * n, kv, -1, dim)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5).masked_fill_(~visible[:, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s, v) / total.masked_fill_(total == 0, 1)
    return blocks, out.view(state["q"].shape).to(state["q"].dtype), state["bound_codes"], state["bound_scales"]


# ------------------------------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind == "rotary" and not state["case"]["cached"]:
            return state["rotary"].apply(state["q"], state["k"], state["positions"], out=(state["q_out"], state["k_out"]))
        if kind == "rotary":
            turned = state["cache"].append_rotated(state["rotary"], state["q"], state["k"], state["v"], state["positions"], state["slots"],
                                                   q_out=state["q_out"], k_out=state["k_out"])
            return tuple(x for x in turned if x is not None) + tuple(state["cache"].read(state["slots"], out=state["back"]))
        if kind == "pages":
            pages = state["pages"]
            pages.fork(state["parents"])
            given = pages.extend(state["more"], state["rows"])
            state["cache"].copy_pages(given.copies)
            table = pages.table.clone()
            pages.extend(state["less"], 0)
            return (table, given.slots, given.starts, given.granted, given.copies, pages.table, pages.lengths, pages.refs) + tuple(state["held"])
        if kind == "compact":
            pages = state["pages"]
            for a, b in zip((pages.table, pages.refs), state["before"]):
                a.copy_(b)
            moves = pages.compact()
            state["cache"].copy_pages(moves)
            return (moves, pages.table, pages.refs) + tuple(state["held"])
        state["cache"].append(state["k"], state["v"], state["written"])
        state["cache"].bound(state["written"])
        out = state["call"].run()
        return state["call"].blocks, out, state["cache"].bound_codes, state["cache"].bound_scales
    return {"rotary": _run_rotary, "pages": _run_pages, "compact": _run_compact, "sparse": _run_sparse}[kind](state)


# ------------------------------------------------------------------------------------------------- the same in 64 bits

def _held(x, bits, symmetric):
    """What a cache of `bits` bits holds of rows x.  The format keeps scales in 32 bits, and the quotient that a code is rounded
    from is one of 32 bits, which decides the ties; everything else is exact"""
    x, held = x.double(), lambda a: a.float().double()
    levels = 2 ** bits - 1
    if symmetric:
        half = (levels - 1) / 2
        step = held((x.abs().amax(-1, keepdim=True) / half).clamp(1e-5, 1e4))
        return held(x / step).round().clamp(-half - 1, half), step, torch.zeros_like(step)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = held((held(high - low) / levels).clamp(1e-5, 1e4))
    shift = held(-low / step).clamp(-1e4, 1e4).round()
    return (held(x / step).round() + shift).clamp(0, levels) - shift, step, shift


def _exact_rotary(case, seed):
    state = _prepare_rotary({**case, "cached": False}, seed)
    pairs, out = case["turned"] // 2, []
    angle = 2 * math.pi * torch.frac(state["positions"][state["axis"].long()].double() * state["turns"][:, None])
    unit = torch.polar(torch.ones_like(angle), angle).T[:, None]  # [tokens, 1, pairs]
    for x in (state["q"], state["k"]):
        y = x.double().clone()
        where = torch.arange(pairs, device="cuda")
        first, second = (2 * where, 2 * where + 1) if case["beside"] else (where, where + pairs)
        z = torch.complex(y[..., first], y[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    q, k = out
    answer = [q] + ([k] if case["keep"] else [])
    if case["cached"]:  # the cache's rows are the keys as they are kept, rounded to their type
        for x in (k.to(_TYPES[case["type"]]), state["v"]):
            code, step, _ = _held(x, case["bits"], case["symmetric"])
            answer.append(code * step)
    return tuple(answer)


def _exact_sparse(case, seed):
    q, k, v, lens, _, _, _ = _sparse_inputs(case, seed)
    n, kv, page, dim = case["drafts"], case["kv_heads"], case["page"], case["dim"]
    group, masks = case["heads"] // kv, [m % (1 << 64) for m in _ancestors(case, seed).tolist()]
    out = torch.zeros_like(q, dtype=torch.float64)
    blocks = torch.full((case["seqs"] * n, kv, case["chosen"]), -1, dtype=torch.int32, device="cuda")
    q_code, q_step, _ = _held(q, 8, True)
    single = lambda a: a.float().double()  # noqa: E731
    first = 0
    for s, c in enumerate(lens):
        (ku, ks, _), (vu, vs, _) = (_held(x[first:first + c + n], case["bits"], case["symmetric"]) for x in (k, v))
        keys, values, full = ku * ks, vu * vs, c // page
        # what the cache's keys are in 32 bits bounds the pages
        ends = single(keys[:full * page]).unflatten(0, (full, page)) if full else keys[:0].view(0, page, kv, dim)
        if full:
            b_code, b_step, _ = _held(torch.cat([ends.amax(1), ends.amin(1)], -1), 8, True)
        for i in range(s * n, (s + 1) * n):
            for h in range(kv):
                mine = slice(h * group, (h + 1) * group)
                picked = list(range(full))
                if full > case["chosen"]:
                    up, down = q_code[i, mine].clamp(min=0), q_code[i, mine].clamp(max=0)
                    dot = up @ b_code[:, h, :dim].T + down @ b_code[:, h, dim:].T
                    score = single(single(dot * q_step[i, mine]).amax(0) * b_step[:, h, 0])
                    score[:case["first"]] = math.inf
                    score[full - case["last"]:] = math.inf
                    picked = sorted(torch.sort(score, descending=True, stable=True)[1][:case["chosen"]].tolist())
                blocks[i, h, :len(picked)] = torch.tensor(picked, dtype=torch.int32, device="cuda")
                sees = torch.zeros(c + n, dtype=torch.bool, device="cuda")
                sees[:full * page].view(full, page)[picked] = True
                sees[full * page:c] = True
                sees[c:] = torch.tensor([bool(masks[i] >> j & 1) for j in range(n)], device="cuda")
                weight = torch.softmax(q[i, mine].double() @ keys[sees, h].T * dim ** -0.5, -1)
                out[i, mine] = weight @ values[sees, h]
        first += c + n
    return blocks, out, None, None  # (the bounds are whole numbers, and scales that the choice of blocks went by)


def exact(case, seed):
    if case["kind"] == "rotary":
        return _exact_rotary(case, seed)
    if case["kind"] == "sparse" and case["seqs"] * case["drafts"] * case["kv_heads"] <= 3000:
        return _exact_sparse(case, seed)
    return None  # whole numbers and bytes that are moved
