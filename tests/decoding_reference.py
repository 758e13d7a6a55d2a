"""Rotary positions, pages of sequences and the choice of pages in plain Python and numpy, from the formulas of the header: test code."""
import numpy as np
import torch

from attention_reference import attend, cache_contents

def turned(x, positions, turns, axis, interleaved):
    """(x [tokens, heads, dim] turned, in 64 bits, and the error allowed of a result of x's type): the product of position and revolutions in
    fp64 is the formula's own; cosine, sine and the sums are off by a few 2^-53; roundings to fp32 and to the type by half a step each"""
    pairs = turns.numel()
    y = x.cpu().double().numpy().copy()
    t = positions.cpu().numpy().astype(np.float64)[axis.numpy()].T * turns.numpy()  # [tokens, pairs]
    angle = (2 * np.pi * (t - np.rint(t)))[:, None, :]
    first, second = (np.arange(pairs) * 2, np.arange(pairs) * 2 + 1) if interleaved else (np.arange(pairs), np.arange(pairs) + pairs)
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    size = np.zeros_like(y)
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    half, tiny = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}[x.dtype]
    allowed = np.abs(y) * (half + 2.0 ** -23) + size * 2.0 ** -49 + tiny
    return torch.from_numpy(y), torch.from_numpy(np.where(size == 0, 0, allowed)) if pairs * 2 < x.shape[-1] else torch.from_numpy(allowed)


class Pages:
    """The table of pages as the header states it, sequence by sequence"""

    def __init__(self, num_pages, size, seqs, most):
        self.size, self.most, self.refs = size, most, [0] * num_pages
        self.of, self.lengths = [[] for _ in range(seqs)], [0] * seqs

    def table(self):
        return [p + [-1] * (self.most - len(p)) for p in self.of]

    def count(self):
        self.refs = [0] * len(self.refs)
        for pages in self.of:
            for p in pages:
                self.refs[p] += 1

    def fork(self, parents):
        of, lengths, seqs = self.of, self.lengths, range(len(self.of))
        self.of = [list(of[p]) if p in seqs else [] for p in parents]
        self.lengths = [lengths[p] if p in seqs else 0 for p in parents]
        self.count()

    def extend(self, counts, rows):
        free = [p for p, n in enumerate(self.refs) if n == 0]
        need = []
        for s, c in enumerate(counts):
            n = self.lengths[s]
            wanted = -(-(n + max(c, 0)) // self.size)
            copied = c > 0 and n % self.size > 0 and wanted <= self.most and self.refs[self.of[s][n // self.size]] > 1
            need.append((wanted - len(self.of[s]) + copied if c > 0 and wanted <= self.most else 0, copied, wanted <= self.most))
        slots, starts, granted, copies, taken = [], [0], [], [], 0
        for s, c in enumerate(counts):
            pages, copied, fits = need[s]
            taken += pages
            starts.append(starts[-1] + max(c, 0))
            pair = [-1, -1]
            if c <= 0:
                less = min(-c, self.lengths[s])
                granted.append(-less)
            elif not fits or (pages and taken > len(free)):
                granted.append(0)
                slots += [-1] * c
            else:
                mine = free[taken - pages:taken]
                if copied:
                    at = self.lengths[s] // self.size
                    pair = [self.of[s][at], mine[0]]
                    self.of[s][at] = mine[0]
                    mine = mine[1:]
                self.of[s] += mine
                granted.append(c)
                slots += [self.of[s][t // self.size] * self.size + t % self.size for t in range(self.lengths[s], self.lengths[s] + c)]
            copies.append(pair)
        for s, g in enumerate(granted):
            self.lengths[s] += g
            self.of[s] = self.of[s][:-(-self.lengths[s] // self.size)]
        self.count()
        return (slots + [-1] * rows)[:rows], starts, granted, copies

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        self.of = [[to.get(p, p) for p in pages] for pages in self.of]
        self.count()
        half = len(self.refs) // 2
        return ([[a, b] for a, b in zip(movers, holes)] + [[-1, -1]] * half)[:half]


def signed_rows(x):
    """(codes, scale) of rows x [..., n] as symmetric rows of 8 bits, every step an fp32 operation"""
    x = np.asarray(x, np.float32)
    scale = np.clip(np.abs(x).max(-1, keepdims=True) / np.float32(127), np.float32(1e-5), np.float32(1e4))
    return np.clip(np.rint(x / scale), -128, 127).astype(np.int64), scale[..., 0]


def bounds_of(keys):
    """(codes [..., 2, dim], scale) of pages of keys [..., size, dim] in fp32"""
    both = np.concatenate([keys.max(-2), keys.min(-2)], -1)
    codes, scale = signed_rows(both)
    return codes.reshape(codes.shape[:-1] + (2, -1)), scale


def choice(q, bound_codes, bound_scales, pages, num_pages, full, first, last, count):
    """The pages of one row and key head: q [group, dim], bounds of all pages of the cache for that head, the sequence's pages"""
    if full <= count:
        return list(range(full)) + [-1] * (count - full)
    codes, scale = signed_rows(q.float().numpy())
    pages = np.asarray(pages[:full])
    there = (pages >= 0) & (pages < num_pages)
    bound = bound_codes[np.where(there, pages, 0)]
    dot = np.maximum(codes, 0) @ bound[:, 0].T + np.minimum(codes, 0) @ bound[:, 1].T
    score = (dot.astype(np.float32) * scale[:, None]).max(0) * bound_scales[np.where(there, pages, 0)]
    score = np.where(there, score, -np.inf)
    at = np.arange(full)
    score[(at < first) | (at >= full - last)] = np.inf
    return sorted(np.argsort(-score, kind="stable")[:count].tolist())


def sparse_reference(q, cache, table, context, lens, mask, scale, blocks):
    """Attention to listed pages and to what stands behind the complete ones, in 64 bits, with the error that the kernel may make: scores
    are taken from codes and zero points apart, and so are the second product's sums"""
    kc, vc, (ks, kz), (vs, vz) = cache_contents(cache)
    size, pages, kv = cache.desc.page_size, cache.desc.num_pages, cache.desc.kv_heads
    half, group = 2 ** (cache.desc.bits - 1), q.shape[1] // kv
    out, allowed = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    row = 0
    for s, n in enumerate(lens):
        places = table.shape[1] * size
        c = min(max(context[s], 0), places)
        full, m = c // size, min(c + n, places)
        for i in range(n):
            bits = (1 << (i + 1)) - 1 if mask is None else int(mask[row]) % (1 << 64)
            newest = [t for t in range(full * size, m) if t < c or bits >> (t - c) & 1]
            for g in range(kv):
                at = np.array([b * size + t for b in blocks[row][g] if 0 <= b < full for t in range(size)] + newest, dtype=np.int64)
                page = np.asarray(table[s])[at // size] if at.size else at
                at, page = at[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
                slot = page * size + at % size
                k, v = ((x[slot, g] - z[slot, g, None].astype(np.float64)) * w[slot, g, None].astype(np.float64) for x, z, w in ((kc, kz, ks), (vc, vz, vs)))
                heads = slice(g * group, (g + 1) * group)
                spread = (np.abs(vc[slot, g] - half) * 2.0 ** -8 + np.abs(vz[slot, g, None] - half) * 2.0 ** -8 + np.abs(vc[slot, g] - vz[slot, g, None])) * vs[slot, g, None]
                top = vs[slot, g].max() / max(1e-30, vs[slot, g].min()) if slot.size else 1.0
                k_spread = torch.from_numpy((np.abs(kc[slot, g] - half) + np.abs(kz[slot, g, None] - half)) * ks[slot, g, None].astype(np.float64))
                rows = q[row, heads].cpu()
                seen = torch.ones((group, slot.size), dtype=torch.bool)
                out[row, heads], some = attend(rows, torch.from_numpy(k), torch.from_numpy(v), seen, scale, q.dtype, torch.from_numpy(spread), top)
                if slot.size:
                    more = (rows.double().abs() @ k_spread.T * scale).amax(-1, keepdim=True) * (q.shape[2] + 8) * 2.0 ** -23
                    some = some + more * (torch.from_numpy(spread).amax(0)[None, :])
                allowed[row, heads] = some
            row += 1
    return out, allowed
