"""Attention on a quantised cache in 64 bits and plain indexing, on the CPU, with the error that the kernels may make: test code."""
import math

import numpy as np
import torch


def load_abq_attention():
    """The package directory name is not a Python identifier, so load the binding by path."""
    import importlib.util
    import os
    import sys

    from conftest import PKG, load_abq_gemm
    load_abq_gemm()
    if "abq_attention" not in sys.modules:
        spec = importlib.util.spec_from_file_location("abq_attention", os.path.join(PKG, "abq_attention.py"))
        module = importlib.util.module_from_spec(spec)
        sys.modules["abq_attention"] = module
        spec.loader.exec_module(module)
    return sys.modules["abq_attention"]


def quantise(x, bits, symmetric):
    """(unsigned codes, scale, zero point) of rows x [..., dim], every step an fp32 operation as the format states it"""
    x = x.float().numpy().astype(np.float32)
    half = np.float32(2 ** (bits - 1))
    with np.errstate(invalid="ignore", over="ignore"):
        if symmetric:
            scale = np.clip(np.abs(x).max(-1, keepdims=True) / (half - 1), np.float32(1e-5), np.float32(1e4))
            zero = np.full_like(scale, half)
            code = np.clip(np.rint(x / scale), -half, half - 1) + half
        else:
            low = x.min(-1, keepdims=True)
            scale = np.clip((x.max(-1, keepdims=True) - low) / (2 * half - 1), np.float32(1e-5), np.float32(1e4))
            zero = np.rint(np.clip(-low / scale, np.float32(-1e4), np.float32(1e4)))
            code = np.clip(np.rint(x / scale) + zero, 0, 2 * half - 1)
    return code.astype(np.int64), scale[..., 0], zero[..., 0]


def cache_contents(cache):
    """(k codes, v codes [slots, heads, dim], (k scale, k zero), (v scale, v zero) [slots, heads]) by the stated layout"""
    d = cache.desc
    pages, heads, size, dim, row = d.num_pages, d.kv_heads, d.page_size, d.head_dim, d.head_dim * d.bits // 8
    k = cache.k_codes.cpu().numpy().reshape(pages, heads, size, row).astype(np.int64)
    v = cache.v_codes.cpu().numpy().reshape(pages, heads, size // 4, row, 4).astype(np.int64)
    if d.bits == 8:
        v = v.transpose(0, 1, 2, 4, 3).reshape(pages, heads, size, dim)
    else:
        nibbles = np.stack([k & 15, k >> 4], -1).reshape(pages, heads, size, dim // 8, 8)
        k = nibbles[..., [0, 4, 1, 5, 2, 6, 3, 7]].reshape(pages, heads, size, dim)
        v = v[..., [0, 2, 1, 3]].transpose(0, 1, 2, 4, 3).reshape(pages, heads, size, row)
        v = np.concatenate([v & 15, v >> 4], -1)

    def by_slot(a):
        return a.swapaxes(1, 2).reshape((pages * size, heads) + a.shape[3:])

    def scales(t):
        a = t.cpu().numpy()
        if d.symmetric:
            a = a.reshape(pages, heads, size)
            return by_slot(a), np.full((pages * size, heads), np.float32(2 ** (d.bits - 1)))
        a = a.reshape(pages, heads, 2, size)
        return by_slot(np.ascontiguousarray(a[:, :, 0])), by_slot(np.ascontiguousarray(a[:, :, 1]))
    return by_slot(k), by_slot(v), scales(cache.k_scales), scales(cache.v_scales)


def attend(q, k, v, visible, scale, dtype, spread=None, top=0.0):
    """softmax(scale q k^T) v over what is visible (q [n, dim], k, v [m, dim], visible [n, m]) in 64 bits, and the error allowed per
    element for a result of type dtype:
      scores   fp32 sums of dim products, and the exponent's own rounding: relative errors of a weight, twice (numerator, denominator)
      weights  rounded once to 11 bits, or 8 for bf16 in prompts (u); those below fp16's normal range to steps of 2^-24 of the largest
      sums     fp32 over m terms
      result   rounded once to dtype, its subnormals included.
    spread [m, dim]: what stands in the second product in place of |v|, where that is larger; top: what the largest weight stands for."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0 or q.shape[0] == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    dim, m = q.shape[1], k.shape[0]
    clean_k, clean_v = (torch.where(visible.any(0)[:, None], x, torch.zeros_like(x)) for x in (k, v))
    s = (q @ clean_k.T * scale).masked_fill(~visible, -math.inf)
    best = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(best == -math.inf, torch.zeros_like(best), best)).masked_fill(~visible, 0)
    total = w.sum(-1, keepdim=True)
    p = w / torch.where(total == 0, torch.ones_like(total), total)
    out = p @ clean_v
    size = clean_v.abs() if spread is None else spread.double()
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    u_weight = u if spread is None else 2.0 ** -11
    magnitude = (q.abs() @ clean_k.abs().T * scale).amax(-1, keepdim=True)
    score = magnitude * (dim + 8) * 2.0 ** -24 + (best.abs().clamp(max=1e30) + magnitude) * 2.0 ** -22 + 2.0 ** -20
    small = 2.0 ** -25 * (visible.double() @ size) * (top if spread is not None else 1.0)
    allowed = (p @ size) * (u_weight + 2 * score + m * 2.0 ** -23) + (p @ clean_v.abs()) * u * 2.0 ** -8 + small + out.abs() * u * 1.01 + 2.0 ** -25
    return out, allowed


def check(got, want, allowed, what):
    got, bad = got.double(), ~torch.isfinite(want)
    assert got.shape == want.shape, what
    assert torch.isfinite(got[~bad]).all(), ("not finite", what)
    off = (got - want).abs()[~bad] - allowed[~bad]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()), float(((got - want).abs() / allowed)[~bad].max()))
    assert not torch.isfinite(got[bad]).any(), ("finite where it cannot be", what)
