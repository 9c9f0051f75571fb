"""Inputs and tolerances shared by the paged-cache tests."""
import math

import torch

from tests.gpu_util import DEV

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def lengths(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def bounds(v):
    return torch.tensor([0] + list(v), device=DEV).cumsum(0).to(torch.int32)


def make_cache(total, kv_heads, D, block, kind, dtype, seed=0, poison=True, spare=2):
    """A cache with shuffled pages.  kind: "float", "head" (int8, scale per head), "token" (int8, scale per token and head).
    What no sequence owns - spare pages, the rest of a last page - holds NaN (float), a NaN scale (token) or code 127 (head)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    pages = [-(-n // block) for n in total]
    nb = sum(pages) + spare
    order = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    width = max(pages + [1])
    tables = torch.full((len(total), width), -7, dtype=torch.int32, device=DEV)  # entries behind the last page are never read
    owned = torch.zeros(nb, block, dtype=torch.bool, device=DEV)
    at = 0
    for b, (n, p) in enumerate(zip(total, pages)):
        tables[b, :p] = order[at:at + p]
        for i in range(p):
            owned[order[at + i].long(), :min(block, n - i * block)] = True
        at += p
    shape = (nb, block, kv_heads, D)
    if kind == "float":
        k, v = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
        if poison:
            k[~owned], v[~owned] = math.nan, math.inf
        return dict(k=k, v=v, ks=None, vs=None, tables=tables, owned=owned)
    k, v = ((torch.randn(shape, generator=g, device=DEV) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
    of = (kv_heads,) if kind == "head" else (nb, block, kv_heads)
    ks, vs = ((torch.rand(of, generator=g, device=DEV) + 0.5) * 0.03 for _ in range(2))
    if poison:
        k[~owned], v[~owned] = 127, 127
        if kind == "token":
            ks[~owned], vs[~owned] = math.nan, math.inf
    return dict(k=k, v=v, ks=ks.contiguous(), vs=vs.contiguous(), tables=tables, owned=owned)


def attention_tolerance(ref, lse, spread, mass, reach, D, kind, dtype):
    """(for out, for lse).  out: half a step of its own rounding; each weight is rounded once to the 16-bit type that multiplies V
    (f16 wherever the cache is int8) - at most half a step of it per weight, so that much of sum p |v|; a logit is an fp32 sum of D
    exact products: its error is at most (D + 4) * 2^-24 times sum |q k|, and moves each weight by twice that, relatively (the
    numerator and the total); 2^-17 covers exp2, log2 and the fp32 sums (2^-22 each, up to 32 of them in a row).  Weights far below the largest one, which is 1 or more as they are formed, leave the normal
    range: then the error is absolute, 2^-25 in f16 (half its subnormal step), 2^-126 where small numbers become 0 in fp32 and bf16,
    times sum |v|.  (With a scale per token the largest product of weight and scale takes the place of the largest weight: the
    tests' scales lie within a factor of 3, so 2^-25 becomes at most 2^-23.)"""
    logit = (D + 4) * 2.0 ** -24 * reach
    weight = HALF[torch.float16 if kind != "float" else dtype]
    tol = HALF[dtype] * ref.abs() + (weight + 2 * logit + 2.0 ** -17)[..., None] * spread * (1 + HALF[dtype])
    tol = tol + mass * (2.0 ** -23 if kind == "token" else 2.0 ** -25 if kind == "head" or dtype == torch.float16 else 2.0 ** -126)
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)  # half the output's own subnormal step
    return tol, logit + 2.0 ** -17 + 2.0 ** -23 * lse.abs()


def compare(got, ref, tol, what):
    got = got.double()
    same = (got == ref) | (got.isnan() & ref.isnan())
    off = torch.where(same, 0.0, (got - ref).abs())
    bad = ~(off <= tol) & ~same
    if bool(bad.any()):
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got {got[tuple(i)].item()}, "
                             f"expected {ref[tuple(i)].item()}, tolerance {tol[tuple(i)].item()}")
