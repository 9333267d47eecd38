"""The row operators' definitions in 64 bits on the host, and what rounding lets a kernel differ by."""
from __future__ import annotations

import numpy as np
import torch

GOLDEN, STEP = 0x9E3779B97F4A7C15, 0xD1342543DE82EF95
MASK64 = (1 << 64) - 1


def mix(z: np.ndarray) -> np.ndarray:
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def numbers(index: np.ndarray, seed: int, substream: int) -> np.ndarray:
    """The 48-bit numbers of elements ``index``, one hash at a time from the definition."""
    index = index.astype(np.uint64)
    key = mix(np.array([(seed ^ (GOLDEN * (substream + 1))) & MASK64], dtype=np.uint64))
    h = mix(key + np.uint64(STEP) * (index >> np.uint64(2)))
    lane = index & np.uint64(3)
    high = (h >> (np.uint64(16) * lane)) & np.uint64(0xFFFF)
    low = mix(h + np.uint64(GOLDEN) * (lane + np.uint64(1))) >> np.uint64(32)
    return (high << np.uint64(32)) | low


def kept(shape, p: float, seed: int, substream: int = 0, first_index: int = 0) -> torch.Tensor:
    """Which elements stay, as a tensor of 1.0 and 0.0."""
    n = int(np.prod(shape, dtype=np.int64))
    index = np.arange(n, dtype=np.uint64) + np.uint64(first_index)
    keep = numbers(index, seed, substream) >= np.uint64(round(p * 2.0 ** 48))
    return torch.from_numpy(keep.reshape(shape).astype(np.float64))


# One rounding to type t is off by at most half a step: eps / 2 of the value, or half the smallest
# subnormal below the normal range.
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in HALF_STEP}
F32 = HALF_STEP[torch.float32]


def assert_within(got: torch.Tensor, want: torch.Tensor, before: torch.Tensor, what: str = "") -> None:
    """``got`` is a value that differs from ``want`` (64 bits) by at most ``before``, rounded to got's type."""
    got64 = got.detach().double().cpu()
    allowed = before + (want.abs() + before) * HALF_STEP[got.dtype] + TINY[got.dtype]
    off = (got64 - want).abs()
    bad = ~(off <= allowed) & ~(torch.isnan(got64) & torch.isnan(want)) & ~(got64 == want)
    if bool(bad.any()):
        at = int(torch.nonzero(bad.flatten())[0, 0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got64.flatten()[at]} for {want.flatten()[at]} "
                             f"(allowed {allowed.flatten()[at]})")


def lookup(tokens, table, scale=1.0, first_row=0, p=0.0, seed=0, substream=0, first_index=0):
    """(result in 64 bits, what the fp32 arithmetic before the last rounding may be off)."""
    tokens, table = tokens.cpu().long(), table.detach().cpu().double()
    at = tokens - first_row
    inside = (at >= 0) & (at < table.shape[0])
    out = table[at.clamp(0, max(0, table.shape[0] - 1))] * inside.unsqueeze(-1) if table.shape[0] else torch.zeros((*tokens.shape, table.shape[1]), dtype=torch.float64)
    if p:
        out = torch.where(kept(out.shape, p, seed, substream, first_index) > 0, out, 0.0)
    out = out * (scale / (1.0 - p) if p < 1.0 else 0.0)
    return out, out.abs() * 2.01 * F32  # the factor and the product are rounded


def gradient(acc, tokens, grads, scale=1.0, first_row=0, padding_token=None, accumulate=True, p=0.0, seed=0, substream=0, first_index=0):
    """(new accumulator in 64 bits, what the fp32 sums may be off): k terms are k - 1 additions, then
    the factor's rounding, the product's and the last addition's."""
    acc, grads, flat = acc.detach().cpu().double(), grads.detach().cpu().double(), tokens.cpu().long().reshape(-1)
    if p:
        grads = torch.where(kept(grads.shape, p, seed, substream, first_index) > 0, grads, 0.0)
    grads = grads.reshape(flat.numel(), acc.shape[1])
    at = flat - first_row
    use = (at >= 0) & (at < acc.shape[0])
    if padding_token is not None:
        use &= flat != padding_token
    at, grads = at[use], grads[use]
    factor = scale / (1.0 - p) if p < 1.0 else 0.0
    total = torch.zeros_like(acc).index_add_(0, at, grads)
    sizes = torch.zeros_like(acc).index_add_(0, at, grads.abs())
    terms = torch.zeros(acc.shape[0], dtype=torch.float64).index_add_(0, at, torch.ones(at.numel(), dtype=torch.float64))
    before = sizes * abs(factor) * (terms[:, None] + 2.01) * F32
    out = total * factor
    if accumulate:
        out = out + acc
        before = torch.where(terms[:, None] > 0, before + out.abs() * F32, 0.0)
    return out, before


def dropout(x, p, seed, substream=0, first_index=0, residual=None):
    x = x.detach().cpu().double()
    y = torch.where(kept(x.shape, p, seed, substream, first_index) > 0, x, 0.0) * (1.0 / (1.0 - p) if p < 1.0 else 0.0)
    before = y.abs() * 2.01 * F32
    if residual is not None:
        y = y + residual.detach().cpu().double()
        before = before + y.abs() * F32
    return y, before
