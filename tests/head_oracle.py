"""Plain 64-bit forms of the retrieval head's operators, on the CPU, from the
definitions in include/silvertorch_hip.h.  Gradients come from autograd in
64 bits over these forms."""

from __future__ import annotations

import math

import torch


def bits(words, columns):
    """bool[rows, columns]: document d is bit 63 - d % 64 of word d // 64."""
    at = torch.arange(columns)
    return ((words[:, at >> 6] >> (63 - (at & 63))) & 1).bool()


def pack(passes):
    """int64 words of a bool[rows, columns], whole bundles of 32 words."""
    rows, columns = passes.shape
    words = max(32, (columns + 2047) // 2048 * 32)
    full = torch.zeros((rows, words * 64), dtype=torch.bool)
    full[:, :columns] = passes
    weights = torch.tensor([1 << (63 - i) if i else -(1 << 63) for i in range(64)], dtype=torch.int64)
    return (full.view(rows, words, 64).long() * weights).sum(2)


def best(z, k):
    """(ids, values) of the k largest above -inf, ties by column, NaN never; padded with -1 / -inf."""
    rows, columns = z.shape
    z = torch.where(torch.isnan(z), -math.inf, z)
    values, ids = torch.sort(z, dim=1, descending=True, stable=True)
    pad = max(0, k - columns)
    values = torch.nn.functional.pad(values[:, :k], (0, pad), value=-math.inf)
    ids = torch.nn.functional.pad(ids[:, :k], (0, pad), value=-1)
    return torch.where(values == -math.inf, -1, ids), values


def target_logprobs(logits, targets, topk=0, mask=None, temperature=1.0):
    """float64 logits (a leaf for gradients) -> the operator's outputs."""
    rows, columns = logits.shape
    raw = logits.detach()
    allowed = raw != -math.inf
    if mask is not None:
        allowed = allowed & bits(mask.expand(rows, -1), columns)
    some = allowed.any(1) if columns else torch.zeros(rows, dtype=torch.bool)
    logprobs, entropy, lse = [], [], []
    ids, _ = best(torch.where(allowed, raw, -math.inf), topk)
    tops = []
    for r in range(rows):
        t = int(targets[r])
        if not some[r]:
            logprobs.append(torch.tensor(0.0 if t == -1 else -math.inf, dtype=torch.float64))
            entropy.append(torch.tensor(0.0, dtype=torch.float64))
            lse.append(torch.tensor(-math.inf, dtype=torch.float64))
            tops.append(torch.full((topk,), -math.inf, dtype=torch.float64))
            continue
        z = logits[r, allowed[r]] / temperature
        total = torch.logsumexp(z, 0)
        if not torch.isfinite(total.detach()):
            total = total * math.nan
        log_p = z - total
        p = log_p.exp()
        entropy.append(-(p * torch.where(p > 0, log_p, 0.0)).sum() if torch.isfinite(total.detach()) else total)
        lse.append(total)
        ok = 0 <= t < columns and bool(allowed[r, t])
        logprobs.append(logits[r, t] / temperature - total if ok
                        else torch.tensor(0.0 if t == -1 else -math.inf, dtype=torch.float64))
        tops.append(torch.where(ids[r] >= 0, logits[r, ids[r].clamp(min=0)] / temperature - total, -math.inf))
    stack = lambda v, shape: torch.stack(v) if v else torch.zeros(shape, dtype=torch.float64)
    return (stack(logprobs, (0,)), stack(entropy, (0,)), stack(lse, (0,)), ids, stack(tops, (0, topk)))


def cluster_route(logits, probes, valid=None):
    rows, clusters = logits.shape
    raw = logits.detach()
    on = torch.ones(rows, dtype=torch.bool) if valid is None else valid.clone()
    on &= (raw != -math.inf).any(1)
    n = int(on.sum())
    ids, _ = best(torch.where(on.unsqueeze(1), raw, -math.inf), probes)
    p = torch.zeros_like(raw)
    weights = torch.zeros((rows, probes), dtype=torch.float64)
    lse = torch.full((rows,), -math.inf, dtype=torch.float64)
    if n:
        q = torch.softmax(logits[on], 1)
        p = torch.zeros_like(raw).index_put((on.nonzero().flatten(),), q)
        weights = torch.where(ids >= 0, p.gather(1, ids.clamp(min=0)), 0.0)
        lse = lse.index_put((on.nonzero().flatten(),), torch.logsumexp(logits[on], 1))
    counts = torch.bincount(ids[ids >= 0], minlength=clusters)
    loss = clusters * (counts.double() / (probes * max(n, 1)) * p.sum(0) / max(n, 1)).sum()
    return ids, weights, lse, counts, loss


def unpack4(packed, dim):
    """Codes [rows, dim] of a packed table."""
    return torch.stack([packed & 15, packed >> 4], -1).flatten(1)[:, :dim]


def dequantize(packed, scales, zeros, dim, group):
    of = torch.arange(dim) // group
    zero = zeros.double()[:, of] if zeros is not None else 8.0
    return (unpack4(packed, dim).double() - zero) * scales.double()[:, of]


def quantize(w, group, symmetric):
    """The rule of st_int4_quantize in IEEE float32 arithmetic: codes [rows, dim], scales, zeros."""
    rows, dim = w.shape
    groups = -(-dim // group)
    f = torch.nn.functional.pad(w.float(), (0, groups * group - dim)).view(rows, groups, group)
    lo, hi = f.amin(2).clamp(max=0), f.amax(2).clamp(min=0)
    s = torch.maximum(-lo, hi) / 7 if symmetric else (hi - lo) / 15
    s = torch.where(torch.isfinite(f).all(2), s, math.nan).to(w.dtype)
    sf = s.float()
    any_ = sf > 0
    zero = torch.full_like(sf, 8.0) if symmetric else torch.where(any_, (-lo / sf).round().clamp(0, 15), 0.0)
    q = torch.where(any_.unsqueeze(2), (f / sf.unsqueeze(2)).round() + zero.unsqueeze(2), zero.unsqueeze(2))
    q = q.clamp(0, 15).view(rows, -1)[:, :dim]
    return q.to(torch.uint8), s, zero.to(torch.uint8)
