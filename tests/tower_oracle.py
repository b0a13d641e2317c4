"""Plain forms of the query tower's operators on the CPU, from the definitions
in include/silvertorch_hip.h: layer norm in 64 bits, dropout's random numbers
in whole numbers, rows in 8 bits by their rule in IEEE float32 arithmetic."""

from __future__ import annotations

import numpy as np
import torch

EPS = 1e-5


def philox(counter, key, rounds=10):
    """Philox4x32 of uint64 arrays that hold 32-bit words: four words of counter, two of key."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [np.uint64(w) for w in key]
    for _ in range(rounds):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def units(p):
    """p in units of 2^-16."""
    return int(round(p * 65536))


def times(p):
    return 65536 / (65536 - units(p)) if units(p) < 65536 else 0.0


def keeps(shape, p, state):
    """bool of `shape`: which elements stay."""
    count = int(np.prod(shape))
    seed, offset = (int(v) & (2**64 - 1) for v in state)
    blocks = np.arange((count + 7) // 8, dtype=np.uint64)
    whole = np.zeros_like(blocks)
    words = philox([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), whole + np.uint64(offset & 0xFFFFFFFF),
                    whole + np.uint64(offset >> 32)], [seed & 0xFFFFFFFF, seed >> 32])
    halves = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)[:count]
    return torch.from_numpy((halves >= units(p)).reshape(shape))


def dropped(x, p, state):
    """x through dropout in float32, not rounded to x's type."""
    factor = torch.tensor(times(p), dtype=torch.float32)
    return torch.where(keeps(x.shape, p, state), x.float() * factor, 0.0)


def layer_norm(h, weight=None, bias=None, eps=EPS):
    """float64, over the last dimension; differentiable."""
    centred = h - h.mean(-1, keepdim=True)
    n = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    y = n if weight is None else n * weight
    return y if bias is None else y + bias


def codes(x):
    """(codes, scales) of rows by the rule, in float32."""
    f = x.float()
    dim = f.shape[-1]
    most = f.abs().amax(-1)
    fine = torch.isfinite(f).all(-1)
    small = most < 2.0 ** -119
    # quotients of two tensors, which are rounded once
    times_ = torch.where(fine & ~small, torch.ones_like(most) / most * 127.0, 0.0)
    scales = torch.where(fine, torch.where(small, 0.0, most / torch.full_like(most, 127.0)), torch.nan)
    q = torch.where((times_ != 0).unsqueeze(-1), (f * times_.unsqueeze(-1)).round(), 0.0)
    return torch.nn.functional.pad(q, (0, -dim % 16)).to(torch.int8), scales


def matmul(table, scales, x, x_scales, bias=None):
    """float64 from codes."""
    y = (x.double() @ table.double().t()) * x_scales.double().unsqueeze(-1) * scales.double()
    return y if bias is None else y + bias.double()
