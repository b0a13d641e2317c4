"""The layers of a query tower and 8-bit score tables, as a user's program calls them, and their plain forms.

    layer_norm              rows to mean 0 and variance 1, times a weight plus a bias; with its gradients
    dropout                 elements kept or zeroed by counter-based random numbers, with no stored mask; with its
                            gradient
    dropout_add_layer_norm  residual + dropout(x) and its layer norm in one pass; with its gradients
    int8_matmul             products of a table held in 8 bits (a scale for each row) with vectors that are taken to
                            8 bits on the way (a scale for each vector), also right after a layer norm (layer_norm_int8)

Each case is one pass through one operator (training cases: forward and backward).  `own` chooses between the
framework's operators and plain forms of the same formulas in elementary torch operations in 32 bits.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call
    run(state)           one pass; its outputs
    work(case)           bytes and flops a pass cannot do without
    exact(case, seed)    the outputs in 64 bits, from the definitions
"""

import math

import torch

DEVICE = "cuda"
EPS = 1e-5

own = False


def listed():
    return [
        # One request's vector in a served tower: launch and latency.
        dict(name="norm_one", op="norm", rows=1, dim=1_024, dtype="bfloat16", weights="bfloat16", train=False),
        # A training step over a large batch of queries, weights kept in 32 bits.
        dict(name="norm_train", op="norm", rows=65_536, dim=1_024, dtype="bfloat16", weights="float32", train=True),
        # Short embeddings of many documents, as a document tower ends.
        dict(name="norm_embeddings", op="norm", rows=1_000_003, dim=128, dtype="float16", weights="float16", train=True),
        # A wide layer of odd length in 32 bits.
        dict(name="norm_odd", op="norm", rows=8_191, dim=5_003, dtype="float32", weights="float32", train=True),
        # A layer's end in training: dropout, residual stream in 32 bits, layer norm.
        dict(name="residual_train", op="residual", rows=32_768, dim=2_048, dtype="bfloat16", residual="float32",
             weights="float32", p=0.1, train=True),
        # The same for a small batch of ragged width.
        dict(name="residual_small", op="residual", rows=511, dim=777, dtype="float16", residual="float16",
             weights="float32", p=0.25, train=True),
        # Dropout of a small batch's features.
        dict(name="dropout_small", op="dropout", rows=64, dim=256, dtype="bfloat16", p=0.1, train=False),
        # Dropout of a wide hidden layer in training.
        dict(name="dropout_train", op="dropout", rows=32_768, dim=4_096, dtype="bfloat16", p=0.2, train=True),
        # One request's scores over the whole corpus.
        dict(name="int8_corpus", op="int8", tokens=1, dim=128, rows=20_000_000, x="bfloat16", norm=False, bias=False,
             out="float32"),
        # The scores of a batch of requests over a ragged shard.
        dict(name="int8_shard", op="int8", tokens=64, dim=128, rows=2_499_999, x="float32", norm=False, bias=False,
             out="float32"),
        # A layer for a few requests: the norm to 8 bits, then the product.
        dict(name="int8_layer_few", op="int8", tokens=4, dim=2_048, rows=8_192, x="bfloat16", norm=True, bias=True,
             out="bfloat16"),
        # The same layer over a large batch.
        dict(name="int8_layer_batch", op="int8", tokens=16_384, dim=4_096, rows=8_192, x="bfloat16", norm=True, bias=True,
             out="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "residual", "dropout", "int8", "int8"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "int8":
        dim = rng.choice([_log_int(rng, 16, 8_192), 64, 128, 256, 1_024])
        rows = _log_int(rng, 64, min(20_000_000, 2_000_000_000 // dim))
        tokens = _log_int(rng, 1, max(1, min(16_384, 160_000_000 // rows, 500_000_000_000 // (dim * rows))))
        norm = rng.random() < 0.4
        return dict(op=op, tokens=tokens, dim=dim, rows=rows, x=rng.choice([dtype, dtype, "codes"]) if not norm else dtype,
                    norm=norm, bias=rng.random() < 0.5, out=rng.choice(["bfloat16", "float16"] + ([] if norm else ["float32", "float32"])))
    dim = rng.choice([_log_int(rng, 8, 16_384), 64, 128, 256, 512, 1_024, 4_096])
    case = dict(op=op, rows=_log_int(rng, 1, min(1_000_000, 100_000_000 // dim)), dim=dim, dtype=dtype)
    if op != "dropout":
        case["weights"] = rng.choice([dtype, "float32"])
    if op == "residual":
        case["residual"] = rng.choice([dtype, "float32"])
    if op != "norm":
        case["p"] = rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    case["train"] = rng.random() < 0.7
    return case


# ---------------------------------------------------------------- inputs


def _generator(seed, stream):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 1_000_003 + stream)
    return g


def _normal(shape, dtype, scale, g, shift=0.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale + shift).to(dtype)


def _columns(dim):
    """8-bit rows are whole blocks of 16 columns; those past the last hold zeros."""
    return -(-dim // 16) * 16


def prepare(case, seed):
    op = case["op"]
    g = _generator(seed, 1)
    s = dict(case=case)
    if op == "int8":
        tokens, dim, rows = case["tokens"], case["dim"], case["rows"]
        width = _columns(dim)
        codes = torch.randint(-127, 128, (rows, width), generator=g, device=DEVICE, dtype=torch.int8)
        codes[:, dim:] = 0
        s.update(codes=codes, scales=(0.5 + torch.rand(rows, generator=g, device=DEVICE)) * (dim ** -0.5 / 64),
                 bias=_normal((rows,), torch.float32, 0.1, g) if case["bias"] else None, out=getattr(torch, case["out"]))
        if case["x"] == "codes":
            x = torch.randint(-127, 128, (tokens, width), generator=g, device=DEVICE, dtype=torch.int8)
            x[:, dim:] = 0
            s.update(x=x, x_scales=(0.5 + torch.rand(tokens, generator=g, device=DEVICE)) / 64)
        else:
            s.update(x=_normal((tokens, dim), getattr(torch, case["x"]), 1.0, g), x_scales=None)
        if case["norm"]:
            s.update(weight=_normal((dim,), torch.float32, 0.1, g, 1.0), shift=_normal((dim,), torch.float32, 0.1, g))
        return s
    rows, dim, dtype, train = case["rows"], case["dim"], getattr(torch, case["dtype"]), case["train"]
    s["x"] = _normal((rows, dim), dtype, 1.5, g, 0.3).requires_grad_(train)
    if op != "norm":
        s["rng"] = torch.randint(0, 1 << 62, (2,), generator=g, device=DEVICE)
    if op != "dropout":
        weights = getattr(torch, case["weights"])
        s.update(weight=_normal((dim,), weights, 0.1, g, 1.0).requires_grad_(train),
                 bias=_normal((dim,), weights, 0.1, g).requires_grad_(train))
    if op == "residual":
        residual = getattr(torch, case["residual"])
        s["residual"] = _normal((rows, dim), residual, 2.0, g).requires_grad_(train)
        if train:
            s["grad_sum"] = _normal((rows, dim), residual, 0.5, g)
    if train:
        s["grad"] = _normal((rows, dim), dtype, 1.0, g)
    return s


# ---------------------------------------------------------------- one pass


def run(state):
    op, form = state["case"]["op"], 0 if own else 1
    return {"norm": (_norm, _plain_norm), "residual": (_residual, _plain_residual), "dropout": (_dropout, _plain_dropout),
            "int8": (_int8, _plain_int8)}[op][form](state)


def _norm(s):
    import silvertorch_amd.ops._load_ops  # noqa: F401  (registers torch.ops.st)

    y = torch.ops.st.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not s["case"]["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["grad"])]


def _residual(s):
    import silvertorch_amd.ops._load_ops  # noqa: F401

    y, total = torch.ops.st.dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], s["case"]["p"], s["rng"], EPS)
    if not s["case"]["train"]:
        return [y, total]
    return [y.detach(), total.detach(), *torch.autograd.grad(
        [y, total], [s["x"], s["residual"], s["weight"], s["bias"]], [s["grad"], s["grad_sum"]])]


def _dropout(s):
    import silvertorch_amd.ops._load_ops  # noqa: F401

    y = torch.ops.st.dropout(s["x"], s["case"]["p"], s["rng"])
    if not s["case"]["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s["x"]], s["grad"])]


def _int8(s):
    import silvertorch_amd.ops._load_ops  # noqa: F401

    x, x_scales = s["x"], s["x_scales"]
    if s["case"]["norm"]:
        x, x_scales = torch.ops.st.layer_norm_int8(x, s["weight"], s["shift"], EPS)
    return torch.ops.st.int8_matmul(s["codes"], s["scales"], x, x_scales, s["bias"], s["out"])


# ---------------------------------------------------------------- plain forms


def _statistics(h):
    centred = h - h.mean(1, keepdim=True)
    return centred, 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)


def _norm_gradients(centred, scale, weight, grad):
    """Of the rows, the weight and the bias."""
    normed, g = centred * scale, grad * weight
    rows = scale * (g - g.mean(1, keepdim=True) - normed * (g * normed).mean(1, keepdim=True))
    return rows, (grad * normed).sum(0), grad.sum(0)


def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    centred, scale = _statistics(x)
    y = (centred * scale * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return [y]
    gx, gw, gb = _norm_gradients(centred, scale, w, s["grad"].float())
    return [y, gx.to(s["x"].dtype), gw.to(s["weight"].dtype), gb.to(s["bias"].dtype)]


def _keep(rng, p, shape):
    """Which elements stay, and what they are multiplied with.  Philox4x32-10 (Salmon et al., 2011) with key rng[0] and
    counter (element / 8, rng[1]) gives 8 halves of words, the low one of word i / 2 for an even element i, and an
    element stays if its half is at least p in units of 2^-16."""
    low = 0xFFFFFFFF
    count = shape[0] * shape[1]
    at = torch.arange((count + 7) // 8, device=DEVICE)
    c = [at & low, at >> 32, (rng[1] & low).expand_as(at), ((rng[1] >> 32) & low).expand_as(at)]
    k = [rng[0] & low, (rng[0] >> 32) & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # the low 64 bits; their upper half masked below
        c = [((b >> 32) & low) ^ c[1] ^ k[0], b & low, ((a >> 32) & low) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    words = torch.stack(c, 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)[:count].view(shape)
    dropped = int(round(p * 65_536))
    return halves >= dropped, 65_536.0 / (65_536 - dropped) if dropped < 65_536 else 0.0


def _plain_residual(s):
    w, b, residual = s["weight"].detach().float(), s["bias"].detach().float(), s["residual"].detach()
    keep, times = _keep(s["rng"], s["case"]["p"], residual.shape)
    total = (residual.float() + torch.where(keep, s["x"].detach().float() * times, 0.0)).to(residual.dtype)
    centred, scale = _statistics(total.float())
    y = (centred * scale * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return [y, total]
    rows, gw, gb = _norm_gradients(centred, scale, w, s["grad"].float())
    rows = rows + s["grad_sum"].float()
    gx = torch.where(keep, rows * times, 0.0)
    return [y, total, gx.to(s["x"].dtype), rows.to(residual.dtype), gw.to(s["weight"].dtype), gb.to(s["bias"].dtype)]


def _plain_dropout(s):
    keep, times = _keep(s["rng"], s["case"]["p"], s["x"].shape)
    y = torch.where(keep, s["x"].detach().float() * times, 0.0).to(s["x"].dtype)
    if not s["case"]["train"]:
        return [y]
    return [y, torch.where(keep, s["grad"].float() * times, 0.0).to(s["x"].dtype)]


def _codes(x):
    """Rows in 8 bits: the scale is max |x| / 127, a code x times 127 / max |x| to the nearest even."""
    most = x.abs().amax(1, keepdim=True)
    return torch.round(x * (127.0 / most)), most / 127.0


def _plain_int8(s):
    x, dim = s["x"].float(), s["case"]["dim"]
    if s["case"]["norm"]:
        centred, scale = _statistics(x)
        x = centred * scale * s["weight"] + s["shift"]
    if s["x_scales"] is None:
        x, x_scales = _codes(x)
    else:
        x, x_scales = x[:, :dim], s["x_scales"].unsqueeze(1)
    y = x @ s["codes"][:, :dim].float().t() * x_scales * s["scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"])


# ---------------------------------------------------------------- work


def _bytes(name):
    return {"float32": 4, "codes": 1}.get(name, 2)


def work(case):
    op = case["op"]
    if op == "int8":
        tokens, dim, rows = case["tokens"], case["dim"], case["rows"]
        per = _columns(dim)
        return {"bytes": rows * (per + 4 + (4 if case["bias"] else 0)) + tokens * dim * _bytes(case["x"])
                + tokens * rows * _bytes(case["out"]), "flops": 2 * tokens * rows * dim}
    rows, dim, size = case["rows"], case["dim"], _bytes(case["dtype"])
    # x and the result, the result's gradient and that of x
    each = 2 * size * (2 if case["train"] else 1)
    flops = 3
    if op == "residual":
        each += 2 * _bytes(case["residual"]) * (2 if case["train"] else 1)
    total = rows * dim * each
    if op != "dropout":
        total += 2 * dim * _bytes(case["weights"]) * (2 if case["train"] else 1)
        flops += 8 * (3 if case["train"] else 1)
    return {"bytes": total, "flops": rows * dim * flops}


# ---------------------------------------------------------------- 64 bits


def _exact_keep(state, p, rows, dim):
    """The same numbers by the cipher's rounds on 32-bit words, multiplied in 16-bit halves."""
    key, offset = int(state[0]), int(state[1])
    blocks = torch.arange((rows * dim + 7) // 8, device=DEVICE)
    word = lambda v, i: (v >> (32 * i)) & 0xFFFFFFFF  # noqa: E731

    def product(m, v):
        low = m * (v & 0xFFFF)
        high = m * (v >> 16) + (low >> 16)
        return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)

    x0, x1 = word(blocks, 0), word(blocks, 1)
    x2, x3 = torch.full_like(blocks, word(offset, 0)), torch.full_like(blocks, word(offset, 1))
    for r in range(10):
        k0, k1 = (word(key, 0) + r * 0x9E3779B9) & 0xFFFFFFFF, (word(key, 1) + r * 0xBB67AE85) & 0xFFFFFFFF
        (h0, l0), (h2, l2) = product(0xD2511F53, x0), product(0xCD9E8D57, x2)
        x0, x1, x2, x3 = h2 ^ x1 ^ k0, l2, h0 ^ x3 ^ k1, l0
    halves = torch.stack([part for x in (x0, x1, x2, x3) for part in (x % 65_536, x // 65_536)], 1)
    t = round(p * 65_536)
    kept = (halves.flatten()[: rows * dim] >= t).reshape(rows, dim)
    return kept.double() * (65_536 / (65_536 - t) if t < 65_536 else 0.0)


def _exact_layer_norm(x, w, b):
    variance, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    return (x - mean) / (variance + EPS).sqrt() * w + b


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "int8":
        x = s["x"].double()
        if case["norm"]:
            x = _exact_layer_norm(x, s["weight"].double(), s["shift"].double())
        if s["x_scales"] is None:
            scales = x.abs().amax(1) / 127
            x = (x / scales.unsqueeze(1)).round()
        else:
            scales = s["x_scales"].double()
        y = torch.empty((case["tokens"], case["rows"]), dtype=torch.float64, device=DEVICE)
        for at in range(0, case["rows"], 1_000_000):
            part = slice(at, at + 1_000_000)
            y[:, part] = (x @ s["codes"][part, : x.shape[1]].t().contiguous().double()) * torch.outer(scales, s["scales"][part].double())
            if s["bias"] is not None:
                y[:, part] += s["bias"][part].double()
        return y
    train = case["train"]
    leaf = lambda name: s[name].detach().double().requires_grad_(train)  # noqa: E731
    x = leaf("x")
    if op == "dropout":
        factor = _exact_keep(s["rng"], case["p"], *x.shape)
        y = x.detach() * factor
        return [y, s["grad"].double() * factor] if train else [y]
    w, b = leaf("weight"), leaf("bias")
    if op == "norm":
        y = _exact_layer_norm(x, w, b)
        return [y.detach(), *(torch.autograd.grad(y, [x, w, b], s["grad"].double()) if train else ())]
    residual = leaf("residual")
    factor = _exact_keep(s["rng"], case["p"], *x.shape)
    total = residual + x * factor
    # the norm is of the sum as it is held; its gradient goes to the sum as it is
    held = total + (total.detach().to(s["residual"].dtype).double() - total.detach())
    y = _exact_layer_norm(held, w, b)
    return [y.detach(), total.detach(), *(torch.autograd.grad(
        [y, total], [x, residual, w, b], [s["grad"].double(), s["grad_sum"].double()]) if train else ())]
