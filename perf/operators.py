"""The operators of a block over packed rows, as measurable cases.

A case is a dict of plain values; its "op" says which operator it goes through:

  attention   softmax attention over packed sequences, grouped heads, causal or not
              (`FusedKernels.packed_attention`)
  projection  a matrix product with bias, activation, scale and residual (`FusedKernels.projection`)
  norm        the norm after a block, its gate and residual scale, and the norm before the next
              (`FusedKernels.block_norm`)

Together they are one block: norm, projection, attention, projection, norm, projection, projection.
`run` computes each in elementary torch operations in 32 bits where `own` is false and calls
the framework where it is true.  Types are fp16 and bf16 (a residual stream may be fp32).  Widths are the
encoder's (1,024, 4,096, 16 heads of 64) and generic ones of wider blocks (4,096, heads of 128).
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _attention(name, dtype, heads, kv_heads, dim, q_lengths, k_lengths, causal=True):
    """k_lengths None: every sequence attends to itself and q, k, v are one projection's output."""
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q_lengths": " ".join(map(str, q_lengths)),
            "k_lengths": "" if k_lengths is None else " ".join(map(str, k_lengths)), "causal": causal}


def _lengths(case):
    """(queries, keys) of every sequence."""
    q = [int(n) for n in case["q_lengths"].split()]
    return q, [int(n) for n in case["k_lengths"].split()] or q


def _projection(name, dtype, m, n, k, activation, bias, residual, scale=1.0):
    return {"name": name, "op": "projection", "dtype": dtype, "m": m, "n": n, "k": k, "activation": activation,
            "bias": bias, "residual": residual, "scale": scale}


def _norm(name, dtype, rows, cols, kind, stream, post, gate, scale=1.0):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "kind": kind, "stream": stream,
            "post": post, "gate": gate, "scale": scale}


def listed():
    ragged = random.Random(7)
    texts = [ragged.randint(16, 256) for _ in range(32)]
    contexts = [round(2 ** ragged.uniform(10, 15)) for _ in range(16)]
    return [
        # The next token of one short text: what an interactive caller waits for.
        _attention("attention_one_token", "fp16", 16, 4, 64, [1], [512]),
        # The next tokens of a batch of conversations, each with its own long context.
        _attention("attention_next_tokens", "bf16", 32, 8, 128, [1] * 16, contexts),
        # The serving batch: 32 texts of up to 256 tokens, packed, straight from their projection.
        _attention("attention_texts", "fp16", 16, 4, 64, texts, None),
        # Pieces of prompts whose beginnings are in the cache, one of them a single token.
        _attention("attention_pieces", "fp16", 12, 2, 128, [257, 1, 64], [8448, 4099, 64]),
        # One long prompt.
        _attention("attention_prompt", "bf16", 32, 8, 128, [16384], None),
        # The encoder's widening projection for one token.
        _projection("projection_one_row", "fp16", 1, 4096, 1024, "gelu", True, False),
        # Rows and columns that fill no tile, onto the residual stream.
        _projection("projection_odd", "bf16", 777, 1000, 4096, "silu", True, True, 0.5),
        # The encoder's widening projection for a batch.
        _projection("projection_up", "fp16", 8192, 4096, 1024, "gelu", True, False),
        # The narrowing projection of a wide block onto the residual stream.
        _projection("projection_down", "bf16", 8192, 4096, 16384, "none", False, True),
        # One token between two blocks.
        _norm("norm_one_row", "fp16", 1, 1024, "layer", "fp16", True, "column"),
        # A packed batch between two blocks, a gate for each row.
        _norm("norm_texts", "fp16", 4103, 1024, "layer", "fp16", True, "row", 0.5),
        # A wide block's long prompt, the residual stream in fp32.
        _norm("norm_wide", "bf16", 16384, 4096, "rms", "fp32", True, "column"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("attention", "projection", "norm"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "attention":
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
        dim = rng.choice((64, 64, 96, 128, 128, 256))
        shape = rng.choice(("prompts", "pieces", "tokens"))
        causal = rng.random() < 0.8
        while True:
            batch = _log_int(rng, 1, 48)
            if shape == "prompts":
                top = _log_int(rng, 16, 8192)
                q = [rng.randint(1, top) for _ in range(batch)]
                k = None
            elif shape == "pieces":
                q = [rng.choice((1, _log_int(rng, 1, 700))) for _ in range(batch)]
                k = [n + _log_int(rng, 1, 16000) for n in q]
            else:
                q = [1] * batch
                k = [_log_int(rng, 1, 32768) for _ in q]
            case = _attention("", dtype, heads, kv_heads, dim, q, k, causal)
            w = work(case)
            if w["flops"] <= 1.0e12 and w["bytes"] <= 6.0e8:
                break
    elif op == "projection":
        while True:
            m, n, k = _log_int(rng, 1, 16384), _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
            kind = rng.random()
            if kind < 0.7:  # widths of blocks
                n, k = -(-n // 64) * 64, -(-k // 64) * 64
            elif kind < 0.9:  # a head of any number of outputs
                k = -(-k // 8) * 8
            if m * n * k <= 2 ** 38:
                break
        case = _projection("", dtype, m, n, k, rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                           rng.random() < 0.7, rng.random() < 0.6, rng.choice((1.0, 0.5, 0.17)))
    else:
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 64, 8192)
            if rows * cols <= 2 ** 26:
                break
        if rng.random() < 0.8:
            cols = -(-cols // 8) * 8
        case = _norm("", dtype, rows, cols, rng.choice(("rms", "layer")), rng.choice((dtype, "fp32")),
                     rng.random() < 0.7, rng.choice(("none", "column", "row")), rng.choice((1.0, 0.5, 0.17)))
    del case["name"]
    return case


def _pairs(case):
    """Query-key pairs that the mask leaves, over all sequences."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        if not case["causal"]:
            total += nq * nk
            continue
        # query i sees keys 0 .. nk - nq + i
        first = max(0, nq - nk)  # queries before it see no key
        total += (nk - nq + first + 1 + nk) * (nq - first) // 2
    return total


def work(case):
    if case["op"] == "attention":
        tq, tk = map(sum, _lengths(case))
        return {"bytes": 2 * case["dim"] * (2 * tq * case["heads"] + 2 * tk * case["kv_heads"]),
                "flops": 4 * case["dim"] * case["heads"] * _pairs(case)}
    if case["op"] == "projection":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    stream = 4 if case["stream"] == "fp32" else 2
    gate = {"none": 0, "column": 1, "row": rows}[case["gate"]]
    weights = (2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1)
    return {"bytes": cols * (rows * (2 + 2 + 2 * stream) + 2 * gate + 2 * weights), "flops": 12 * rows * cols}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _offsets(lengths, device):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dtype):
        return torch.empty(shape, dtype=torch.float32, device=device).normal_(mean, scale, generator=gen).to(dtype)

    s = {"case": case}
    if case["op"] == "attention":
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        q_lengths, k_lengths = _lengths(case)
        tq, tk = sum(q_lengths), sum(k_lengths)
        if not case["k_lengths"]:
            qkv = normal(tq, hq + 2 * hk, d)
            s["q"], s["k"], s["v"] = qkv.split((hq, hk, hk), dim=1)
            s["k_offsets"] = None
        else:
            s["q"], s["k"], s["v"] = normal(tq, hq, d), normal(tk, hk, d), normal(tk, hk, d)
            s["k_offsets"] = _offsets(k_lengths, device)
        s["q_offsets"] = _offsets(q_lengths, device)
    elif case["op"] == "projection":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = normal(m, k)
        s["weight"] = normal(n, k, scale=k ** -0.5)
        s["bias"] = normal(n, scale=0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
    else:
        rows, cols = case["rows"], case["cols"]
        layer = case["kind"] == "layer"
        s["y"] = normal(rows, cols)
        s["residual"] = normal(rows, cols, dtype=DTYPES[case["stream"]])
        s["pre_weight"] = normal(cols, scale=0.1, mean=1.0)
        s["pre_bias"] = normal(cols, scale=0.1) if layer else None
        s["post_weight"] = normal(cols, scale=0.1, mean=1.0) if case["post"] else None
        s["post_bias"] = normal(cols, scale=0.1) if case["post"] and layer else None
        s["gate"] = {"none": lambda: None, "column": lambda: normal(cols), "row": lambda: normal(rows, cols)}[
            case["gate"]]()
    if own:
        import sys
        from pathlib import Path
        package = str(Path.cwd() / "gliner-decide-metal_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from gliner_decide import FusedKernels
        s["kernels"] = FusedKernels()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](state, case)
    with torch.no_grad():
        return _PLAIN[case["op"]](state, case)


def _own_attention(s, case):
    return s["kernels"].packed_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"],
                                         causal=case["causal"])


def _own_projection(s, case):
    return s["kernels"].projection(s["x"], s["weight"], s["bias"], s["residual"], activation=case["activation"],
                                   scale=case["scale"])


def _own_norm(s, case):
    return s["kernels"].block_norm(s["y"], s["residual"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"],
                                   post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                                   scale=case["scale"], eps=EPS, kind=case["kind"])


_OWN = {"attention": _own_attention, "projection": _own_projection, "norm": _own_norm}


def _plain_attention(s, case):
    q, k, v = s["q"], s["k"], s["v"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group = hq // hk
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    q0 = k0 = 0
    for nq, nk in zip(*_lengths(case)):
        keys = k[k0:k0 + nk].float().permute(1, 2, 0).contiguous()  # [hk, d, nk]
        values = v[k0:k0 + nk].float().permute(1, 0, 2).contiguous()  # [hk, nk, d]
        step = max(1, (1 << 28) // (hq * max(nk, 1)))
        for a in range(0, nq, step):
            b = min(nq, a + step)
            seen = min(nk, nk - nq + b) if case["causal"] else nk
            if seen <= 0:
                continue
            rows = q[q0 + a:q0 + b].float().view(b - a, hk, group, d).permute(1, 2, 0, 3)
            rows = rows.reshape(hk, group * (b - a), d) * d ** -0.5
            scores = rows @ keys[:, :, :seen]
            if case["causal"]:
                last = torch.arange(a, b, device=q.device) + (nk - nq)
                hidden = torch.arange(seen, device=q.device)[None] > last[:, None]
                scores = scores.view(hk, group, b - a, seen).masked_fill_(hidden, float("-inf")).view(scores.shape)
            top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
            weights = scores.sub_(top).exp_()
            total = weights.sum(-1, keepdim=True)
            rows = (weights @ values[:, :seen]) / torch.where(total > 0, total, 1.0)
            out[q0 + a:q0 + b] = rows.view(hk, group, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d).to(q.dtype)
        q0 += nq
        k0 += nk
    return out


def _plain_projection(s, case):
    y = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    activation = case["activation"]
    if activation == "relu":
        y = y.clamp(min=0.0)
    elif activation == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))
    elif activation == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    elif activation == "silu":
        y = y / (1.0 + torch.exp(-y))
    y = y * case["scale"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_norm(s, case):
    def norm(x, weight, bias):
        if case["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        return x if bias is None else x + bias.float()

    z = s["y"].float()
    if s["post_weight"] is not None:
        z = norm(z, s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        z = z * s["gate"].float()
    h = s["residual"].float() + case["scale"] * z
    return h.to(s["residual"].dtype), norm(h, s["pre_weight"], s["pre_bias"]).to(s["y"].dtype)


_PLAIN = {"attention": _plain_attention, "projection": _plain_projection, "norm": _plain_norm}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "projection": _exact_projection, "norm": _exact_norm}[case["op"]](
            s, case)


def _exact_attention(s, case):
    """out[t, h] = sum_j exp(z_j) v_j / sum_j exp(z_j), z_j = q_t . k_j / sqrt(d), one head at a time."""
    group = case["heads"] // case["kv_heads"]
    scale = 1.0 / math.sqrt(case["dim"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    starts_q = starts_k = 0
    for nq, nk in zip(*_lengths(case)):
        positions = torch.arange(nk, device=out.device)
        for h in range(case["heads"]):
            kk = s["k"][starts_k:starts_k + nk, h // group].double()
            vv = s["v"][starts_k:starts_k + nk, h // group].double()
            for a in range(0, nq, 4096):
                b = min(nq, a + 4096)
                z = torch.mm(s["q"][starts_q + a:starts_q + b, h].double(), kk.t().contiguous()) * scale
                if case["causal"]:
                    border = torch.arange(nk - nq + a, nk - nq + b, device=out.device)
                    z = torch.where(positions <= border[:, None], z, -math.inf)
                lse = torch.logsumexp(z, dim=-1, keepdim=True)
                weights = torch.where(torch.isinf(lse), 0.0, torch.exp(z - lse))
                out[starts_q + a:starts_q + b, h] = torch.mm(weights, vv)
        starts_q += nq
        starts_k += nk
    return out


def _exact_projection(s, case):
    y = torch.mm(s["x"].double(), s["weight"].double().t().contiguous())
    if case["bias"]:
        y += s["bias"].double()
    kind = case["activation"]
    if kind == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif kind == "gelu":
        y = y * torch.special.erfc(-y / math.sqrt(2.0)) / 2.0
    elif kind == "gelu_tanh":
        inner = math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)
        y = y / (1.0 + torch.exp(-2.0 * inner))
    elif kind == "silu":
        y = y * torch.special.expit(y)
    y = case["scale"] * y
    return y + s["residual"].double() if case["residual"] else y


def _exact_norm(s, case):
    def normed(x, name):
        centre = x.mean(-1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(x[..., :1])
        spread = ((x - centre) ** 2).sum(-1, keepdim=True) / x.shape[-1]
        y = (x - centre) / torch.sqrt(spread + EPS) * s[name + "_weight"].double()
        return y if s[name + "_bias"] is None else y + s[name + "_bias"].double()

    block = normed(s["y"].double(), "post") if case["post"] else s["y"].double()
    if case["gate"] != "none":
        block = block * s["gate"].double()
    stream = s["residual"].double() + case["scale"] * block
    return stream, normed(stream, "pre")
