"""Cases of the transformer-layer operators: layer norm, counter-based dropout, the fused
dropout + residual + layer norm, and attention with a learned relative position bias.

`run` computes a case either in plain torch operations (own = False) or through the
framework's entry points in cgt_amd.kernels (own = True) on the same inputs.
"""
import math

import numpy as np
import torch

own = False

M32 = 0xFFFFFFFF

# ---------------------------------------------------------------- cases


def _ln(name, op, rows, cols):
    return {"name": name, "op": op, "rows": rows, "cols": cols}


def _drop(name, n, p, residual):
    return {"name": name, "op": "dropout", "n": n, "p": p, "residual": residual}


def _daln(name, op, rows, cols, p):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "p": p}


def _att(name, op, B, H, Tq, Tk, D, causal=False, buckets=32, max_distance=128, p=0.0, ragged=False, empty=False, layout="bhtd"):
    return {"name": name, "op": op, "B": B, "H": H, "Tq": Tq, "Tk": Tk, "D": D, "causal": causal, "buckets": buckets,
            "max_distance": max_distance, "p": p, "ragged": ragged, "empty": empty, "layout": layout}


def listed():
    return [
        # one new token in each of eight sequences: what counts is the latency of the call
        _ln("layer_norm_fwd_8x768", "layer_norm_fwd", 8, 768),
        # the activations of a training step: 16 sequences of 512 tokens
        _ln("layer_norm_fwd_8192x1024", "layer_norm_fwd", 8192, 1024),
        # the same gradient for a ragged token count and a width that is no power of two
        _ln("layer_norm_bwd_4093x1000", "layer_norm_bwd", 4093, 1000),
        # a large batch: the weight gradient is a sum over 65536 rows
        _ln("layer_norm_bwd_65536x1024", "layer_norm_bwd", 65536, 1024),
        # the activations of a feed-forward layer, forward or backward (the same call on the cotangent)
        _drop("dropout_16384x2048", 16384 * 2048, 0.1, False),
        # a ragged batch added to its residual branch
        _drop("dropout_residual_1000003", 1000003, 0.25, True),
        # the end of a sub-layer: residual + dropout, normalised for the next one
        _daln("dropout_add_layer_norm_fwd_16384x1024", "dropout_add_layer_norm_fwd", 16384, 1024, 0.1),
        # and its gradients (input, residual, weights) for an odd number of rows
        _daln("dropout_add_layer_norm_bwd_4095x768", "dropout_add_layer_norm_bwd", 4095, 768, 0.1),
        # an encoder layer over a padded batch
        _att("attention_fwd_b8_h16_t1024_d64", "attention_fwd", 8, 16, 1024, 1024, 64, ragged=True),
        # the same layer in training, with dropout on the probabilities, read as the projections leave it
        _att("attention_bwd_b8_h8_t512_d64_drop", "attention_bwd", 8, 8, 512, 512, 64, p=0.1, ragged=True, layout="bthd"),
        # a decoder layer in training: causal, an odd length, wide heads
        _att("attention_bwd_b2_h8_t2047_d128_causal", "attention_bwd", 2, 8, 2047, 2047, 128, causal=True),
        # serving: one new token of each sequence against its cache
        _att("attention_fwd_b16_h16_t1_of_8192_d64", "attention_fwd", 16, 16, 1, 8192, 64, causal=True, ragged=True),
    ]


def _spread(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm_fwd", "layer_norm_bwd", "dropout", "dropout_add_layer_norm_fwd",
                     "dropout_add_layer_norm_bwd", "attention_fwd", "attention_bwd", "attention_token"])
    if op in ("layer_norm_fwd", "layer_norm_bwd", "dropout_add_layer_norm_fwd", "dropout_add_layer_norm_bwd"):
        cols = _spread(rng, 2, 8192)
        rows = _spread(rng, 1, min(65536, (1 << 24) // cols))
        if op.startswith("layer_norm"):
            return {"op": op, "rows": rows, "cols": cols}
        return {"op": op, "rows": rows, "cols": cols, "p": rng.choice([0.1, 0.2, 0.5])}
    if op == "dropout":
        return {"op": op, "n": _spread(rng, 1, 1 << 24), "p": rng.choice([0.1, 0.25, 0.5]), "residual": rng.random() < 0.5}
    causal = rng.random() < 0.5
    D = rng.choice([16, 20, 32, 40, 63, 64, 64, 80, 96, 128])
    buckets = rng.choice([8, 16, 32, 64])
    case = {"op": op, "D": D, "causal": causal, "buckets": buckets, "max_distance": rng.choice([64, 128, 200]), "p": 0.0,
            "ragged": rng.random() < 0.5, "empty": rng.random() < 0.3, "layout": rng.choice(["bhtd", "bthd"]),
            "B": rng.randint(1, 8), "H": rng.randint(1, 12)}
    case["empty"] = case["empty"] and case["B"] > 1         # a batch has at least one sequence with something in it
    if op == "attention_token":
        case["op"] = "attention_fwd"
        case["Tq"] = rng.choice([1, 1, 1, 2, 4])
        case["Tk"] = _spread(rng, 16, 8192)
        return case
    most = 24e6 if op == "attention_bwd" else 48e6      # score elements
    side = int(math.sqrt(most / (case["B"] * case["H"])))
    case["Tk"] = _spread(rng, 2, min(2048, side))
    case["Tq"] = case["Tk"] if causal or rng.random() < 0.6 else _spread(rng, 2, min(2048, side))
    case["p"] = rng.choice([0.0, 0.1]) if op == "attention_bwd" else 0.0
    return case


def _lengths(case):
    """Key lengths of a padded batch (of the queries too where a sequence attends to itself), by the case alone."""
    B, Tk = case["B"], case["Tk"]
    lens = [Tk - (b * Tk) // (2 * B) if case["ragged"] else Tk for b in range(B)]
    if case["empty"]:
        lens[-1] = 0
    return lens


def _self_attention(case):
    return case["Tq"] == case["Tk"]


def _padded(case):
    return case["ragged"] or case["empty"]


def _offset(case):
    """Position of the first query among the keys."""
    return case["Tk"] - case["Tq"] if case["causal"] else 0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale + shift

    s = {"case": case, "op": case["op"], "rng": torch.tensor([seed * 0x9E3779B1 + 12345, seed % 1000], dtype=torch.int64, device="cuda")}
    op = case["op"]
    if "layer_norm" in op:
        R, C = case["rows"], case["cols"]
        s["gamma"], s["beta"] = randn(C, scale=0.2, shift=1.0), randn(C, scale=0.2)
        s["x"] = randn(R, C) + randn(R, 1, scale=0.5)
        if op.startswith("dropout"):
            s["residual"] = randn(R, C)
        if op.endswith("bwd"):
            # what the forward pass left: the normalised sum, its row statistics, and the cotangents
            x = s.pop("x")
            s.pop("residual", None)
            s["h"] = x
            s["mean"] = x.double().mean(1).float()
            s["rstd"] = (x.double().var(1, unbiased=False) + 1e-5).rsqrt().float()
            s["gy"] = randn(R, C, scale=0.1)
            if op.startswith("dropout"):
                s["gh"] = randn(R, C, scale=0.1)
    elif op == "dropout":
        s["x"] = randn(case["n"])
        if case["residual"]:
            s["residual"] = randn(case["n"])
    else:
        B, H, Tq, Tk, D = (case[k] for k in ("B", "H", "Tq", "Tk", "D"))
        shape = (lambda T: (B, H, T, D)) if case["layout"] == "bhtd" else (lambda T: (B, T, H, D))
        s["q"], s["k"], s["v"] = randn(*shape(Tq)), randn(*shape(Tk)), randn(*shape(Tk))
        s["table"] = randn(case["buckets"], H, scale=0.5)
        s["k_lengths"] = s["q_lengths"] = None
        if _padded(case):
            s["k_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
            s["q_lengths"] = s["k_lengths"].clone() if _self_attention(case) else None
        if op == "attention_bwd":
            s["go"] = randn(*shape(Tq), scale=0.5)
            o, lse = _attention(s)[:2]
            s["o"], s["lse"] = o, lse
    return s


# ---------------------------------------------------------------- plain forms


def _philox(g, channel, rng):
    """Eight 16-bit numbers for every group number in `g` (int64): Philox4x32 with 7 rounds, key = the seed, counter =
    (group low, group high, channel, step).  -> [..., 8]"""
    c0, c1 = g & M32, (g >> 32) & M32
    c2 = torch.full_like(g, channel)
    c3 = torch.zeros_like(g) + (rng[1] & M32)
    k0, k1 = rng[0] & M32, (rng[0] >> 32) & M32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & M32) ^ c1 ^ k0, b & M32, ((a >> 32) & M32) ^ c3 ^ k1, a & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], -1)


def _threshold(p):
    return int(round(p * 65536))


def _keep_factor(shape, p, channel, rng):
    """keep / (1 - p) for a whole array: element e of it takes 16-bit number e % 8 of group e // 8."""
    n, t = math.prod(shape), _threshold(p)
    u = _philox(torch.arange(-(-n // 8), dtype=torch.int64, device=rng.device), channel, rng)
    return (u.reshape(-1)[:n] >= t).float().mul_(65536.0 / (65536 - t)).reshape(shape)


def _normalise(h, gamma, beta, eps=1e-5):
    mean = h.mean(1, keepdim=True)
    xc = h - mean
    rstd = ((xc * xc).mean(1, keepdim=True) + eps).rsqrt()
    return xc * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def _normalise_back(h, gamma, mean, rstd, gy):
    xhat = (h - mean[:, None]) * rstd[:, None]
    gg = gy * gamma
    gx = (gg - gg.mean(1, keepdim=True) - xhat * (gg * xhat).mean(1, keepdim=True)) * rstd[:, None]
    return gx, (gy * xhat).sum(0), gy.sum(0)


def _buckets(rel, buckets, max_distance, bidirectional):
    """Bucket of each relative position (key minus query): the distances below half a side's buckets one by one, then
    logarithmic ones up to max_distance, the last for everything beyond."""
    side = buckets // 2 if bidirectional else buckets
    n = rel.abs() if bidirectional else (-rel).clamp(min=0)
    first = side // 2
    # 64 bits, and a nudge far below the gap between neighbouring distances: the borders fall on whole distances
    far = torch.log(n.clamp(min=1).double() / first) / math.log(max_distance / first) * (side - first)
    b = torch.where(n < first, n, (first + torch.floor(far + 1e-9).long()).clamp(max=side - 1))
    return b + torch.where(rel > 0, side, 0) if bidirectional else b


def _seen(case, q_lengths, k_lengths, device):
    """[B or 1, 1, Tq, Tk]: which keys a query may see."""
    Tq, Tk = case["Tq"], case["Tk"]
    i, j = torch.arange(Tq, device=device)[:, None], torch.arange(Tk, device=device)[None, :]
    seen = torch.ones(1, 1, Tq, Tk, dtype=torch.bool, device=device)
    if case["causal"]:
        seen = seen & (j <= i + _offset(case))
    if k_lengths is not None:
        seen = seen & (j < k_lengths[:, None, None, None])
    if q_lengths is not None:
        seen = seen & (i < q_lengths[:, None, None, None])
    return seen


def _rel_bucket(case, device):
    rel = torch.arange(1 - case["Tq"], case["Tk"], device=device) - _offset(case)      # by j - i, ascending
    return _buckets(rel, case["buckets"], case["max_distance"], not case["causal"])


def _attention(s):
    """(o, lse, scores' probabilities, keep factors) in 32 bits; o in the case's layout."""
    case = s["case"]
    q, k, v = (t if case["layout"] == "bhtd" else t.transpose(1, 2) for t in (s["q"], s["k"], s["v"]))
    Tq, Tk, D = case["Tq"], case["Tk"], case["D"]
    by_rel = s["table"].t()[:, _rel_bucket(case, q.device)]                            # [H, Tq + Tk - 1]
    at = torch.arange(Tk, device=q.device)[None, :] - torch.arange(Tq, device=q.device)[:, None] + Tq - 1
    a = torch.matmul(q * D ** -0.5, k.transpose(2, 3)) + by_rel[:, at]
    a = a.masked_fill(~_seen(case, s["q_lengths"], s["k_lengths"], q.device), -math.inf)
    top = a.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(a - top)
    total = e.sum(3, keepdim=True)
    prob = e / torch.where(total == 0, 1.0, total)
    keep = _attention_keep(case, s["rng"]) if case["p"] else None
    o = torch.matmul(prob if keep is None else prob * keep, v)
    lse = (top + torch.log(total))[..., 0]
    return (o if case["layout"] == "bhtd" else o.transpose(1, 2).contiguous()), lse, prob, keep


def _attention_keep(case, rng):
    """Keep factors [B, H, Tq, Tk]: row r = (b * H + h) * Tq + i has two groups of eight keys for each 16 keys, the first
    with keys 0-3 and 8-11 of them, the second with keys 4-7 and 12-15."""
    B, H, Tq, Tk, t = case["B"], case["H"], case["Tq"], case["Tk"], _threshold(case["p"])
    blocks = -(-Tk // 16)
    u = _philox(torch.arange(B * H * Tq * blocks * 2, dtype=torch.int64, device=rng.device), 0, rng)
    u = u.reshape(B, H, Tq, blocks, 2, 2, 4).transpose(4, 5).reshape(B, H, Tq, blocks * 16)[..., :Tk]
    return (u >= t).float().mul_(65536.0 / (65536 - t))


def _attention_back(s):
    case = s["case"]
    o, lse, prob, keep = _attention_from_lse(s)
    q, k, v, go = (t if case["layout"] == "bhtd" else t.transpose(1, 2) for t in (s["q"], s["k"], s["v"], s["go"]))
    seen_q = None if s["q_lengths"] is None else (
        torch.arange(case["Tq"], device=q.device)[None, None, :, None] < s["q_lengths"][:, None, None, None])
    if seen_q is not None:
        go = go * seen_q                                          # padded queries give nothing
    Tq, Tk, D = case["Tq"], case["Tk"], case["D"]
    gp = torch.matmul(go, v.transpose(2, 3))
    kept = prob
    if keep is not None:
        gp, kept = gp * keep, prob * keep
    gv = torch.matmul(kept.transpose(2, 3), go)
    ga = prob * (gp - (go * o).sum(3, keepdim=True))
    gq = torch.matmul(ga, k) * D ** -0.5
    gk = torch.matmul(ga.transpose(2, 3), q) * D ** -0.5
    # sums along the diagonals: rows in reverse order, each padded by Tq zeros, read with a row shorter by one
    H = case["H"]
    skew = torch.cat([ga.sum(0).flip(1), torch.zeros(H, Tq, Tq, device=q.device)], 2).reshape(H, -1)
    by_rel = skew[:, : Tq * (Tk + Tq) - Tq].reshape(H, Tq, Tk + Tq - 1).sum(1, dtype=torch.float64)
    onehot = (_rel_bucket(case, q.device)[:, None] == torch.arange(case["buckets"], device=q.device)).double()
    gtable = torch.matmul(by_rel, onehot).t().float().contiguous()
    if case["layout"] != "bhtd":
        gq, gk, gv = (t.transpose(1, 2).contiguous() for t in (gq, gk, gv))
    return gq, gk, gv, gtable


def _attention_from_lse(s):
    """(o, lse, probabilities, keep factors) with the probabilities formed from the saved row statistics."""
    case = s["case"]
    q, k = (t if case["layout"] == "bhtd" else t.transpose(1, 2) for t in (s["q"], s["k"]))
    o = s["o"] if case["layout"] == "bhtd" else s["o"].transpose(1, 2)
    Tq, Tk, D = case["Tq"], case["Tk"], case["D"]
    by_rel = s["table"].t()[:, _rel_bucket(case, q.device)]
    at = torch.arange(Tk, device=q.device)[None, :] - torch.arange(Tq, device=q.device)[:, None] + Tq - 1
    a = torch.matmul(q * D ** -0.5, k.transpose(2, 3)) + by_rel[:, at]
    prob = torch.exp(a - s["lse"][..., None])
    prob = prob.masked_fill(~_seen(case, s["q_lengths"], s["k_lengths"], q.device), 0.0)
    return o, s["lse"], prob, (_attention_keep(case, s["rng"]) if case["p"] else None)


def _run_plain(s):
    op, case = s["op"], s["case"]
    if op == "layer_norm_fwd":
        return _normalise(s["x"], s["gamma"], s["beta"])
    if op == "layer_norm_bwd":
        return _normalise_back(s["h"], s["gamma"], s["mean"], s["rstd"], s["gy"])
    if op == "dropout":
        y = s["x"] * _keep_factor(s["x"].shape, case["p"], 0, s["rng"])
        return y + s["residual"] if case["residual"] else y
    if op == "dropout_add_layer_norm_fwd":
        h = s["x"] * _keep_factor(s["x"].shape, case["p"], 0, s["rng"]) + s["residual"]
        y, mean, rstd = _normalise(h, s["gamma"], s["beta"])
        return y, h, mean, rstd
    if op == "dropout_add_layer_norm_bwd":
        gh, ggamma, gbeta = _normalise_back(s["h"], s["gamma"], s["mean"], s["rstd"], s["gy"])
        gh = gh + s["gh"]
        return gh * _keep_factor(gh.shape, case["p"], 0, s["rng"]), gh, ggamma, gbeta
    if op == "attention_fwd":
        return _attention(s)[:2]
    return _attention_back(s)


# ---------------------------------------------------------------- the framework's calls


def _arrays(s):
    """The state's tensors as device arrays of the framework (views, no copies), and arrays for the results, which a
    program keeps from step to step."""
    if "own" in s:
        return s["own"]
    from cgt_amd import gpuarray

    def like(*names):
        return tuple(torch.empty_like(s[n]) for n in names)

    op = s["op"]
    rows = s["h"].shape[0] if "h" in s else s["x"].shape[0] if "x" in s and s["x"].dim() == 2 else 0
    stat = lambda: torch.empty(rows, device="cuda")      # noqa: E731
    results = {
        "layer_norm_fwd": lambda: like("x") + (stat(), stat()),
        "layer_norm_bwd": lambda: like("h", "gamma", "gamma"),
        "dropout": lambda: like("x"),
        "dropout_add_layer_norm_fwd": lambda: like("x", "x") + (stat(), stat()),
        "dropout_add_layer_norm_bwd": lambda: like("h", "h", "gamma", "gamma"),
        "attention_fwd": lambda: like("q") + (torch.empty(*(s["case"][k] for k in ("B", "H", "Tq")), device="cuda"),),
        "attention_bwd": lambda: like("q", "k", "v", "table"),
    }[op]()
    a = {n: gpuarray.as_gpuarray(t) for n, t in s.items() if isinstance(t, torch.Tensor)}
    s["own"] = (a, results, tuple(gpuarray.as_gpuarray(t) for t in results))
    return s["own"]


def _run_own(s):
    from cgt_amd import kernels
    op, case = s["op"], s["case"]
    a, results, out = _arrays(s)
    if op == "layer_norm_fwd":
        kernels.layer_norm_fwd(a["x"], a["gamma"], a["beta"], out=out)
    elif op == "layer_norm_bwd":
        kernels.layer_norm_bwd(a["h"], a["gamma"], a["mean"], a["rstd"], a["gy"], out=out)
    elif op == "dropout":
        kernels.dropout(a["x"], case["p"], a["rng"], residual=a.get("residual"), out=out[0])
    elif op == "dropout_add_layer_norm_fwd":
        kernels.dropout_add_layer_norm_fwd(a["x"], a["residual"], a["gamma"], a["beta"], case["p"], a["rng"], out=out)
    elif op == "dropout_add_layer_norm_bwd":
        kernels.dropout_add_layer_norm_bwd(a["h"], a["gamma"], a["mean"], a["rstd"], a["gy"], a["gh"], case["p"], a["rng"], out=out)
    else:
        more = dict(causal=case["causal"], max_distance=case["max_distance"], q_offset=_offset(case), q_lengths=a.get("q_lengths"),
                    k_lengths=a.get("k_lengths"), p=case["p"], rng=a["rng"], layout=case["layout"], out=out)
        if op == "attention_fwd":
            kernels.rel_attention_fwd(a["q"], a["k"], a["v"], a["table"], **more)
        else:
            kernels.rel_attention_bwd(a["q"], a["k"], a["v"], a["table"], a["o"], a["lse"], a["go"], **more)
    return results if len(results) > 1 else results[0]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- work


def _pairs(case):
    """Query-key pairs that a pass has to look at, per head."""
    n = 0
    for length in _lengths(case):
        Tq = min(case["Tq"], length) if _self_attention(case) else case["Tq"]
        if not case["causal"]:
            n += Tq * length
        else:
            first = _offset(case)
            n += sum(min(length, first + i + 1) for i in range(Tq))
    return n


def work(case):
    op = case["op"]
    if "layer_norm" in op:
        n, R, C = case["rows"] * case["cols"], case["rows"], case["cols"]
        arrays = {"layer_norm_fwd": 2, "layer_norm_bwd": 3, "dropout_add_layer_norm_fwd": 4, "dropout_add_layer_norm_bwd": 5}[op]
        return {"bytes": 4.0 * (arrays * n + 2 * R + 2 * C), "flops": (14.0 if op.endswith("bwd") else 8.0) * n}
    if op == "dropout":
        return {"bytes": 4.0 * case["n"] * (3 if case["residual"] else 2), "flops": 2.0 * case["n"]}
    B, H, Tq, Tk, D = (case[k] for k in ("B", "H", "Tq", "Tk", "D"))
    pairs = H * _pairs(case)
    keys = H * sum(_lengths(case))
    queries = H * sum(min(Tq, n) if _self_attention(case) else Tq for n in _lengths(case))
    if op == "attention_fwd":       # q, o and the row statistics; k and v
        return {"bytes": 4.0 * (queries * D + B * H * Tq * (D + 1) + 2 * keys * D), "flops": 4.0 * D * pairs}
    # q, o, go and the statistics, k and v; gq, gk, gv
    return {"bytes": 4.0 * (queries * (3 * D + 1) + 2 * keys * D + B * H * (Tq + 2 * Tk) * D), "flops": 10.0 * D * pairs}


# ---------------------------------------------------------------- the definition in 64 bits


def _random16(groups, channel, rng):
    """The generator in unsigned numpy arithmetic -> [groups, 8] of uint16."""
    seed, step = (int(v) for v in rng.tolist())
    mask, sh = np.uint64(M32), np.uint64(32)
    index = np.arange(groups, dtype=np.uint64)
    c = [index & mask, index >> sh, np.full(groups, channel, np.uint64), np.full(groups, step & M32, np.uint64)]
    key = [seed & M32, (seed >> 32) & M32]
    for _ in range(7):
        x, y = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(y >> sh) ^ c[1] ^ np.uint64(key[0]), y & mask, (x >> sh) ^ c[3] ^ np.uint64(key[1]), x & mask]
        key = [(key[0] + 0x9E3779B9) & M32, (key[1] + 0xBB67AE85) & M32]
    words = np.stack([w.astype(np.uint32) for w in c], 1)
    return np.ascontiguousarray(words).view("<u2")


def _kept(n, p, rng):
    t = _threshold(p)
    u = _random16((n + 7) // 8, 0, rng).reshape(-1)[:n]
    return torch.from_numpy((u >= t).astype(np.float64) * (65536.0 / (65536 - t))).to(rng.device)


def _exact_buckets(case):
    """By whole numbers: distance n is at or beyond log bucket e of a side when (n / first)^(side - first) >= (max / first)^e."""
    side = case["buckets"] // (1 if case["causal"] else 2)
    first, most = side // 2, case["max_distance"]
    found = []
    for rel in range(1 - case["Tq"] - _offset(case), case["Tk"] - _offset(case)):
        n = abs(rel) if not case["causal"] else max(0, -rel)
        b = n
        if n >= first:
            e, n = 0, min(n, most)
            while e + 1 < side - first and n ** (side - first) * first ** (e + 1) >= most ** (e + 1) * first ** (side - first):
                e += 1
            b = first + e
        found.append(b + (side if rel > 0 and not case["causal"] else 0))
    return found


def _exact_norm(h, gamma, beta):
    var, mean = torch.var_mean(h, 1, correction=0, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + 1e-5)
    return (h - mean) * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def _exact_attention(case, s, q, k, v, table):
    B, H, Tq, Tk, D = (case[n] for n in ("B", "H", "Tq", "Tk", "D"))
    if case["layout"] == "bthd":
        q, k, v = q.permute(0, 2, 1, 3), k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    bucket = torch.tensor(_exact_buckets(case), device=q.device)
    rel = torch.arange(Tk, device=q.device) - torch.arange(Tq, device=q.device)[:, None] + (Tq - 1)
    a = q @ k.mT / math.sqrt(D) + table[bucket[rel]].permute(2, 0, 1)
    lens = torch.tensor(_lengths(case), device=q.device).view(B, 1, 1, 1)
    hidden = torch.arange(Tk, device=q.device) >= lens
    if _self_attention(case) and _padded(case):
        hidden = hidden | (torch.arange(Tq, device=q.device)[:, None] >= lens)
    if case["causal"]:
        hidden = hidden | torch.triu(torch.ones(Tq, Tk, dtype=torch.bool, device=q.device), diagonal=1 + _offset(case))
    hidden = hidden.expand(B, 1, Tq, Tk)
    blind = hidden.all(3, keepdim=True)
    a = torch.where(hidden, -math.inf, a)
    lse = torch.logsumexp(torch.where(blind, 0.0, a), 3, keepdim=True)
    prob = torch.where(hidden, 0.0, torch.exp(torch.where(hidden, 0.0, a) - lse))
    if case["p"]:
        t, blocks = _threshold(case["p"]), (Tk + 15) // 16
        u = _random16(B * H * Tq * blocks * 2, 0, s["rng"])
        j = np.arange(Tk)
        u = u.reshape(B * H * Tq, blocks * 16)[:, (j // 16) * 16 + (j // 4 % 2) * 8 + j // 8 % 2 * 4 + j % 4]
        keep = torch.from_numpy(u >= t).to(q.device).view(B, H, Tq, Tk)
        prob = prob * keep * (65536.0 / (65536 - t))
    o = prob @ v
    lse = torch.where(blind, -math.inf, lse)[..., 0]
    return (o if case["layout"] == "bhtd" else o.permute(0, 2, 1, 3)), lse


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {n: t.double() for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if op == "layer_norm_fwd":
        return _exact_norm(d["x"], d["gamma"], d["beta"])
    if op == "dropout":
        y = _kept(case["n"], case["p"], s["rng"]) * d["x"]
        return y + d["residual"] if case["residual"] else y
    if op == "dropout_add_layer_norm_fwd":
        h = d["residual"] + _kept(d["x"].numel(), case["p"], s["rng"]).view_as(d["x"]) * d["x"]
        y, mean, rstd = _exact_norm(h, d["gamma"], d["beta"])
        return y, h, mean, rstd
    if op.endswith("layer_norm_bwd"):
        h, gamma, beta = d["h"].requires_grad_(), d["gamma"].requires_grad_(), torch.zeros_like(d["gamma"]).requires_grad_()
        y = _exact_norm(h, gamma, beta)[0]
        gh, ggamma, gbeta = torch.autograd.grad(y, (h, gamma, beta), d["gy"])
        if op == "layer_norm_bwd":
            return gh, ggamma, gbeta
        gh = gh + d["gh"]
        return _kept(gh.numel(), case["p"], s["rng"]).view_as(gh) * gh, gh, ggamma, gbeta
    if op == "attention_fwd":
        return _exact_attention(case, s, d["q"], d["k"], d["v"], d["table"])
    wrt = tuple(d[n].requires_grad_() for n in ("q", "k", "v", "table"))
    o, _lse = _exact_attention(case, s, *wrt)
    return torch.autograd.grad(o, wrt, d["go"])
