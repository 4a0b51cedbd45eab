"""Local attention with a learned relative position bias: what is measured, and its plain forms.

Three operators that are used together.  i is a query, j a key; a query stands at position
p = i + (n_k - n_q) (queries end where the keys end), and delta = p - j.

* ``relative_position_bias``: bias[h, i, j] = pos_weight[h, bucket(delta)], added to logits or costs;
  its gradient sums d bias over every pair of a bucket.
* ``flash_window_attn``: softmax over the visible keys of q.k * scale + pos_weight[h, bucket(delta)].
  A key is visible when it is not masked, not in the future (causal), and either within the window
  (0 <= delta < window; |delta| < window without causal) or one of the first `sinks` keys.  A query
  that sees no key gives zeros.  Its training step gives the gradients of q, k, v and pos_weight.
* ``window_attn_decode``: the same attention for the one newest token of each sequence over a cache,
  with a length for each sequence.
"""

import functools
import math
import os
import sys

import torch

own = False

# the package's root, as tests and examples put it on the path
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepfold-linear_b200")
if PACKAGE not in sys.path:
    sys.path.insert(0, PACKAGE)

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases
def _bias(name, H, n_q, n_k, dtype, kind, buckets, distance, grad):
    return dict(name=name, op="bias", H=H, n_q=n_q, n_k=n_k, dtype=dtype, kind=kind, buckets=buckets,
                distance=distance, grad=grad)


def _attn(name, B, H, H_kv, n_q, n_k, d, dtype, window, sinks, causal, kind, buckets, distance, shortest, layout, grad):
    return dict(name=name, op="attn", B=B, H=H, H_kv=H_kv, n_q=n_q, n_k=n_k, d=d, dtype=dtype, window=window,
                sinks=sinks, causal=causal, kind=kind, buckets=buckets, distance=distance, shortest=shortest,
                layout=layout, grad=grad)


def _decode(name, B, H, H_kv, n_k, d, dtype, window, sinks, kind, buckets, distance, shortest, layout):
    return dict(name=name, op="decode", B=B, H=H, H_kv=H_kv, n_k=n_k, d=d, dtype=dtype, window=window, sinks=sinks,
                kind=kind, buckets=buckets, distance=distance, shortest=shortest, layout=layout)


def listed():
    return [
        # the bias of one trunk block at the smallest configuration (H = 8, N = 384), with the position
        # rule of compute_bins within a chain: one call before a dense-cost solve
        _bias("bias 384", 8, 384, 384, "bf16", "clip", 65, 32, False),
        # cross attention between two ragged lengths, forward and gradient, 32-bit parameters
        _bias("bias 1000x1537 step", 4, 1000, 1537, "f32", "log", 32, 128, True),
        # the long-sequence configuration (H = 16, N = 8192): forward and gradient at full size
        _bias("bias 8192 step", 16, 8192, 8192, "bf16", "log2", 32, 128, True),
        # one small forward (B = 2, H = 8, N = 384, d = 32): latency counts
        _attn("attn 384", 2, 8, 8, 384, 384, 32, "bf16", 128, 4, True, "log", 32, 128, -1, "bhnd", False),
        # a padded batch (B = 8, H = 16, d = 64, N = 1024, lengths from 64): an encoder's local layer
        _attn("attn 1024 padded", 8, 16, 16, 1024, 1024, 64, "bf16", 256, 0, False, "clip", 65, 32, 64, "bnhd", False),
        # long context, a wide window: prefill
        _attn("attn 8192 wide", 1, 16, 4, 8192, 8192, 64, "bf16", 4096, 4, True, "log", 32, 128, -1, "bnhd", False),
        # a training step of the padded batch: both directions of a bidirectional layer
        _attn("attn 1024 padded step", 8, 16, 16, 1024, 1024, 64, "bf16", 256, 1, False, "log2", 32, 128, 64, "bnhd", True),
        # an odd length, shared key heads, a head dim of 40, 16-bit floats: a fine-tuning step
        _attn("attn 1537 step", 3, 12, 4, 1537, 1537, 40, "f16", 200, 3, True, "log", 32, 128, -1, "bnhd", True),
        # a training step at the long-sequence configuration (H = 16, N = 8192, d = 64)
        _attn("attn 8192 step", 1, 16, 16, 8192, 8192, 64, "bf16", 1024, 4, True, "log", 32, 128, -1, "bhnd", True),
        # one sequence, one new token: the smallest call of a decoding loop
        _decode("decode 1", 1, 16, 4, 8192, 64, "bf16", 1024, 4, "log", 32, 128, 5001, "bhnd"),
        # a serving batch of ragged sequences, from an empty one to a full cache, a window of half of it
        _decode("decode 64", 64, 16, 4, 8192, 64, "bf16", 4096, 4, "log", 32, 128, 0, "bnhd"),
        # a few long sequences without a window: the whole cache is read
        _decode("decode 12 long", 12, 32, 8, 32768, 64, "f16", 0, 0, "log", 32, 128, 20001, "bhnd"),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind, buckets, distance = rng.choice(
        [("log", 32, 128), ("log2", 32, 128), ("clip", 65, 32), ("log", 16, rng.randint(40, 900)),
         ("log2", 24, rng.randint(40, 600)), ("clip", 2 * 19 + 1, 19)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    op = rng.choice(["bias", "attn", "attn", "decode"])
    d = rng.choice([16, 24, 32, 40, 64, 64])
    H_kv = rng.choice([1, 2, 3, 4, 8])
    H = H_kv * rng.choice([1, 1, 2, 3, 4])
    layout = rng.choice(["bhnd", "bnhd"])
    window = rng.choice([0, _between(rng, 1, 2048), _between(rng, 16, 1024)])
    sinks = rng.choice([0, 0, 1, 4, rng.randint(1, 40)])
    if op == "bias":
        n_q, n_k = _between(rng, 1, 4096), _between(rng, 1, 4096)
        case = _bias("", H, n_q, n_k, dtype, kind, buckets, distance, rng.random() < 0.5)
    elif op == "decode":
        n_k = _between(rng, 1, 24000)
        B = _between(rng, 1, max(1, min(64, 500000 // (n_k * H_kv))))
        case = _decode("", B, H, H_kv, n_k, d, dtype, window, sinks, kind, buckets, distance,
                       rng.randint(0, n_k), layout)
    else:
        grad = rng.random() < 0.5
        least = 8 if grad else 1  # a query that sees one key has a gradient of exactly nothing: no measure of any code
        n_k = _between(rng, least, 4096)
        n_q = n_k if rng.random() < 0.7 else _between(rng, least, n_k)
        window = max(window, least) if window else 0
        B = rng.randint(1, 4)
        causal = rng.random() < 0.6
        while B > 1 and B * H * n_q * n_k > 2e8:
            B -= 1
        if H * n_q * n_k > 2e8:
            H = H_kv
        case = _attn("", B, H, H_kv, n_q, n_k, d, dtype, window, sinks, causal, kind, buckets, distance,
                     rng.choice([-1, -1, rng.randint(0 if least == 1 else least, n_k)]), layout, grad)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """The sequences' lengths: from the shortest to the full one, spread evenly (the same for every seed)."""
    B, n, lo = case["B"], case["n_k"], case["shortest"]
    return [lo + (n - lo) * b // max(1, B - 1) for b in range(B)]


def _buckets_of(case):
    """The bucket of delta = -distance .. distance (those further off have the end's bucket)."""
    D, n = case["distance"], case["buckets"]
    delta = torch.arange(-D, D + 1, dtype=torch.float64)
    if case["kind"] == "clip":
        return (delta + D).long()
    half = n // 2 if case["kind"] == "log2" else n
    first = torch.where(delta < 0, n - half, 0) if case["kind"] == "log2" else torch.zeros_like(delta).long()
    far = delta.abs() if case["kind"] == "log2" else delta.clamp(min=0)
    exact_up_to = half // 2
    wide = torch.log(far.clamp(min=1) / exact_up_to) / math.log(D / exact_up_to) * (half - exact_up_to)
    wide = (exact_up_to + torch.floor(wide + 1e-9)).clamp(max=half - 1)
    return first + torch.where(far < exact_up_to, far, wide).long()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = dict(case)
    if own:
        from deepfold.model.position_encoding import RelativeBuckets  # the table that a model's module keeps

        s["table"] = RelativeBuckets(_buckets_of(case).tolist(), num_buckets=case["buckets"], device="cuda")
    else:
        s["table"] = _buckets_of(case).cuda()
    if case["op"] == "bias":
        s["pos_weight"] = normal(case["H"], case["buckets"], scale=0.5)
        if case["grad"]:
            s["pos_weight"].requires_grad_()
            s["d_bias"] = normal(case["H"], case["n_q"], case["n_k"])
        return s

    def heads(H, n):  # (B, H, n, d), in memory as (B, H, n, d) or as a projection leaves it, (B, n, H, d)
        B, d = case["B"], case["d"]
        return normal(B, n, H, d).transpose(1, 2) if case["layout"] == "bnhd" else normal(B, H, n, d)

    s["k"], s["v"] = heads(case["H_kv"], case["n_k"]), heads(case["H_kv"], case["n_k"])
    s["pos_weight"] = normal(case["H"], case["buckets"], scale=0.5)
    lengths = torch.tensor(_lengths(case) if case["shortest"] >= 0 else [case["n_k"]] * case["B"], dtype=torch.int32)
    if case["op"] == "decode":
        s["q"] = normal(case["B"], case["H"], case["d"])
        s["lengths"] = lengths.cuda()
        return s
    s["q"] = heads(case["H"], case["n_q"])
    s["mask"] = None
    if case["shortest"] >= 0:
        s["mask"] = (torch.arange(case["n_k"])[None] < lengths[:, None]).cuda()
    if case["grad"]:
        s["d_o"] = heads(case["H"], case["n_q"])
        for name in ("q", "k", "v", "pos_weight"):
            s[name].requires_grad_()
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"bias": _plain_bias, "attn": _plain_attn, "decode": _plain_decode}[state["op"]](state)


def _run_own(s):
    from deepfold.model.kernels.flash_window_attn import flash_window_attn, window_attn_decode
    from deepfold.model.position_encoding import relative_position_bias

    window = s.get("window") or None
    if s["op"] == "bias":
        bias = relative_position_bias(s["pos_weight"], s["table"], s["n_q"], s["n_k"])
        if not s["grad"]:
            return {"bias": bias}
        (d_w,) = torch.autograd.grad(bias, [s["pos_weight"]], s["d_bias"])
        return {"bias": bias, "d_pos_weight": d_w}
    if s["op"] == "decode":
        return {"o": window_attn_decode(s["q"], s["k"], s["v"], s["lengths"], window=window, sinks=s["sinks"],
                                        pos_weight=s["pos_weight"], buckets=s["table"])}
    o = flash_window_attn(s["q"], s["k"], s["v"], window=window, sinks=s["sinks"], causal=s["causal"],
                          pos_weight=s["pos_weight"], buckets=s["table"], mask=s["mask"])
    if not s["grad"]:
        return {"o": o}
    d_q, d_k, d_v, d_w = torch.autograd.grad(o, [s["q"], s["k"], s["v"], s["pos_weight"]], s["d_o"])
    return {"o": o, "d_q": d_q, "d_k": d_k, "d_v": d_v, "d_pos_weight": d_w}


def _delta(n_q, n_k):
    return (torch.arange(n_q, device="cuda") + (n_k - n_q))[:, None] - torch.arange(n_k, device="cuda")[None]


def _bias_of(s, delta):
    D = s["distance"]
    return s["pos_weight"].float()[:, s["table"][delta.clamp(-D, D) + D]]


def _d_bias_to_weight(s, d_bias):
    """Sums d_bias (H, n_q, n_k) over its diagonals (rows skewed by a pad), then over the diagonals of a bucket."""
    H, n_q, n_k = d_bias.shape
    x = torch.nn.functional.pad(d_bias.flip(2), (0, n_q)).reshape(H, -1)
    x = x[:, :n_q * (n_k + n_q - 1)].reshape(H, n_q, n_k + n_q - 1)  # [i, c]: j = n_k - 1 - (c - i)
    by_diagonal = x.sum(1)
    delta = torch.arange(n_k + n_q - 1, device="cuda") - (n_k - 1) + (n_k - n_q)
    D = s["distance"]
    hot = torch.nn.functional.one_hot(s["table"][delta.clamp(-D, D) + D], s["buckets"]).float()
    return by_diagonal @ hot


def _plain_bias(s):
    t = TYPES[s["dtype"]]
    bias = _bias_of(s, _delta(s["n_q"], s["n_k"])).to(t)
    if not s["grad"]:
        return {"bias": bias}
    return {"bias": bias, "d_pos_weight": _d_bias_to_weight(s, s["d_bias"].float()).to(t)}


def _softmax(x, visible):
    x = torch.where(visible, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _visible(s, delta, j):
    near = torch.ones_like(delta, dtype=torch.bool)
    if s["window"]:
        near = (delta.abs() < s["window"]) | (j < s["sinks"])
    return near & (delta >= 0) if s.get("causal", True) else near


def _plain_attn(s):
    t = TYPES[s["dtype"]]
    B, H, G, d = s["B"], s["H"], s["H"] // s["H_kv"], s["d"]
    q, k, v = (x.float() for x in (s["q"], s["k"], s["v"]))
    k, v = (x.repeat_interleave(G, 1) for x in (k, v))
    delta = _delta(s["n_q"], s["n_k"])
    visible = _visible(s, delta, torch.arange(s["n_k"], device="cuda")[None])
    if s["mask"] is not None:
        visible = visible & s["mask"][:, None, None, :]
    scale = d ** -0.5
    p = _softmax(q @ k.transpose(2, 3) * scale + _bias_of(s, delta), visible)
    o = p @ v
    if not s["grad"]:
        return {"o": o.to(t)}
    d_o = s["d_o"].float()
    d_v = p.transpose(2, 3) @ d_o
    d_s = p * (d_o @ v.transpose(2, 3) - (d_o * o).sum(-1, keepdim=True))
    d_q, d_k = d_s @ k * scale, d_s.transpose(2, 3) @ q * scale
    d_k, d_v = (x.reshape(B, H // G, G, s["n_k"], d).sum(2) for x in (d_k, d_v))
    return {"o": o.to(t), "d_q": d_q.to(t), "d_k": d_k.to(t), "d_v": d_v.to(t),
            "d_pos_weight": _d_bias_to_weight(s, d_s.sum(0)).to(t)}


def _plain_decode(s):
    B, H, K, d = s["B"], s["H"], s["H_kv"], s["d"]
    q, k, v = s["q"].float().reshape(B, K, H // K, d), s["k"].float(), s["v"].float()
    j = torch.arange(s["n_k"], device="cuda")[None]
    delta = s["lengths"].long()[:, None] - 1 - j  # (B, n_k)
    bias = _bias_of(s, delta).transpose(0, 1).reshape(B, K, H // K, s["n_k"])
    p = _softmax(q @ k.transpose(2, 3) * d ** -0.5 + bias, _visible(s, delta, j)[:, None, None])
    return {"o": (p @ v).reshape(B, H, d).to(TYPES[s["dtype"]])}


# ---------------------------------------------------------------- what a pass cannot do without
@functools.lru_cache(maxsize=None)
def _pairs(n_q, n_k, window, sinks, causal, length):
    """Visible (query, key) pairs of one head, keys from `length` on masked."""
    p = torch.arange(n_q, dtype=torch.int64) + (n_k - n_q)
    top = torch.full_like(p, length) if not causal else (p + 1).clamp(0, length)
    if not window:
        return int(top.sum())
    if not causal:
        top = (p + window).clamp(0, length)
    low = (p - window + 1).clamp(min=0).minimum(top)
    first = torch.full_like(p, min(sinks, length)) if not causal else (p + 1).clamp(0, min(sinks, length))
    return int((top - low).sum() + first.minimum(low).sum())


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "bias":
        pairs = case["H"] * case["n_q"] * case["n_k"]
        table = case["H"] * case["buckets"] * size
        passes = 2 if case["grad"] else 1  # the bias is written; d bias is read, an addition for each pair
        return {"bytes": passes * (pairs * size + table), "flops": (passes - 1) * pairs}
    B, H, K, n_k, d = (case[x] for x in ("B", "H", "H_kv", "n_k", "d"))
    lengths = _lengths(case) if case["shortest"] >= 0 else [n_k] * B
    if case["op"] == "decode":
        seen = sum(_pairs(1, x, case["window"], case["sinks"], True, x) for x in lengths)
        return {"bytes": (2 * seen * K + 2 * B * H) * d * size + H * case["buckets"] * size, "flops": 4 * seen * H * d}
    n_q = case["n_q"]
    seen = H * sum(_pairs(n_q, n_k, case["window"], case["sinks"], case["causal"], x) for x in lengths)
    rows, keys = B * H * n_q * d * size, B * K * n_k * d * size
    table = H * case["buckets"] * size
    if not case["grad"]:
        return {"bytes": 2 * rows + 2 * keys + table, "flops": 4 * seen * d}
    # forward: q, k, v in, o out; backward: q, k, v, o, d_o in, d_q, d_k, d_v out; two and five products
    return {"bytes": (2 * rows + 2 * keys) + (4 * rows + 4 * keys) + 3 * table, "flops": 14 * seen * d}


# ---------------------------------------------------------------- in 64 bits, from the definition
def _bucket_by_rule(case, delta):
    """The bucket of one distance, in whole numbers."""
    D, n = case["distance"], case["buckets"]
    if case["kind"] == "clip":
        return max(-D, min(D, delta)) + D
    at, half = 0, n
    if case["kind"] == "log2":
        half = n // 2
        at = n - half if delta < 0 else 0
        delta = abs(delta)
    e, x = half // 2, min(max(delta, 0), D)
    if x < e:
        return at + x
    m, step = half - e, 0  # the largest step with (x / e)^m >= (D / e)^step
    while step + 1 < m and x ** m * e ** (step + 1) >= D ** (step + 1) * e ** m:
        step += 1
    return at + e + step


def exact(case, seed):
    s = prepare(case, seed)
    w = s["pos_weight"].detach().double()
    n_k = case["n_k"]
    n_q = case.get("n_q", 1)

    def row_table(lo, hi):  # bucket of delta = lo .. hi - 1
        return torch.tensor([_bucket_by_rule(case, x) for x in range(lo, hi)], device="cuda")

    def spread(table, lo, first, rows):  # [i, j] -> table[(first + i - j) - lo]
        i, j = torch.arange(rows, device="cuda"), torch.arange(n_k, device="cuda")
        return table[first + i[:, None] - j[None, :] - lo]

    if case["op"] == "bias":
        first = n_k - n_q
        buckets = spread(row_table(first - n_k + 1, first + n_q), first - n_k + 1, first, n_q)
        out = {"bias": torch.stack([x[buckets].to(torch.float64 if case["dtype"] == "f32" else torch.float32) for x in w])
               if n_q * n_k * case["H"] < 1e8 else None}
        if case["grad"]:
            d_w = torch.zeros_like(w)
            for h in range(case["H"]):
                for i0 in range(0, n_q, 1024):
                    at = buckets[i0:i0 + 1024].reshape(-1)
                    d_w[h] += torch.bincount(at, s["d_bias"][h, i0:i0 + 1024].double().reshape(-1), case["buckets"])
            out["d_pos_weight"] = d_w
        return out

    B, H, G, d = case["B"], case["H"], case["H"] // case["H_kv"], case["d"]
    decode = case["op"] == "decode"
    grad = not decode and case["grad"]
    q, k, v = (s[x].detach().double() for x in ("q", "k", "v"))
    q = q[:, :, None] if decode else q
    o = torch.zeros(B, H, n_q, d, dtype=torch.float64, device="cuda")
    if grad:
        d_q, d_k, d_v, d_w = (torch.zeros_like(x) for x in (q, k, v, w))
        d_o = s["d_o"].double()
    j = torch.arange(n_k, device="cuda")
    lengths = s["lengths"].tolist() if decode else [n_k - n_q + 1] * B
    lo = min(min(lengths) - 1, n_k - n_q) - n_k + 1
    table = row_table(lo, n_k + n_q)
    for b in range(B):
        first = lengths[b] - 1
        buckets = spread(table, lo, first, n_q)
        delta = first + torch.arange(n_q, device="cuda")[:, None] - j[None, :]
        ok = torch.ones_like(delta, dtype=torch.bool)
        if decode or case["causal"]:
            ok &= delta >= 0
        if case["window"]:
            ok &= ((delta < case["window"]) & (delta > -case["window"])) | (j < case["sinks"])[None, :]
        if not decode and s["mask"] is not None:
            ok &= s["mask"][b][None, :]
        some = ok.any(1, keepdim=True)
        for h in range(H):
            K, V = k[b, h // G], v[b, h // G]
            x = (q[b, h] @ K.T / math.sqrt(d) + w[h][buckets]).masked_fill_(~ok, -math.inf)
            p = torch.where(some, torch.softmax(torch.where(some, x, 0.0), 1), 0.0)
            o[b, h] = p @ V
            if not grad:
                continue
            d_v[b, h // G] += p.T @ d_o[b, h]
            d_p = d_o[b, h] @ V.T
            d_x = p * (d_p - (p * d_p).sum(1, keepdim=True))
            d_q[b, h] = d_x @ K / math.sqrt(d)
            d_k[b, h // G] += d_x.T @ q[b, h] / math.sqrt(d)
            d_w[h] += torch.bincount(buckets.reshape(-1), d_x.reshape(-1), case["buckets"])
    if not grad:
        return {"o": o[:, :, 0] if decode else o}
    return {"o": o, "d_q": d_q, "d_k": d_k, "d_v": d_v, "d_pos_weight": d_w}
