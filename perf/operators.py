"""The operators between the decoder's last state and the token it answers with: the product with 4-bit weights and group
scales that makes the logits, and the draw of a token from them (temperature, top-k, top-p, min-p, given random numbers).

`run` computes them in their plain form out of elementary torch operations, or, where `own` is true, through the
framework's entry points."""
import math

import numpy as np
import torch

own = False

#: the token and state types that the entry points take
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: sizes of a drawn case stay under these
MOST_LOGITS, MOST_ROWS, MOST_VOCAB = 1 << 25, 4096, 1 << 17
MOST_M, MOST_N, MOST_K = 256, 32768, 4096


def listed():
    lin = lambda name, m, n, k, g, t, zeros, bias: dict(  # noqa: E731
        name=name, op="linear", m=m, n=n, k=k, group=g, type=t, zeros=zeros, bias=bias)
    smp = lambda name, b, v, t, temp, top_k, top_p, min_p, mixed=False, masked=False: dict(  # noqa: E731
        name=name, op="sample", b=b, v=v, type=t, temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p, mixed=mixed, masked=masked)
    return [
        # one sentence's decode step: the yelp generator [9339, 256] on one row
        lin("head, one sentence", 1, 9339, 256, 32, "f32", False, True),
        # one token through a wide layer, group scales and zero points: the weights are all there is to read
        lin("wide layer, one token", 1, 16384, 4096, 128, "bf16", True, False),
        # ragged in every direction: rows, columns, and a last group that is cut short
        lin("ragged", 7, 1001, 777, 64, "f16", True, True),
        # the live rows late in a batch of the amazon corpus, [19724, 256]
        lin("head, 64 rows", 64, 19724, 256, 64, "f32", True, True),
        # feed_forward.w_2 of the autoencoder, [256, 1024], at the attack's batch
        lin("feed-forward", 256, 256, 1024, 128, "bf16", False, True),
        # the largest: a batch of tokens through a wide layer
        lin("wide layer, 256 tokens", 256, 32768, 4096, 128, "bf16", False, False),
        # one sentence, the usual serving settings on the yelp vocabulary
        smp("one sentence", 1, 9339, "f32", 0.8, 50, 0.95, 0.0),
        # one sequence over a large vocabulary, nothing but the nucleus
        smp("one row, large vocabulary", 1, 131072, "bf16", 1.0, 0, 0.9, 0.0),
        # a training batch of the corpus, min-p
        smp("a batch, min-p", 128, 9339, "f32", 1.2, 0, 1.0, 0.05),
        # requests of many users: settings of their own, banned words, one row banned altogether
        smp("mixed requests", 64, 50001, "f16", 1.0, 0, 1.0, 0.0, mixed=True, masked=True),
        # the attack's large batches, amazon vocabulary: plain draws
        smp("plain draws", 1024, 19724, "f32", 1.0, 0, 1.0, 0.0),
        # the largest: many rows of the yelp vocabulary, top-k and nucleus
        smp("many rows, top-k", 4096, 9339, "f32", 0.7, 40, 0.9, 0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    t = rng.choice(sorted(TYPES))
    if rng.random() < 0.5:
        return dict(op="linear", m=_log_int(rng, 1, MOST_M), n=_log_int(rng, 64, MOST_N), k=_log_int(rng, 64, MOST_K),
                    group=rng.choice((32, 64, 128)), type=t, zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
    v = _log_int(rng, 64, MOST_VOCAB)
    return dict(op="sample", b=_log_int(rng, 1, min(MOST_ROWS, MOST_LOGITS // v)), v=v, type=t,
                temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice((0, 0, 1, 20, 50, 400, v // 2)),
                top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.95)), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)),
                mixed=rng.random() < 0.25, masked=rng.random() < 0.25)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g, dev, t = _generator(seed), "cuda", TYPES[case["type"]]
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if case["op"] == "linear":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        groups = -(-k // group)
        s = dict(case)
        s["x"] = randn(m, k).to(t)
        # two codes a byte, the even column's in the low four bits
        s["codes"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
        s["scales"] = (0.3 / math.sqrt(k) * (0.5 + rand(n, groups))).to(torch.float16)
        s["zeros"] = torch.randint(5, 11, (n, groups), generator=g, device=dev, dtype=torch.uint8) if case["zeros"] else None
        s["bias_row"] = randn(n) if case["bias"] else None
        if own:  # the weights as a program keeps them
            from style_transfer_amd import ops
            s["packed"] = ops.pack_weight_q4(s["codes"], s["scales"], s["zeros"], k=k, group=group)
        return s
    b, v = case["b"], case["v"]
    s = dict(case)
    # a language model's logits: words of very unequal frequency, and rows between sure and undecided
    freq = -1.0 * torch.log1p(torch.arange(v, device=dev, dtype=torch.float32))[torch.randperm(v, generator=g, device=dev)]
    logits = freq + randn(b, v) * (1.0 + 2.0 * rand(b, 1))
    if case["masked"]:
        low = torch.where(rand(b, 1) < 0.5, -math.inf, torch.finfo(t).min)
        logits = torch.where(rand(b, v) < 0.3, low, logits)
        if b >= 4:
            logits[b // 2] = -math.inf
    s["logits"] = logits.to(t)
    s["u"] = rand(b)
    if case["mixed"]:  # settings of its own for every row, greedy ones among them
        pick = lambda values, dtype: torch.tensor(values, device=dev, dtype=dtype)[  # noqa: E731
            torch.randint(0, len(values), (b,), generator=g, device=dev)]
        s["temperature"] = pick((0.0, 0.5, 0.7, 1.0, 1.3), torch.float32)
        s["top_k"] = pick((0, 0, 1, 20, 50, 1000), torch.int32)
        s["top_p"] = pick((1.0, 0.5, 0.9, 0.99), torch.float32)
        s["min_p"] = pick((0.0, 0.0, 0.02, 0.2), torch.float32)
    return s


def _settings(s, dev):
    """the four settings as columns [B, 1] (or [1, 1]) in 64 bits, from the 32 bits that a caller gives"""
    col = lambda x, dt: torch.as_tensor(x, dtype=dt, device=dev).reshape(-1, 1)  # noqa: E731
    f = lambda x: col(x, torch.float32).double()  # noqa: E731
    return f(s["temperature"]), col(s["top_k"], torch.int64), f(s["top_p"]), f(s["min_p"])


def _sample(s):
    """plain form: sort every row, cumulative sums, masks.  64 bits: a draw next to a border has to fall on its side"""
    logits = s["logits"].double()
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    n, v = logits.shape
    temp, top_k, top_p, min_p = _settings(s, logits.device)
    vals, order = torch.sort(logits, dim=1, descending=True, stable=True)
    top = vals[:, :1]
    w = torch.where(vals == top, 1.0, torch.exp((vals - top) / temp))
    w = torch.where(vals == -math.inf, 0.0, w)
    c = torch.cumsum(w, 1)
    rank = torch.arange(v, device=logits.device)
    k = torch.where(top_k <= 0, v, top_k.clamp(max=v)).expand(n, 1)
    mass = torch.gather(c, 1, k - 1)
    keep = (rank < k) & ((top_p >= 1) | (c - w < top_p * mass)) & (w >= min_p) & (w > 0) & (temp > 0)
    keep |= rank == 0
    last = keep.sum(1, keepdim=True) - 1
    total = torch.gather(c, 1, last)
    at = (keep & (c <= s["u"].double()[:, None] * total)).sum(1, keepdim=True)
    at = torch.minimum(at, last)
    ids = torch.gather(order, 1, at)
    logp = torch.log(torch.gather(w, 1, at) / total)
    none = top == -math.inf
    ids = torch.where(none, -1, ids)[:, 0].to(torch.int32)
    return {"ids": ids, "logp": torch.where(none, -math.inf, logp)[:, 0].float()}


def _codes(s):
    """[N, K] the codes one by one"""
    c = s["codes"]
    return torch.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)[:, :s["k"]]


def _linear(s):
    """plain form: the weights in full, one product"""
    full = lambda a: a.float().repeat_interleave(s["group"], 1)[:, :s["k"]]  # noqa: E731
    zeros = full(s["zeros"]) if s["zeros"] is not None else 8.0
    w = (_codes(s).float() - zeros) * full(s["scales"])
    y = s["x"].float() @ w.t()
    if s["bias_row"] is not None:
        y = y + s["bias_row"]
    return y.to(s["x"].dtype)


def run(s):
    if own:
        from style_transfer_amd import ops
        if s["op"] == "linear":
            return ops.gemm_q4(s["x"], s["packed"], s["bias_row"])
        ids, logp = ops.sample_logits(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                      min_p=s["min_p"])
        return {"ids": ids, "logp": logp}
    return _linear(s) if s["op"] == "linear" else _sample(s)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * ((k + 1) // 2) + n * groups * (2 + (0.5 if case["zeros"] else 0)) + (4 * n if case["bias"] else 0)
                + (m * k + m * n) * size, "flops": 2 * m * n * k}
    b, v = case["b"], case["v"]
    # one subtraction, product, exponential and addition an entry
    return {"bytes": b * v * size + 4 * b + 8 * b + (16 * b if case["mixed"] else 0), "flops": 4 * b * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":  # group by group: (x . codes - zero * sum of x) * scale
        k, group = s["k"], s["group"]
        low = torch.bitwise_and(s["codes"], 15).double()
        high = torch.div(s["codes"], 16, rounding_mode="floor").double()
        codes = torch.empty(low.shape[0], 2 * low.shape[1], dtype=torch.float64, device=low.device)
        codes[:, 0::2], codes[:, 1::2] = low, high
        x = s["x"].double()
        y = torch.zeros(x.shape[0], codes.shape[0], dtype=torch.float64, device=x.device)
        for i, k0 in enumerate(range(0, k, group)):
            xs, k1 = x[:, k0:min(k, k0 + group)], min(k, k0 + group)
            zero = 8.0 if s["zeros"] is None else s["zeros"][:, i].double()
            y += (xs @ codes[:, k0:k1].t().contiguous() - xs.sum(1, keepdim=True) * zero) * s["scales"][:, i].double()
        return y if s["bias_row"] is None else y + s["bias_row"].double()
    # row by row on the host, walking down from the largest
    rows = s["logits"].float().cpu().numpy().astype(np.float64)
    u = s["u"].cpu().numpy().astype(np.float64)
    each = lambda x: np.broadcast_to(x.cpu().numpy() if torch.is_tensor(x) else np.float32(x), u.shape).astype(np.float64)  # noqa: E731
    temp, top_k, top_p, min_p = (each(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    ids, logp = np.full(len(u), -1, np.int32), np.full(len(u), -np.inf)
    for i, row in enumerate(rows):
        if not (row > -np.inf).any():
            continue
        order = np.argsort(-row, kind="stable")
        if temp[i] <= 0:
            ids[i], logp[i] = order[0], 0.0
            continue
        order = order[:int(np.count_nonzero(row > -np.inf))]
        if top_k[i] > 0:
            order = order[:int(top_k[i])]
        w = np.exp((row[order] - row[order[0]]) / temp[i])
        before = np.concatenate(([0.0], np.cumsum(w)))
        stop = len(w)
        if top_p[i] < 1:
            stop = int(np.searchsorted(before[:-1], top_p[i] * before[-1], side="left"))
        stop = max(1, min(stop, int(np.count_nonzero(w >= min_p[i]))))
        at = min(int(np.searchsorted(before[1:stop + 1], u[i] * before[stop], side="right")), stop - 1)
        ids[i], logp[i] = order[at], math.log(w[at] / before[stop])
    return {"ids": ids, "logp": logp}
