"""The operators a service needs that answers many questions about one long prompt and keeps its caches within a budget:

  prefix    attention of a batch whose sequences share one prefix: hawkeye_amd.ops.prefix_attention
  prompt    the attention weight every key collects from the queries of a prompt: hawkeye_amd.ops.attn_key_weights
  step      one decode step's attention that adds its weights to what the keys have collected: hawkeye_amd.ops.decode_attn_weights
  evict     the keys with the most weight, and the most recent ones, moved to the front of a cache: hawkeye_amd.ops.cache_evict

Queries carry softmax_scale * log2(e), as everywhere in hawkeye_amd.ops.  A key whose bias is -1e4 or less is removed (the
framework's own mask value is -1e4); a query that sees no key gives zeros and adds nothing.
"""
import math

import torch

own = False

LOG2E = 1.4426950408889634
REMOVED = -1.0e4


def listed():
    return [
        # a few questions about one clip whose prompt is the reference's usual length, one token each: latency
        {"name": "prefix step 4x352", "op": "prefix", "B": 4, "Nq": 1, "P": 352, "Nk": 20, "H": 32, "hd": 128, "pad": False},
        # the decode step's largest batch over a prompt near the model's 2048 positions, answers of different lengths left-padded
        {"name": "prefix step 16x1985", "op": "prefix", "B": 16, "Nq": 1, "P": 1985, "Nk": 61, "H": 32, "hd": 128, "pad": True},
        # a long shared document and many requests
        {"name": "prefix step 64x16384", "op": "prefix", "B": 64, "Nq": 1, "P": 16384, "Nk": 333, "H": 32, "hd": 128, "pad": False},
        # the questions themselves, short, ragged and left-padded, against the prompt
        {"name": "prefix questions 7x37", "op": "prefix", "B": 7, "Nq": 37, "P": 1201, "Nk": 37, "H": 32, "hd": 128, "pad": True},
        # long questions (dialogue history, multiple choice with explanations)
        {"name": "prefix questions 8x512", "op": "prefix", "B": 8, "Nq": 512, "P": 1400, "Nk": 512, "H": 32, "hd": 128, "pad": False},
        # a few tokens at once behind what a sequence has already, head size 64
        {"name": "prefix tokens 5x3", "op": "prefix", "B": 5, "Nq": 3, "P": 777, "Nk": 130, "H": 12, "hd": 64, "pad": False},
        # the weights of a usual prompt, one sequence: what a cache is cut by before the first token
        {"name": "prompt 1x352", "op": "prompt", "B": 1, "Nq": 352, "Nk": 352, "H": 32, "hd": 128, "pad": False},
        # two prompts near the model's 2048 positions, left-padded
        {"name": "prompt 2x2047", "op": "prompt", "B": 2, "Nq": 2047, "Nk": 2047, "H": 32, "hd": 128, "pad": True},
        # one sequence's step behind the usual prompt: latency
        {"name": "step 1x353", "op": "step", "B": 1, "Nk": 353, "H": 32, "hd": 128, "pad": False},
        # the largest batch, long caches, left-padded
        {"name": "step 16x1500", "op": "step", "B": 16, "Nk": 1500, "H": 32, "hd": 128, "pad": True},
        # one layer's caches cut as the answers grow
        {"name": "evict 4x353 to 256", "op": "evict", "B": 4, "Nk": 353, "budget": 256, "recent": 64, "H": 32, "hd": 128, "pad": False},
        # eight layers of two left-padded prompts cut to half on their way into the decode caches
        {"name": "evict 16x2047 to 1024", "op": "evict", "B": 16, "Nk": 2047, "budget": 1024, "recent": 256, "H": 32, "hd": 128, "pad": True},
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _some(rng):
    op = rng.choice(["prefix", "prefix", "prefix", "prompt", "step", "evict"])
    case = {"op": op, "H": rng.choice([2, 8, 12, 16, 32, 32]), "hd": rng.choice([64, 128, 128]), "pad": rng.random() < 0.5}
    if op == "prefix":
        form = rng.choice(["step", "tokens", "questions"])
        nq = {"step": 1, "tokens": rng.randint(2, 16), "questions": _log(rng, 8, 512)}[form]
        case.update(B=_log(rng, 1, 8 if form == "questions" else 64), Nq=nq, P=_log(rng, 1, 2048 if form == "questions" else 16384),
                    Nk=nq + (0 if form == "questions" else _log(rng, 1, 512) - 1))
    elif op == "prompt":
        n = _log(rng, 1, 2047)
        case.update(B=rng.randint(1, 2), Nq=rng.choice([n, n, max(1, n // 8)]), Nk=n)
    elif op == "step":
        case.update(B=_log(rng, 1, 16), Nk=_log(rng, 1, 4096))
    else:
        n = _log(rng, 2, 4096)
        budget = rng.randint(1, n)
        case.update(B=_log(rng, 1, 16), Nk=n, budget=budget, recent=rng.randint(0, budget))
    return case


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in w:
            most[c["op"], k] = max(most.get((c["op"], k), 0), w[k])
    while True:
        case = _some(rng)
        w = work(case)
        if all(w[k] <= most[case["op"], k] for k in w):
            return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, hd, n = case["B"], case["H"], case["hd"], case["Nk"]
    bf16 = torch.bfloat16

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=bf16) * scale).to(bf16)

    st = {"op": case["op"], "n": n, "bias": None}
    qs = 1.5 * hd ** -0.5 * LOG2E           # what the producer of q folds in, and queries that favour some keys
    if case["pad"]:                         # left-padded rows of different lengths; the first row is whole
        valid = torch.randint(1, n + 1, (B,), generator=g, device="cuda")
        valid[0] = n
        pad = torch.arange(n, device="cuda")[None, :] < (n - valid)[:, None]
        st["bias"] = pad.to(torch.float32) * REMOVED
    if case["op"] == "prefix":
        st["q"] = rnd(B, case["Nq"], H, hd, scale=qs)
        st["k_prefix"], st["v_prefix"] = rnd(case["P"], H, hd), rnd(case["P"], H, hd)
        rows = -(-(n + 1) // 64) * 64       # the sequences' caches have rows to spare
        st["k"], st["v"] = rnd(B, rows, H, hd)[:, :n], rnd(B, rows, H, hd)[:, :n]
    elif case["op"] == "prompt":
        qkv = rnd(B, n, 3, H, hd)           # q | k | v side by side, as the projection leaves them
        qkv[:, :, 0] *= qs
        st["q"], st["k"] = qkv[:, n - case["Nq"]:, 0], qkv[:, :, 1]
    elif case["op"] == "step":
        rows = -(-(n + 1) // 64) * 64
        st["q"] = rnd(B, H * hd, scale=qs)
        st["k"], st["v"] = rnd(B, rows, H * hd), rnd(B, rows, H * hd)
        st["weight"] = torch.rand((B, H, rows), generator=g, device="cuda") ** 4 * 8
        st["weight_out"] = torch.empty_like(st["weight"])
    else:
        budget = case["budget"]
        st["budget"], st["recent"] = budget, case["recent"]
        qkv = rnd(B, n, 3, H, hd)
        st["k"], st["v"] = qkv[:, :, 1], qkv[:, :, 2]
        w = torch.rand((B, H, n), generator=g, device="cuda")
        st["weight"] = torch.where(w < 0.2, 0.0, w ** 4 * 8)        # some keys were never looked at: ties
        if st["bias"] is not None:
            st["bias"] = st["bias"][:, None, :].repeat(1, H, 1)     # every head has its own rows once it has chosen
        rows = -(-(budget + 1) // 64) * 64
        st["out"] = (torch.empty((B, rows, H, hd), dtype=bf16, device="cuda"), torch.empty((B, rows, H, hd), dtype=bf16, device="cuda"),
                     torch.empty((B, H, rows), device="cuda"), None if st["bias"] is None else torch.empty((B, H, rows), device="cuda"))
    return st


def _visible(scores, nq, nk, bias):
    """scores [B, H, nq, nk] in powers of two with the bias added, removed keys and keys behind the query at -inf."""
    if bias is not None:
        b = bias[:, None, None, :]
        scores = (scores + b * LOG2E).masked_fill(b <= REMOVED, -math.inf)
    ahead = torch.ones((nq, nk), dtype=torch.bool, device=scores.device).triu(nk - nq + 1)
    return scores.masked_fill(ahead, -math.inf)


def _softmax2(scores):
    top = scores.amax(-1, keepdim=True)
    e = torch.exp2(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prefix(q, kp, vp, k, v, bias):
    B, nq, H, hd = q.shape
    P, nk = kp.shape[0], k.shape[1]
    q = q.float().permute(0, 2, 1, 3).contiguous()                                  # [B, H, nq, hd]
    rows = q.transpose(0, 1).reshape(H, B * nq, hd)
    shared = (rows @ kp.float().permute(1, 2, 0).contiguous()).view(H, B, nq, P).transpose(0, 1)
    mine = _visible(q @ k.float().permute(0, 2, 3, 1).contiguous(), nq, nk, bias)
    p = _softmax2(torch.cat([shared, mine], -1))
    out = p[..., P:] @ v.float().permute(0, 2, 1, 3).contiguous()
    ps = p[..., :P].transpose(0, 1).reshape(H, B * nq, P)
    out = out + (ps @ vp.float().transpose(0, 1).contiguous()).view(H, B, nq, hd).transpose(0, 1)
    return out.transpose(1, 2).to(torch.bfloat16)


def _plain_weights(q, k, bias):
    nq, nk = q.shape[1], k.shape[1]
    scores = q.float().transpose(1, 2).contiguous() @ k.float().permute(0, 2, 3, 1).contiguous()
    return _softmax2(_visible(scores, nq, nk, bias))


def _plain_evict(st):
    n, budget, recent = st["n"], st["budget"], st["recent"]
    w, bias = st["weight"], st["bias"]
    rank = w if bias is None else w.masked_fill(bias <= REMOVED, -math.inf)
    order = torch.sort(rank[..., :n - recent], dim=-1, descending=True, stable=True).indices[..., :budget - recent]
    last = torch.arange(n - recent, n, device=w.device).expand(*w.shape[:2], recent)
    kept = torch.cat([torch.sort(order, dim=-1).values, last], -1)                  # [B, H, budget], ascending
    rows = kept.transpose(1, 2)[..., None].expand(-1, -1, -1, st["k"].shape[3])
    res = [st["k"].gather(1, rows), st["v"].gather(1, rows), w.gather(2, kept)]
    if bias is not None:
        res.append(bias.gather(2, kept))
    return [kept.to(torch.int32)] + res


def run(state):
    st = state
    n = st["n"]
    if own:
        from hawkeye_amd import ops
        if st["op"] == "prefix":
            return ops.prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"], key_bias=st["bias"])
        if st["op"] == "prompt":
            return ops.attn_key_weights(st["q"], st["k"], key_bias=st["bias"], causal=True)
        if st["op"] == "step":
            H = st["weight"].shape[1]
            out = ops.decode_attn_weights(st["q"], st["k"], st["v"], n, H, st["q"].shape[1] // H, st["weight"],
                                          key_bias=st["bias"], weight_out=st["weight_out"])
            return [out, st["weight_out"][..., :n]]
        kept = ops.cache_evict(st["k"], st["v"], st["weight"], n, st["budget"], st["recent"], key_bias=st["bias"], out=st["out"])
        b = st["budget"]
        res = [kept, st["out"][0][:, :b], st["out"][1][:, :b], st["out"][2][..., :b]]
        return res if st["bias"] is None else res + [st["out"][3][..., :b]]
    if st["op"] == "prefix":
        return _plain_prefix(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"], st["bias"])
    if st["op"] == "prompt":
        return _plain_weights(st["q"], st["k"], st["bias"]).sum(2)
    if st["op"] == "step":
        B, H = st["weight"].shape[:2]
        hd = st["q"].shape[1] // H
        k, v = (t[:, :n].view(B, n, H, hd) for t in (st["k"], st["v"]))
        p = _plain_weights(st["q"].view(B, 1, H, hd), k, st["bias"])                # [B, H, 1, n]
        out = (p @ v.float().transpose(1, 2).contiguous()).reshape(B, H * hd).to(torch.bfloat16)
        return [out, st["weight"][..., :n] + p[:, :, 0]]
    return _plain_evict(st)


def work(case):
    B, H, hd, n = case["B"], case["H"], case["hd"], case["Nk"]
    row = H * hd * 2
    bias = B * n * 4 if case["pad"] else 0
    if case["op"] == "prefix":
        nq, P = case["Nq"], case["P"]
        pairs = B * (nq * P + nq * n - nq * (nq - 1) // 2)
        return {"bytes": 2 * B * nq * row + 2 * P * row + 2 * B * n * row + bias, "flops": 4 * pairs * H * hd}
    if case["op"] == "prompt":
        nq = case["Nq"]
        return {"bytes": B * (nq + n) * row + B * H * n * 4 + bias, "flops": 2 * B * (nq * n - nq * (nq - 1) // 2) * H * hd}
    if case["op"] == "step":
        return {"bytes": 2 * B * row + 2 * B * n * row + 2 * B * H * n * 4 + bias, "flops": 4 * B * n * H * hd}
    budget = case["budget"]
    return {"bytes": 4 * B * budget * row + B * H * (n + 2 * budget) * 4 + (B * H * (n + budget) * 4 if case["pad"] else 0),
            "flops": B * H * n}


def exact(case, seed):
    """The definitions in 64 bits, one head at a time."""
    st = prepare(case, seed)
    H, n = case["H"], case["Nk"]
    gone = None if st["bias"] is None else st["bias"] <= REMOVED
    if case["op"] == "evict":
        w = st["weight"].double()
        key = w.clone()
        if gone is not None:
            key[gone] = -1.0                # weights are sums of probabilities: nothing else is below zero
        key[..., n - case["recent"]:] = math.inf
        place = torch.argsort(-key, dim=-1, stable=True)[..., :case["budget"]]
        keep = torch.zeros_like(key, dtype=torch.bool).scatter_(2, place, True)
        kept = keep.nonzero()[:, 2].view(case["B"], H, case["budget"])
        b = torch.arange(case["B"], device="cuda")[:, None]
        rows = [torch.stack([t[:, :, h][b, kept[:, h]].double() for h in range(H)], 2) for t in (st["k"], st["v"])]
        res = [kept.to(torch.int32)] + rows + [w[keep].view(kept.shape)]
        return res if gone is None else res + [st["bias"].double()[keep].view(kept.shape)]
    ln2 = math.log(2.0)
    B, hd = case["B"], case["hd"]
    nq = case.get("Nq", 1)
    q = st["q"].view(B, nq, H, hd) if case["op"] == "step" else st["q"]
    k = st["k"][:, :n].reshape(B, n, H, hd)
    pos = torch.arange(nq, device="cuda") + (n - nq)
    hidden = (torch.arange(n, device="cuda")[None, :] > pos[:, None])[None]          # [1, nq, n]
    outs, weights = [], []
    for h in range(H):
        qh = q[:, :, h].double() * ln2
        s = torch.bmm(qh, k[:, :, h].double().transpose(1, 2).contiguous())
        if gone is not None:
            s = s + st["bias"].double()[:, None, :]
            s[gone[:, None, :].expand_as(s)] = -math.inf
        s[hidden.expand_as(s)] = -math.inf
        if case["op"] == "prefix":
            kp, vp = st["k_prefix"][:, h].double(), st["v_prefix"][:, h].double()
            s = torch.cat([torch.matmul(qh, kp.t().contiguous()), s], 2)
        z = torch.logsumexp(s, 2, keepdim=True)
        p = torch.exp(s - z).nan_to_num(0.0)                                        # a row without keys: -inf - -inf
        if case["op"] == "prompt":
            weights.append(p.sum(1))
            continue
        if case["op"] == "step":
            weights.append(p[:, 0])
            outs.append(torch.bmm(p, st["v"][:, :n].view(B, n, H, hd)[:, :, h].double().contiguous()))
        else:
            P = case["P"]
            outs.append(torch.matmul(p[..., :P], vp) + torch.bmm(p[..., P:], st["v"][:, :, h].double().contiguous()))
    if case["op"] == "prompt":
        return torch.stack(weights, 1)
    out = torch.stack(outs, 2)
    if case["op"] == "prefix":
        return out
    return [out.reshape(B, H * hd), st["weight"][..., :n].double() + torch.stack(weights, 1)]
