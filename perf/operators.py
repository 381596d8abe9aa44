"""The operators of a KV cache that many sequences share, or that is held to a budget: what is measured.

Four operators of the device API, each with its plain form in elementary torch operations:

* ``shared``   one decode step of a batch whose sequences share long prefixes (a system prompt, a
  document, few-shot examples): every shared row of the cache is read once for all of them;
* ``weights``  one decode step that also adds each cached key's attention probability, summed over
  the query heads of its KV head, to that key's running weight;
* ``prompt``   the same running weights for the rows of a prompt (all of them, or the last few);
* ``evict``    brings every KV head's cache to its budget: the first tokens, the most recent ones
  and the heaviest of the rest stay, moved into the slots of those that go.

Shapes are those of the decoders this library serves (16 query / 8 KV heads of 128, 8 / 1 of 256,
12 / 12 of 64) or generic.
"""
import math
import os
import sys

import torch

own = False   # True: run() calls the library's entry points instead of the plain form

DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # two chats on one short system prompt, first token: nothing but latency
        dict(name="shared latency", op="shared", seqs=2, prefixes=1, prefix=512, lo=1, hi=5, hq=16, hkv=8, hd=128,
             bf16=False, window=0, cap=0.0),
        # a serving batch on one long prompt, bf16 activations
        dict(name="shared batch", op="shared", seqs=64, prefixes=1, prefix=8192, lo=100, hi=1024, hq=16, hkv=8, hd=128,
             bf16=True, window=0, cap=0.0),
        # four tenants, odd lengths, fp32 activations
        dict(name="shared tenants", op="shared", seqs=200, prefixes=4, prefix=12345, lo=1, hi=2047, hq=16, hkv=8,
             hd=128, bf16=False, window=0, cap=0.0),
        # one KV head of 256, capped scores, a window that ends inside the prefix
        dict(name="shared mqa 256", op="shared", seqs=31, prefixes=1, prefix=4099, lo=3, hi=700, hq=8, hkv=1, hd=256,
             bf16=True, window=4096, cap=50.0),
        # one chat, a short cache
        dict(name="weights latency", op="weights", seqs=1, lo=513, hi=513, hq=16, hkv=8, hd=128, bf16=False, window=0,
             cap=0.0),
        # a serving batch, lengths as drawn for batched decode
        dict(name="weights batch", op="weights", seqs=64, lo=1024, hi=8192, hq=16, hkv=8, hd=128, bf16=True, window=0,
             cap=0.0),
        # heads of 64 without grouping, odd lengths, one of them empty
        dict(name="weights mha 64", op="weights", seqs=9, lo=0, hi=2500, hq=12, hkv=12, hd=64, bf16=False, window=0,
             cap=0.0),
        # the last 32 rows of a long prompt choose what stays
        dict(name="prompt last rows", op="prompt", batch=1, rows=32, keys=16384, hq=16, hkv=8, hd=128, mask=0,
             prefix=0, window=0, cap=0.0),
        # every row of a prompt
        dict(name="prompt causal", op="prompt", batch=1, rows=4096, keys=4096, hq=16, hkv=8, hd=128, mask=0, prefix=0,
             window=0, cap=0.0),
        # image and text prefix seen whole, then text, one KV head of 256
        dict(name="prompt prefix-lm 256", op="prompt", batch=8, rows=451, keys=451, hq=8, hkv=1, hd=256, mask=1,
             prefix=320, window=0, cap=0.0),
        # steady state: each step appends one token and drops one
        dict(name="evict one", op="evict", seqs=32, keys=1025, budget=1024, hkv=8, hd=128, sink=4, recent=256),
        # after long prompts: an eighth stays
        dict(name="evict prompts", op="evict", seqs=8, keys=16384, budget=2048, hkv=8, hd=128, sink=4, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "weights", "prompt", "evict"])
    hq, hkv, hd = rng.choice([(16, 8, 128), (16, 8, 128), (8, 1, 256), (12, 12, 64), (24, 4, 128), (15, 5, 64)])
    cap = rng.choice([0.0, 0.0, 0.0, 50.0])
    if op == "shared":
        seqs = _log(rng, 1, 160)
        prefixes = rng.randint(1, min(4, seqs))
        prefix = _log(rng, 1, 12000 // prefixes)
        hi = _log(rng, 1, 1500)
        window = rng.choice([0, 0, 0, _log(rng, 1, prefix + hi)])
        return dict(op=op, seqs=seqs, prefixes=prefixes, prefix=prefix, lo=rng.choice([0, 1, hi]), hi=hi, hq=hq,
                    hkv=hkv, hd=hd, bf16=rng.random() < 0.5, window=window, cap=cap)
    if op == "weights":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 6000)
        return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi]), hi=hi, hq=hq, hkv=hkv, hd=hd,
                    bf16=rng.random() < 0.5, window=rng.choice([0, 0, _log(rng, 1, hi)]), cap=cap)
    if op == "prompt":
        keys = _log(rng, 1, 3500)
        rows = rng.choice([keys, _log(rng, 1, keys), min(keys, 32)])
        batch = rng.randint(1, max(1, min(6, 3500 // keys)))
        mask = rng.choice([0, 0, 1, 3])
        hq, hkv, hd = rng.choice([(hq, hkv, hd), (4, 2, 72)])
        return dict(op=op, batch=batch, rows=rows, keys=keys, hq=hq, hkv=hkv, hd=hd, mask=mask,
                    prefix=_log(rng, 1, keys) if mask == 1 else 0,
                    window=rng.choice([0, 0, _log(rng, 1, keys)]), cap=cap)
    seqs = _log(rng, 1, 32)
    keys = _log(rng, 2, 120000 // seqs)
    budget = rng.choice([keys - 1, _log(rng, 1, keys), max(1, keys // 8)])
    sink = rng.randint(0, min(4, budget))
    recent = rng.randint(0, budget - sink)
    return dict(op=op, seqs=seqs, keys=keys, budget=budget, hkv=hkv, hd=hd, sink=sink, recent=recent)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(g, n, lo, hi):
    """Lengths spread over [lo, hi], both ends among them, in an order of the seed."""
    x = torch.linspace(lo, hi, n, dtype=torch.float64).round().to(torch.int64)
    return x[torch.randperm(n, generator=g)]


def _group_sizes(n, groups):
    """Uneven sizes of the sequences of each prefix: 1 : 2 : 3 ..., none empty."""
    w = [i + 1 for i in range(groups)]
    cut = [0] + [max(i + 1, n * sum(w[:i + 1]) // sum(w)) for i in range(groups)]
    cut[-1] = n
    for i in range(groups - 1, 0, -1):
        cut[i] = min(cut[i], cut[i + 1] - 1)
    return cut


def _pool(g, rows, hkv, hd):
    k = torch.randn((rows, hkv * hd), device=DEV, generator=g).to(torch.bfloat16)
    v = torch.randn((rows, hkv * hd), device=DEV, generator=g).to(torch.float16)
    return k, v


_module = None


def _library():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "smol-genius_b200"))
        import smol_b200
        _module = smol_b200
    return _module


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    hkv, hd = c["hkv"], c["hd"]
    if c["op"] in ("shared", "weights"):
        n, hq = c["seqs"], c["hq"]
        lens = _lengths(g, n, c["lo"], c["hi"])
        groups = c.get("prefixes", 0)
        cut = _group_sizes(n, groups) if groups else [0]
        # the lengths of the prefixes: the longest, and shorter ones down to half of it
        plen = torch.tensor([c["prefix"] - (c["prefix"] // 2) * i // groups for i in range(groups)], dtype=torch.int64)
        stride = max(1, c["hi"]) + 3
        starts = torch.cumsum(torch.cat([plen, lens + 2]), 0)
        rows = int(starts[-1]) + 1
        first = torch.cat([torch.zeros(1, dtype=torch.int64), starts[:-1]])
        s["k"], s["v"] = _pool(gd, rows, hkv, hd)
        q = torch.randn((n, hq * hd), device=DEV, generator=gd)
        s["q"] = q.to(torch.bfloat16) if c["bf16"] else q
        s["out"] = torch.empty_like(s["q"])
        s["win"] = torch.rand((n, hkv, stride), device=DEV, generator=gd) ** 8
        s["wout"] = torch.zeros_like(s["win"])
        s["row0"] = first[groups:].to(DEV)
        s["len"] = lens.to(torch.int32).to(DEV)
        s["max_len"] = int(lens.max())
        s["rows"], s["stride"], s["scale"] = rows, stride, 1.0 / math.sqrt(hd)
        if groups:
            s["prow0"] = first[:groups].to(DEV)
            s["plen"] = plen.to(torch.int32).to(DEV)
            s["cut"] = torch.tensor(cut, dtype=torch.int32, device=DEV)
            s["max_plen"] = int(plen.max())
            s["max_group"] = max(b - a for a, b in zip(cut, cut[1:]))
    elif c["op"] == "prompt":
        b, hq = c["batch"], c["hq"]
        s["q"] = torch.randn((b, c["rows"], hq * hd), device=DEV, generator=gd).to(torch.bfloat16)
        s["k"] = torch.randn((b, c["keys"], hkv * hd), device=DEV, generator=gd).to(torch.bfloat16)
        s["stride"] = c["keys"] + 1
        s["win"] = torch.rand((b, hkv, s["stride"]), device=DEV, generator=gd) ** 8
        s["wout"] = torch.zeros_like(s["win"])
        s["scale"] = 1.0 / math.sqrt(hd)
    else:
        n, keys = c["seqs"], c["keys"]
        # every length above the budget but one, which needs nothing
        lens = _lengths(g, n, max(c["budget"] + 1, keys - keys // 16), keys)
        if n > 2:
            lens[n // 2] = max(0, c["budget"] - 3)
        stride = keys + 1
        s["k"], s["v"] = _pool(gd, n * stride, hkv, hd)
        s["row0"] = torch.arange(n, device=DEV, dtype=torch.int64) * stride
        s["len"] = lens.to(torch.int32).to(DEV)
        s["len_out"] = torch.zeros_like(s["len"])
        # accumulated probabilities: a few heavy keys, a long tail, some never attended
        w = torch.exp(2.0 * torch.randn((n, hkv, stride), device=DEV, generator=gd))
        s["win"] = torch.where(torch.rand(w.shape, device=DEV, generator=gd) < 0.02, torch.zeros_like(w), w)
        # an earlier eviction left the kept positions in any order; later tokens have none yet
        seen = 2 * lens
        perm = torch.argsort(torch.rand((n, hkv, stride), device=DEV, generator=gd), dim=2)
        idx = torch.arange(stride, device=DEV)
        s["pin"] = torch.where(idx < s["len"].view(n, 1, 1) // 2, perm, -1).to(torch.int32)
        s["wout"], s["pout"] = torch.zeros_like(s["win"]), torch.zeros_like(s["pin"])
        s["seen"] = seen.to(torch.int32).to(DEV)
        s["max_len"], s["rows"], s["stride"] = int(lens.max()), n * stride, stride
    if own:
        lib = _library()
        if c["op"] == "shared":
            size = lib.decode_shared_workspace_bytes(c["seqs"], s["max_len"], c["prefixes"], s["max_plen"],
                                                     s["max_group"], c["hq"], hkv, hd)
        elif c["op"] == "weights":
            size = lib.decode_weights_workspace_bytes(c["seqs"], s["max_len"], c["hq"], hkv, hd)
        elif c["op"] == "prompt":
            size = lib.prefill_weights_workspace_bytes(c["batch"], c["rows"], c["keys"], c["hq"], hkv, hd)
        else:
            size = lib.cache_evict_workspace_bytes(c["seqs"], s["max_len"], hkv)
        s["ws"] = torch.empty(max(1, size), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    return {"shared": _run_shared, "weights": _run_weights, "prompt": _run_prompt, "evict": _run_evict}[c["op"]](s, c)


def _capped(x, cap):
    return cap * torch.tanh(x / cap) if cap > 0 else x


def _probs(x):
    """softmax over the last axis; a row with nothing to see is all zeros."""
    m = x.amax(dim=-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(x - m)
    t = e.sum(dim=-1, keepdim=True)
    return e / torch.where(t > 0, t, torch.ones_like(t))


def _suffix_scores(s, c):
    """Scores [n, hkv, group, L] of every sequence's own keys (-inf where it has none) and its values."""
    n, hkv, hd, L = c["seqs"], c["hkv"], c["hd"], max(1, s["max_len"])
    j = torch.arange(L, device=DEV)
    rows = (s["row0"].view(n, 1) + j).clamp_max(s["rows"] - 1)
    k = s["k"][rows].float().view(n, L, hkv, hd)
    v = s["v"][rows].float().view(n, L, hkv, hd)
    q = s["q"].float().view(n, hkv, -1, hd)
    x = _capped(torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"], c["cap"])
    length = s["len"].view(n, 1).long()
    seen = j < length
    if c["window"] > 0:
        seen &= j >= length - c["window"]
    return torch.where(seen.view(n, 1, 1, L), x, torch.full_like(x, -math.inf)), v, q


def _add_weights(s, probs):
    L = probs.shape[-1]
    inside = torch.arange(L, device=DEV) < s["len"].view(-1, 1, 1)
    w = s["win"][..., :L] + probs.sum(dim=2)
    s["wout"][..., :L] = torch.where(inside, w, s["wout"][..., :L])
    return s["wout"]


def _run_weights(s, c):
    if own:
        _library().decode_attention_weights(
            s["out"], s["q"], s["k"], s["v"], s["rows"], s["row0"], s["len"], c["seqs"], s["max_len"], c["hq"],
            c["hkv"], c["hd"], s["scale"], s["win"], s["wout"], s["stride"], s["ws"], window=c["window"],
            softcap=c["cap"])
        return s["out"], s["wout"]
    x, v, _ = _suffix_scores(s, c)
    p = _probs(x)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(c["seqs"], -1)
    return out.to(s["q"].dtype), _add_weights(s, p)


def _run_shared(s, c):
    if own:
        _library().decode_attention_shared(
            s["out"], s["q"], s["k"], s["v"], s["rows"], s["prow0"], s["plen"], s["cut"], c["prefixes"],
            s["max_plen"], s["max_group"], s["row0"], s["len"], c["seqs"], s["max_len"], c["hq"], c["hkv"], c["hd"],
            s["scale"], s["ws"], window=c["window"], softcap=c["cap"], weights_in=s["win"], weights_out=s["wout"],
            weights_stride=s["stride"])
        return s["out"], s["wout"]
    n, hkv, hd, groups, P, M = c["seqs"], c["hkv"], c["hd"], c["prefixes"], s["max_plen"], s["max_group"]
    x, v, q = _suffix_scores(s, c)
    grp = q.shape[2]
    # the prefixes' keys once, the sequences of a prefix side by side (padded to the largest group)
    j = torch.arange(P, device=DEV)
    rows = (s["prow0"].view(groups, 1) + j).clamp_max(s["rows"] - 1)
    kp = s["k"][rows].float().view(groups, P, hkv, hd)
    vp = s["v"][rows].float().view(groups, P, hkv, hd)
    cut = s["cut"].long()
    slot = (cut[:-1].view(groups, 1) + torch.arange(M, device=DEV)).clamp_max(n - 1)          # [groups, M]
    mine = torch.bucketize(torch.arange(n, device=DEV), cut[1:], right=True)                  # prefix of a sequence
    at = mine * M + torch.arange(n, device=DEV) - cut[mine]                                   # its padded place
    qp = q[slot].permute(0, 2, 1, 3, 4).reshape(groups, hkv, M * grp, hd)
    y = _capped(torch.matmul(qp, kp.permute(0, 2, 3, 1)) * s["scale"], c["cap"])
    y = y.view(groups, hkv, M, grp, P).permute(0, 2, 1, 3, 4).reshape(groups * M, hkv, grp, P)[at]
    plen = s["plen"].long()[mine].view(n, 1)
    seen = j < plen
    if c["window"] > 0:
        seen &= j >= plen + s["len"].view(n, 1).long() - c["window"]
    y = torch.where(seen.view(n, 1, 1, P), y, torch.full_like(y, -math.inf))
    p = _probs(torch.cat([y, x], dim=-1))
    pp, ps = p[..., :P], p[..., P:]
    pad = pp.new_zeros((groups * M, hkv, grp, P))
    pad[at] = pp
    pad = pad.view(groups, M, hkv, grp, P).permute(0, 2, 1, 3, 4).reshape(groups, hkv, M * grp, P)
    op = torch.matmul(pad, vp.permute(0, 2, 1, 3)).view(groups, hkv, M, grp, hd)
    op = op.permute(0, 2, 1, 3, 4).reshape(groups * M, hkv, grp, hd)[at]
    out = op + torch.matmul(ps, v.permute(0, 2, 1, 3))
    return out.reshape(n, -1).to(s["q"].dtype), _add_weights(s, ps)


def _run_prompt(s, c):
    b, R, K, hq, hkv, hd = c["batch"], c["rows"], c["keys"], c["hq"], c["hkv"], c["hd"]
    if own:
        _library().prefill_attention_weights(
            s["win"], s["wout"], s["stride"], s["q"], s["k"], b, R, K, hq, hkv, hd, s["scale"], s["ws"],
            mask_kind=c["mask"], q_offset=K - R, prefix_len=c["prefix"], window=c["window"], softcap=c["cap"])
        return s["wout"]
    q = s["q"].float().view(b, R, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4)
    k = s["k"].float().view(b, K, hkv, 1, hd).permute(0, 2, 3, 4, 1)
    x = _capped(torch.matmul(q, k) * s["scale"], c["cap"])
    pos = torch.arange(K - R, K, device=DEV).view(R, 1)
    j = torch.arange(K, device=DEV)
    seen = {0: j <= pos, 1: (j <= pos) | (j < c["prefix"]), 3: (j < K) & (pos >= 0)}[c["mask"]]
    if c["window"] > 0:
        seen = seen & (j > pos - c["window"])
    p = _probs(torch.where(seen, x, torch.full_like(x, -math.inf)))
    s["wout"][..., :K] = s["win"][..., :K] + p.sum(dim=(2, 3))
    return s["wout"]


def _run_evict(s, c):
    n, hkv, hd, budget = c["seqs"], c["hkv"], c["hd"], c["budget"]
    if own:
        _library().cache_evict(
            s["k"], s["v"], s["rows"], s["row0"], s["win"], s["wout"], s["pin"], s["pout"], s["stride"], s["len"],
            s["len_out"], s["seen"], n, s["max_len"], hkv, hd, budget, c["sink"], c["recent"], s["ws"])
        return s["k"], s["v"], s["wout"], s["pout"], s["len_out"]
    L = s["max_len"]
    j = torch.arange(L, device=DEV).expand(n, hkv, L)
    length, seen = s["len"].view(n, 1, 1).long(), s["seen"].view(n, 1, 1).long()
    new = length.clamp_max(budget)
    w, pos = s["win"][..., :L], s["pin"][..., :L].long()
    pos = torch.where(pos < 0, seen - length + j, pos)       # not yet placed: appended in order, up to the newest
    key = torch.where((pos < c["sink"]) | (pos >= seen - c["recent"]), torch.full_like(w, math.inf), w)
    key = torch.where(j < length, key, torch.full_like(key, -math.inf))
    rank = torch.empty_like(j)
    rank.scatter_(2, torch.sort(key, dim=2, descending=True, stable=True).indices, j.contiguous())
    kept = rank < new
    hole, mover = ~kept & (j < new), kept & (j >= new)
    movers = torch.sort((~mover).to(torch.int8), dim=2, stable=True).indices
    src = torch.where(hole, movers.gather(2, (torch.cumsum(hole, 2) - 1).clamp_min(0)), j)
    inside, changes = j < length, length > new
    placed = torch.where(changes, pos.gather(2, src), s["pin"][..., :L].long()).to(torch.int32)
    s["wout"][..., :L] = torch.where(j < new, w.gather(2, src), torch.where(inside, torch.zeros_like(w),
                                                                            s["wout"][..., :L]))
    s["pout"][..., :L] = torch.where(j < new, placed, torch.where(inside, torch.full_like(placed, -1),
                                                                  s["pout"][..., :L]))
    s["len_out"].copy_(new.view(n))
    top = min(L, budget)
    to = s["row0"].view(n, 1, 1) + j[..., :top]
    frm = s["row0"].view(n, 1, 1) + src[..., :top]
    head = torch.arange(hkv, device=DEV).view(1, hkv, 1)
    for pool in (s["k"], s["v"]):
        rows = pool.view(-1, hkv, hd)
        rows[to, head] = rows[frm, head]
    return s["k"], s["v"], s["wout"], s["pout"], s["len_out"]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(rows, keys, mask, prefix, window):
    """Visible (row, key) pairs of the last `rows` positions of `keys`."""
    pos = torch.arange(keys - rows, keys, dtype=torch.int64)
    hi = {0: pos + 1, 1: (pos + 1).clamp_min(prefix), 3: torch.full_like(pos, keys)}[mask]
    lo = (pos - window + 1).clamp_min(0) if window > 0 else torch.zeros_like(pos)
    return int((hi - lo).clamp_min(0).sum())


def work(case):
    c = case
    hkv, hd = c["hkv"], c["hd"]
    if c["op"] in ("shared", "weights"):
        n, hq = c["seqs"], c["hq"]
        own_keys = torch.linspace(c["lo"], c["hi"], n, dtype=torch.float64).round()
        seen = own_keys.clamp_max(c["window"]) if c["window"] > 0 else own_keys
        size = 2 if c["bf16"] else 4
        nbytes = float(seen.sum()) * hkv * hd * 4 + float(own_keys.sum()) * hkv * 8 + 2 * n * hq * hd * size
        flops = float(seen.sum()) * 4 * hq * hd
        groups = c.get("prefixes", 0)
        cut = _group_sizes(n, groups) if groups else []
        for i in range(groups):
            plen = c["prefix"] - (c["prefix"] // 2) * i // groups
            members = cut[i + 1] - cut[i]
            mean = float(own_keys.mean())
            visible = min(plen, max(0.0, c["window"] - mean)) if c["window"] > 0 else plen
            most = min(plen, max(0, c["window"] - c["lo"])) if c["window"] > 0 else plen
            nbytes += most * hkv * hd * 4
            flops += visible * members * 4 * hq * hd
        return dict(bytes=nbytes, flops=flops)
    if c["op"] == "prompt":
        pairs = _pairs(c["rows"], c["keys"], c["mask"], c["prefix"], c["window"])
        return dict(bytes=c["batch"] * (c["rows"] * c["hq"] * hd * 2 + c["keys"] * hkv * (hd * 2 + 8)),
                    flops=2.0 * hd * c["hq"] * c["batch"] * pairs)
    # weights and positions in and out; rows that move (kept ones are spread over the slots) read and written
    n, keys, budget = c["seqs"], c["keys"], c["budget"]
    moved = budget * (1.0 - budget / keys)
    return dict(bytes=n * hkv * (keys * 16.0 + moved * hd * 8.0) + 12 * n, flops=n * hkv * keys * 4.0)


# ---------------------------------------------------------------------------
# 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    hkv, hd = c["hkv"], c["hd"]
    with torch.no_grad():
        if c["op"] in ("shared", "weights"):
            hq = c["hq"]
            grp = hq // hkv
            out = torch.zeros((c["seqs"], hkv, grp, hd), dtype=torch.float64, device=DEV)
            wts = s["wout"].double().clone()
            cut = s["cut"].tolist() if "cut" in s else [0]
            for b in range(c["seqs"]):
                n, r0 = int(s["len"][b]), int(s["row0"][b])
                at = torch.arange(r0, r0 + n, device=DEV)
                shared = 0
                for i in range(len(cut) - 1):
                    if cut[i] <= b < cut[i + 1]:
                        shared, p0 = int(s["plen"][i]), int(s["prow0"][i])
                        at = torch.cat([torch.arange(p0, p0 + shared, device=DEV), at])
                first = max(0, shared + n - c["window"]) if c["window"] > 0 else 0
                at = at[first:]
                wts[b, :, :n] = s["win"][b, :, :n].double()
                if at.numel() == 0:
                    continue
                k = s["k"][at].double().view(-1, hkv, hd)
                v = s["v"][at].double().view(-1, hkv, hd)
                z = torch.einsum("hgd,jhd->hgj", s["q"][b].double().view(hkv, grp, hd), k) / math.sqrt(hd)
                if c["cap"] > 0:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                p = torch.softmax(z, dim=-1)
                out[b] = torch.einsum("hgj,jhd->hgd", p, v)
                skip = max(0, shared - first)                # visible keys of the prefix
                tail = p[..., skip:].sum(dim=1)
                if tail.shape[-1]:
                    wts[b, :, n - tail.shape[-1]:n] += tail
            return out.view(c["seqs"], hq * hd), wts
        if c["op"] == "prompt":
            R, K = c["rows"], c["keys"]
            grp = c["hq"] // hkv
            wts = s["wout"].double().clone()
            wts[..., :K] = s["win"][..., :K].double()
            at = torch.arange(K, device=DEV)
            for b in range(c["batch"]):
                for h in range(c["hq"]):
                    q = s["q"][b, :, h * hd:(h + 1) * hd].double()
                    k = s["k"][b, :, (h // grp) * hd:(h // grp + 1) * hd].double()
                    for r in range(0, R, 1024):
                        z = q[r:r + 1024] @ k.T / math.sqrt(hd)
                        if c["cap"] > 0:
                            z = c["cap"] * torch.tanh(z / c["cap"])
                        pos = (K - R + r + torch.arange(z.shape[0], device=DEV))[:, None]
                        last = pos if c["mask"] == 0 else pos.clamp_min(c["prefix"] - 1) if c["mask"] == 1 else K - 1
                        hide = (at > last) | ((at <= pos - c["window"]) if c["window"] > 0 else (at < 0))
                        wts[b, h // grp, :K] += torch.softmax(z.masked_fill(hide, -math.inf), dim=-1).sum(dim=0)
            return wts
        wts = s["wout"].double().clone()
        k, v = s["k"].double().view(-1, hkv, hd), s["v"].double().view(-1, hkv, hd)
        for b in range(c["seqs"]):
            n, r0, seen = int(s["len"][b]), int(s["row0"][b]), int(s["seen"][b])
            wts[b, :, :n] = s["win"][b, :, :n].double()
            if n <= c["budget"]:
                continue
            at = torch.arange(n, device=DEV)
            for h in range(hkv):
                pos = s["pin"][b, h, :n].long()
                pos = torch.where(pos < 0, seen - n + at, pos)
                score = s["win"][b, h, :n].double()
                score[(pos < c["sink"]) | (pos >= seen - c["recent"])] = math.inf
                order = torch.argsort(-score, stable=True)
                gone = torch.ones(n, dtype=torch.bool, device=DEV)
                gone[order[:c["budget"]]] = False
                to = at[:c["budget"]][gone[:c["budget"]]]
                frm = at[c["budget"]:][~gone[c["budget"]:]]
                k[r0 + to, h], v[r0 + to, h] = k[r0 + frm, h], v[r0 + frm, h]
                wts[b, h, to] = wts[b, h, frm]
                wts[b, h, c["budget"]:n] = 0.0
        return k.view(s["k"].shape), v.view(s["v"].shape), wts, None, None
