"""Part 6 (smol_b200.h) where its numerics are at their limits: NaN scores, probabilities far
below a row's largest, the rounding of bf16 outputs."""
import pytest
import torch

import smol_b200
from test_cache_shared_gpu import EPS, Case, no_error

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    smol_b200.clear_error()
    yield


def rows_of(c, b):
    """Pool rows that sequence b attends, and how many of them are shared."""
    at = torch.arange(c.first[b], c.first[b] + c.lens[b], device=c.dev)
    for i, plen in enumerate(c.plens):
        if c.cut[i] <= b < c.cut[i + 1]:
            return torch.cat([torch.arange(c.pfirst[i], c.pfirst[i] + plen, device=c.dev), at]), plen
    return at, 0


def reference(c, b):
    """Sequence b in 64 bits: out [hkv, grp, hd], added weights of its own keys [hkv, n], probabilities, values."""
    grp = c.hq // c.hkv
    at, shared = rows_of(c, b)
    k, v = c.k[at].double().view(-1, c.hkv, c.hd), c.v[at].double().view(-1, c.hkv, c.hd)
    p = torch.softmax(torch.einsum("hgd,jhd->hgj", c.q[b].double().view(c.hkv, grp, c.hd), k) * c.scale, dim=-1)
    return torch.einsum("hgj,jhd->hgd", p, v), p[..., shared:].sum(dim=1), p, v


def head_bounds(c, b):
    """The bound on an fp32 output (test_cache_shared_gpu.py) without what its rounding to bf16 adds."""
    out, _, p, v = reference(c, b)
    grp, n = c.hq // c.hkv, p.shape[-1]
    k = c.k[rows_of(c, b)[0]].double().view(-1, c.hkv, c.hd)
    q = c.q[b].double().view(c.hkv, grp, c.hd)
    x = torch.einsum("hgd,jhd->hgj", q, k) * c.scale
    mag = float(torch.einsum("hgd,jhd->hgj", q.abs(), k.abs()).max()) * c.scale
    d = EPS * ((c.hd / 16 * 3 + 4) * mag + 3 * float(x.abs().max()) + 2)
    a = torch.einsum("hgj,jhd->hgd", p, v.abs())
    return out, (2 * d + 2.0 ** -21 + EPS * (n / 16 + 64)) * a


# ---------------------------------------------------------------------------
# bf16 outputs are rounded once: they lie between the roundings of the two ends of the fp32 bound
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256), (12, 12, 64)])
@pytest.mark.parametrize("seqs,plen", [(8, 0), (2, 3), (40, 3), (40, 130)])
def test_bf16_output_is_rounded_once(cuda, hq, hkv, hd, seqs, plen):
    # few keys: each probability is large and its rounding shows
    lens = [1 + i % 5 for i in range(seqs)]
    c = Case(cuda, lens, plens=[plen] if plen else [], cut=[0, seqs] if plen else [0], hq=hq, hkv=hkv, hd=hd, q_bf16=True,
             out_bf16=True, seed=41)
    c.run()
    for b in range(seqs):
        want, tol = head_bounds(c, b)
        got = c.out[b].float().view(want.shape)
        # the ends go to fp32 first: half an fp32 step more on each side
        tol = tol + EPS / 2 * want.abs()
        lo, hi = ((want + s * tol).float().to(torch.bfloat16).float() for s in (-1, 1))
        bad = (got < lo) | (got > hi)
        assert not bad.any(), (b, int(bad.sum()), bad.numel())
    no_error()


# ---------------------------------------------------------------------------
# a key that takes nearly all of a row but has no value (an attention sink): the others, each far
# below it, are the whole output
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256), (4, 2, 64)])
@pytest.mark.parametrize("below", [6.3, 14.3, 19.3, 22.3])
@pytest.mark.parametrize("seqs,where", [(3, "own"), (3, "prefix"), (30, "prefix")])
@pytest.mark.parametrize("bf16", [False, True])
def test_values_far_below_a_sink(cuda, hq, hkv, hd, below, seqs, where, bf16):
    # scores in log2 units are 0 for the sink and -below for every other key.  A probability multiplies V
    # as an fp16 value and its remainder, both subnormal below 2^-14: the bound of test_cache_shared_gpu.py
    # plus 2^-32 of the largest probability (that of a value of at least 2^7 before fp16's 2^-25) for
    # each key that is visible
    own, plen = (900, 40) if where == "own" else (3, 900)
    c = Case(cuda, [own] * seqs, plens=[plen], cut=[0, seqs], hq=hq, hkv=hkv, hd=hd, q_bf16=bf16, out_bf16=bf16, seed=42)
    q = torch.zeros_like(c.q).view(seqs, hq, hd)
    q[..., 0] = 1.0
    c.q = q.view(seqs, hq * hd)
    step = below / 1.4426950408889634 / c.scale      # of a key's first element, q is 1 there
    firsts = c.first if where == "own" else c.pfirst
    for r, n in list(zip(c.pfirst, c.plens)) + list(zip(c.first, c.lens)):
        k = torch.zeros((n, hkv, hd), device=cuda)
        k[..., 0] = -step
        v = 1.0 + torch.rand((n, hkv, hd), device=cuda)
        if r in firsts:
            k[0] = v[0] = 0.0
        c.k[r:r + n] = k.view(n, -1).to(torch.bfloat16)
        c.v[r:r + n] = v.view(n, -1).to(torch.float16)
    c.run()
    for b in range(seqs):
        want, tol = head_bounds(c, b)
        _, _, p, v = reference(c, b)
        tol = tol + p.shape[-1] * 2.0 ** -32 * p.amax(dim=-1, keepdim=True) * float(v.max())
        got = c.out[b].double().view(want.shape)
        if bf16:
            tol = tol + 2.0 ** -8 * want.abs()
        bad = (got - want).abs() > tol
        assert not bad.any(), (b, int(bad.sum()), float(((got - want).abs() / tol).max()))
    no_error()


# ---------------------------------------------------------------------------
# NaN scores reach every output and weight that the formula gives NaN, and no other
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256), (4, 2, 64)])
@pytest.mark.parametrize("kind", ["query", "own key alone in a part", "own key beside others", "only key", "first prefix key",
                                  "prefix key alone in a part", "own key of one head"])
@pytest.mark.parametrize("seqs", [2, 30])
@pytest.mark.parametrize("bf16", [False, True])
def test_nan_scores(cuda, hq, hkv, hd, kind, seqs, bf16):
    # 65 own keys: the last is alone in its tile, and in its part where a part is 64 keys; 129 prefix
    # keys: alone in a part of 128 (tensor-core form) or in a tile
    lens = [65, 1] + [7 + i % 3 for i in range(seqs - 2)]
    plens = [] if kind == "only key" else [129]
    c = Case(cuda, lens, plens=plens, cut=[0, seqs] if plens else [0], hq=hq, hkv=hkv, hd=hd, q_bf16=bf16, out_bf16=bf16,
             seed=43)
    nan = float("nan")
    if kind == "query":
        c.q[0, hd:2 * hd] = nan
    elif kind == "only key":
        c.k[c.first[1], :hd] = nan
    elif kind.startswith("own key"):
        at, cols = {"own key alone in a part": (64, slice(None)), "own key beside others": (3, slice(None)),
                    "own key of one head": (64, slice((hkv - 1) * hd, hkv * hd))}[kind]
        c.k[c.first[0] + at, cols] = nan
    else:
        c.k[c.pfirst[0] + (0 if kind.startswith("first") else 128), :hd] = nan
    w = c.run("zero")
    for b in range(seqs):
        want, add, _, _ = reference(c, b)
        got = c.out[b].view(want.shape)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), b
        assert torch.equal(torch.isnan(w[b, :, :lens[b]]), torch.isnan(add)), b
    no_error()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,keys,mask,window,at", [
    (129, 129, 0, 0, 128),      # the last row's own key, alone in its tile
    (300, 300, 0, 0, 256), (257, 257, 3, 0, 256), (300, 513, 3, 0, 512), (300, 513, 0, 100, 511),
    (1, 129, 0, 0, 128), (20, 257, 3, 0, 256), (40, 1025, 3, 0, 1024), (7, 300, 0, 3, 298), (3, 1, 3, 0, 0),
    (300, 300, 1, 0, 299), (64, 64, 0, 0, 63)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_prompt_nan_key(cuda, hd, rows, keys, mask, window, at, cap):
    hq, hkv = 4, 2
    g = torch.Generator(device=cuda).manual_seed(44)
    q = torch.randn((1, rows, hq * hd), device=cuda, generator=g).to(torch.bfloat16)
    k = torch.randn((1, keys, hkv * hd), device=cuda, generator=g).to(torch.bfloat16)
    k[0, at, :hd] = float("nan")
    w = torch.full((1, hkv, keys), -3.0, device=cuda)
    ws = torch.full((smol_b200.prefill_weights_workspace_bytes(1, rows, keys, hq, hkv, hd),), 255, dtype=torch.uint8,
                    device=cuda)
    prefix = keys // 2 if mask == 1 else 0
    smol_b200.prefill_attention_weights(None, w, keys, q, k, 1, rows, keys, hq, hkv, hd, hd ** -0.5, ws, mask_kind=mask,
                                        q_offset=keys - rows, prefix_len=prefix, window=window, softcap=cap)
    torch.cuda.synchronize()
    j, pos = torch.arange(keys, device=cuda), torch.arange(keys - rows, keys, device=cuda)[:, None]
    see = {0: j <= pos, 1: (j <= pos) | (j < prefix), 3: j < keys + 0 * pos}[mask]
    if window > 0:
        see = see & (j > pos - window)
    for h in range(hkv):
        want = torch.zeros(keys, dtype=torch.float64, device=cuda)
        for hh in (2 * h, 2 * h + 1):
            x = q[0, :, hh * hd:(hh + 1) * hd].double() @ k[0, :, h * hd:(h + 1) * hd].double().T * hd ** -0.5
            x = cap * torch.tanh(x / cap) if cap > 0 else x
            p = torch.softmax(x.masked_fill(~see, -float("inf")), dim=-1)
            want += torch.where(see, p, torch.zeros_like(p)).sum(dim=0)
        assert torch.equal(torch.isnan(w[0, h]), torch.isnan(want)), h
    no_error()
