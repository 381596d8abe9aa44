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
