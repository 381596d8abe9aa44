"""Eviction to a budget and the attention weights of a prompt (Part 6 of smol_b200.h), and the
four operators together as a serving loop uses them.

Eviction is compared exactly with a plain implementation, slot by slot.  Prompt weights are
compared with 64 bits; the bound of a weight, from the arithmetic (x: scores in natural
units, eps = 2^-23): a probability is off by a factor 1 +- 2d with
d = eps * ((hd/16 + 4) * max sum|qk| * scale + 3 |x| + 8 cap + |lse| + 66)
(fp32 accumulation of hd/16 products, the roundings of x, softcap's tanhf and divisions,
the rounding of lse, sums in chains of at most 64, two ex2.approx), the sum over rows adds
64 eps, the addition to the old weight eps of the result.
"""
import math

import numpy as np
import pytest
import torch

import smol_b200

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -23


@pytest.fixture(autouse=True)
def _clean():
    smol_b200.clear_error()
    yield


def no_error():
    assert smol_b200.last_error() == 0
    assert smol_b200.device_error() == 0


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def plan(w, pos, n, seen, budget, sink, recent):
    """(positions made explicit, holes, movers) of one head, plainly."""
    pos = np.where(pos[:n] < 0, seen - n + np.arange(n), pos[:n])
    if n <= budget:
        return pos, [], []
    w = w[:n].astype(np.float64)
    safe = (pos < sink) | (pos >= seen - recent)
    cls = np.where(safe, 0, np.where(np.isnan(w), 2, 1))
    val = np.where(cls == 1, -w + 0.0, 0.0)
    kept = np.zeros(n, bool)
    kept[np.lexsort((np.arange(n), val, cls))[:budget]] = True
    return pos, np.flatnonzero(~kept[:budget]).tolist(), (budget + np.flatnonzero(kept[budget:])).tolist()


class Evict:
    def __init__(self, cuda, lens, hkv, hd, stride=None, seed=0, ties=False, special=False, gap=2):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=cuda).manual_seed(seed)
        self.lens, self.hkv, self.hd, self.n = list(lens), hkv, hd, len(lens)
        self.stride = stride or max(lens) + 3
        self.max_len = max(lens)
        self.row0 = np.cumsum([1] + [x + gap for x in lens])[:-1].astype(np.int64)
        self.rows = int(self.row0[-1]) + self.lens[-1] + gap
        self.k = torch.randn((self.rows, hkv * hd), device=cuda, generator=g).to(torch.bfloat16)
        self.v = torch.randn((self.rows, hkv * hd), device=cuda, generator=g).to(torch.float16)
        w = np.exp(2 * rng.standard_normal((self.n, hkv, self.stride))).astype(np.float32)
        if ties:
            w = rng.integers(0, 3, size=w.shape).astype(np.float32)
        if special:
            pick = rng.integers(0, 8, size=w.shape)
            for i, x in enumerate((np.nan, np.inf, -np.inf, -0.0, 0.0, -1.0)):
                w[pick == i] = x
        self.w = w
        self.pos = np.full(w.shape, -1, np.int32)
        self.seen = []
        for b, n in enumerate(self.lens):
            old = n // 3   # slots placed by an earlier eviction, in any order
            for h in range(hkv):
                self.pos[b, h, :old] = rng.permutation(max(1, 2 * old))[:old]
            self.seen.append(2 * old + (n - old))
        self.cuda = cuda

    def dev(self, a, dtype):
        return torch.from_numpy(np.ascontiguousarray(a)).to(self.cuda).to(dtype)

    def run(self, budget, sink=0, recent=0, in_place=False, max_len=None):
        k0, v0 = self.k.clone(), self.v.clone()
        w, pos = self.dev(self.w, torch.float32), self.dev(self.pos, torch.int32)
        lens = self.dev(np.array(self.lens), torch.int32)
        if in_place:
            wo, po, lo = w, pos, lens
        else:
            wo, po = torch.full_like(w, 7.0), torch.full_like(pos, 77)
            lo = torch.full_like(lens, 777)
        maxl = self.max_len if max_len is None else max_len
        ws = torch.full((smol_b200.cache_evict_workspace_bytes(self.n, maxl, self.hkv),), 255, dtype=torch.uint8,
                        device=self.cuda)
        smol_b200.cache_evict(self.k, self.v, self.rows, self.dev(self.row0, torch.int64), w, wo, pos, po, self.stride,
                              lens, lo, self.dev(np.array(self.seen), torch.int32), self.n, maxl, self.hkv, self.hd,
                              budget, sink, recent, ws)
        torch.cuda.synchronize()
        # the plain form
        wk, wv = k0.view(torch.int16).cpu().numpy().copy(), v0.view(torch.int16).cpu().numpy().copy()
        ww = self.w.copy() if in_place else np.full(self.w.shape, 7.0, np.float32)
        wp = self.pos.copy() if in_place else np.full(self.pos.shape, 77, np.int32)
        wk, wv = wk.reshape(self.rows, self.hkv, self.hd), wv.reshape(self.rows, self.hkv, self.hd)
        for b, n in enumerate(self.lens):
            for h in range(self.hkv):
                p, holes, movers = plan(self.w[b, h], self.pos[b, h], n, self.seen[b], budget, sink, recent)
                assert len(holes) == len(movers)
                ww[b, h, :n] = self.w[b, h, :n]
                wp[b, h, :n] = self.pos[b, h, :n] if n <= budget else p
                r = self.row0[b]
                for d, s in zip(holes, movers):
                    ww[b, h, d], wp[b, h, d] = self.w[b, h, s], p[s]
                    wk[r + d, h], wv[r + d, h] = wk[r + s, h], wv[r + s, h]
                if n > budget:
                    ww[b, h, budget:n], wp[b, h, budget:n] = 0.0, -1
        assert np.array_equal(lo.cpu().numpy(), np.minimum(self.lens, budget))
        assert np.array_equal(wo.cpu().numpy(), ww, equal_nan=True)
        assert np.array_equal(po.cpu().numpy(), wp)
        assert np.array_equal(self.k.view(torch.int16).cpu().numpy().reshape(wk.shape), wk)
        assert np.array_equal(self.v.view(torch.int16).cpu().numpy().reshape(wv.shape), wv)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([1], 1, 0, 0), ([2], 1, 0, 1), ([2], 1, 1, 0), ([5, 9, 3, 10], 4, 1, 2), ([129, 128, 127, 1, 0], 128, 4, 32),
    ([700, 65, 300], 64, 0, 0), ([1500, 1025], 1024, 4, 1020), ([3000], 333, 2, 64)])
def test_evict_small(cuda, lens, budget, sink, recent, in_place):
    Evict(cuda, lens, 3, 64, seed=len(lens) + budget).run(budget, sink, recent, in_place)
    no_error()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,budget", [(4097, 4096), (4099, 50), (9000, 3000), (17000, 16000), (33000, 2048), (70001, 70000),
                                      (140000, 1000)])
def test_evict_long(cuda, n, budget, in_place):
    # one or two heads: clusters of 2 to 8 CTAs, up to 32 slots a thread
    Evict(cuda, [n, n // 2], 1, 8, seed=n).run(budget, 4, min(budget - 4, 40), in_place)
    no_error()


@pytest.mark.parametrize("n,budget", [(20000, 7000), (40000, 39990)])
def test_evict_many_heads_of_long_caches(cuda, n, budget):
    # enough heads that one CTA takes each
    Evict(cuda, [n], 160, 8, seed=n).run(budget, 0, 16, n % 3 == 0)
    no_error()


@pytest.mark.parametrize("hd,hkv", [(8, 2), (72, 3), (128, 8), (256, 1)])
def test_evict_head_dims(cuda, hd, hkv):
    Evict(cuda, [400, 130, 90], hkv, hd, seed=hd).run(100, 4, 20)
    no_error()


@pytest.mark.parametrize("kind", ["ties", "special"])
@pytest.mark.parametrize("n,budget", [(50, 20), (1000, 999), (5000, 100), (20000, 9000)])
def test_evict_ties_and_special_weights(cuda, kind, n, budget):
    # the same weight many times over (lower slots stay), NaN, infinities, both zeros, negatives
    Evict(cuda, [n, n - 1], 2, 8, seed=n, ties=kind == "ties", special=kind == "special").run(budget, 1, 3)
    no_error()


def test_evict_all_equal_and_all_protected(cuda):
    c = Evict(cuda, [300, 100], 2, 16, seed=3)
    c.w[:] = 0.25
    c.run(128, 0, 0)
    c = Evict(cuda, [300, 100], 2, 16, seed=4)
    c.run(64, 32, 32)
    no_error()


def test_evict_larger_bounds(cuda):
    # max_kv_len above every length, and a stride above it
    Evict(cuda, [300, 100], 2, 16, stride=9001, seed=5).run(64, 4, 16, max_len=9000)
    no_error()


def test_evict_flags_what_cannot_be(cuda):
    c = Evict(cuda, [300, 200], 2, 16, seed=6)
    keep = c.lens
    for bad in ("length", "rows"):
        smol_b200.clear_error()
        c = Evict(cuda, [300, 200], 2, 16, seed=6)
        k0 = c.k.clone()
        w, pos = c.dev(c.w, torch.float32), c.dev(c.pos, torch.int32)
        lens = c.dev(np.array([301 if bad == "length" else 300, 200]), torch.int32)
        row0 = c.dev(c.row0 if bad == "length" else np.array([c.rows - 10, c.row0[1]]), torch.int64)
        ws = torch.empty(smol_b200.cache_evict_workspace_bytes(2, 300, 2), dtype=torch.uint8, device=cuda)
        smol_b200.cache_evict(c.k, c.v, c.rows, row0, w, w, pos, pos, c.stride, lens, lens,
                              c.dev(np.array(c.seen), torch.int32), 2, 300, 2, 16, 50, 0, 4, ws)
        torch.cuda.synchronize()
        assert smol_b200.device_error() == 1 << 5
        # the first sequence is left as it was, the second one is evicted
        r1 = int(c.row0[1])
        assert torch.equal(c.k[:r1], k0[:r1]) and not torch.equal(c.k[r1:], k0[r1:])
        assert lens.tolist() == [301 if bad == "length" else 300, 50]
        assert torch.equal(w[0].cpu(), torch.from_numpy(c.w[0]))
    smol_b200.clear_error()
    assert keep == [300, 200]


def test_evict_offsets_past_32_bits(cuda):
    rows = (1 << 32) // 1024 + 4000
    c = Evict(cuda, [900, 500], 8, 128, seed=8)
    k = torch.zeros((rows, 1024), device=cuda, dtype=torch.bfloat16)
    v = torch.zeros((rows, 1024), device=cuda, dtype=torch.float16)
    k[-c.rows:], v[-c.rows:] = c.k, c.v
    ref = Evict(cuda, [900, 500], 8, 128, seed=8)
    ref.run(300, 4, 50)
    w, pos, lens = c.dev(c.w, torch.float32), c.dev(c.pos, torch.int32), c.dev(np.array(c.lens), torch.int32)
    ws = torch.empty(smol_b200.cache_evict_workspace_bytes(2, 900, 8), dtype=torch.uint8, device=cuda)
    smol_b200.cache_evict(k, v, rows, c.dev(c.row0 + (rows - c.rows), torch.int64), w, w, pos, pos, c.stride, lens, lens,
                          c.dev(np.array(c.seen), torch.int32), 2, 900, 8, 128, 300, 4, 50, ws)
    torch.cuda.synchronize()
    assert torch.equal(k[-c.rows:], ref.k) and torch.equal(v[-c.rows:], ref.v)
    assert not k[:-c.rows].any() and not v[:-c.rows].any()
    no_error()


# ---------------------------------------------------------------------------
# prompt weights
# ---------------------------------------------------------------------------
def prompt_check(cuda, batch, rows, keys, hq, hkv, hd, mask=0, q_offset=None, prefix=0, window=0, cap=0.0, weights="add",
                 pad=0, seed=0, big=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q_offset = keys - rows if q_offset is None else q_offset
    # padded rows and batches: strides are not the widths; what lies between is NaN
    qw, kw = hq * hd + pad, hkv * hd + pad
    q = torch.full((batch, rows + 1, qw), float("nan"), device=cuda, dtype=torch.bfloat16)
    k = torch.full((batch, keys + 1, kw), float("nan"), device=cuda, dtype=torch.bfloat16)
    q[:, :rows, :hq * hd] = (torch.randn((batch, rows, hq * hd), device=cuda, generator=g) * big).to(torch.bfloat16)
    k[:, :keys, :hkv * hd] = torch.randn((batch, keys, hkv * hd), device=cuda, generator=g).to(torch.bfloat16)
    stride = keys + 2
    win = torch.rand((batch, hkv, stride), device=cuda, generator=g)
    wout = torch.full_like(win, -3.0)
    if weights == "in place":
        wout = win.clone()
    scale = 1.0 / math.sqrt(hd)
    ws = torch.full((smol_b200.prefill_weights_workspace_bytes(batch, rows, keys, hq, hkv, hd),), 255,
                    dtype=torch.uint8, device=cuda)
    smol_b200.prefill_attention_weights(
        None if weights == "zero" else wout if weights == "in place" else win, wout, stride, q, k, batch, rows, keys, hq,
        hkv, hd, scale, ws, mask_kind=mask, q_offset=q_offset, prefix_len=prefix, window=window, softcap=cap,
        strides=((qw, (rows + 1) * qw), (kw, (keys + 1) * kw)))
    torch.cuda.synchronize()
    grp = hq // hkv
    j = torch.arange(keys, device=cuda)
    for b in range(batch):
        for h in range(hkv):
            kk = k[b, :keys, h * hd:(h + 1) * hd].double()
            add = torch.zeros(keys, dtype=torch.float64, device=cuda)
            d = 0.0
            for hh in range(h * grp, (h + 1) * grp):
                for r0 in range(0, rows, 2048):
                    qq = q[b, r0:min(rows, r0 + 2048), hh * hd:(hh + 1) * hd].double()
                    x = qq @ kk.T * scale
                    if cap > 0:
                        x = cap * torch.tanh(x / cap)
                    pos = (q_offset + r0 + torch.arange(qq.shape[0], device=cuda))[:, None]
                    hi = pos + 1 if mask == 0 else (pos + 1).clamp_min(prefix) if mask == 1 else torch.full_like(pos, keys)
                    see = j < hi
                    if window > 0:
                        see &= j > pos - window
                    xm = x.masked_fill(~see, -math.inf)
                    lse = torch.logsumexp(xm, dim=-1)
                    p = torch.exp(xm - lse[:, None].masked_fill(lse[:, None] == -math.inf, 0.0))
                    add += p.sum(dim=0)
                    mag = float((qq.abs() @ kk.abs().T).max()) * scale
                    fin = lse[torch.isfinite(lse)]
                    d = max(d, EPS * ((hd / 16 + 4) * mag + 3 * float(x.abs().max()) + 8 * cap +
                                      (float(fin.abs().max()) if fin.numel() else 0.0) + 66))
            base = torch.zeros_like(add) if weights == "zero" else win[b, h, :keys].double()
            got = wout[b, h, :keys].double()
            tol = (2 * d + 64 * EPS) * add + EPS * (base + add)
            bad = (got - base - add).abs() > tol
            assert not bad.any(), (b, h, int(bad.sum()), float(((got - base - add).abs() / tol).max()))
            rest = wout[b, h, keys:]
            assert torch.all(rest == (win[b, h, keys:] if weights == "in place" else -3.0))
    no_error()


@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256), (12, 12, 64), (15, 5, 64), (4, 2, 72), (6, 1, 8),
                                       (128, 1, 64), (50, 1, 128)])
@pytest.mark.parametrize("rows,keys", [(1, 1), (7, 7), (130, 130), (5, 300), (300, 700)])
def test_prompt_shapes(cuda, hq, hkv, hd, rows, keys):
    prompt_check(cuda, 2, rows, keys, hq, hkv, hd, pad=8, seed=rows)


@pytest.mark.parametrize("mask,prefix,window", [(0, 0, 1), (0, 0, 100), (0, 0, 500), (1, 1, 0), (1, 200, 0), (1, 600, 0),
                                                (1, 200, 64), (3, 0, 0), (3, 0, 130)])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 128), (15, 5, 64)])
def test_prompt_masks(cuda, mask, prefix, window, hq, hkv, hd):
    prompt_check(cuda, 1, 333, 450, hq, hkv, hd, mask=mask, prefix=prefix, window=window, seed=mask + window)
    prompt_check(cuda, 1, 20, 450, hq, hkv, hd, mask=mask, prefix=prefix, window=window, seed=mask + window)


@pytest.mark.parametrize("rows,keys,q_offset,window", [(50, 20, -30, 0), (40, 100, 500, 64), (300, 100, -100, 0),
                                                       (64, 64, -64, 0)])
def test_prompt_rows_without_keys(cuda, rows, keys, q_offset, window):
    # rows before every key, rows whose window lies behind the last key
    prompt_check(cuda, 1, rows, keys, 4, 2, 64, q_offset=q_offset, window=window, seed=2)


@pytest.mark.parametrize("big,cap", [(1.0, 50.0), (20.0, 30.0), (15.0, 0.0)])
def test_prompt_large_scores_and_softcap(cuda, big, cap):
    prompt_check(cuda, 1, 200, 600, 4, 2, 128, cap=cap, big=big, seed=4)


@pytest.mark.parametrize("weights", ["in place", "zero"])
def test_prompt_weight_arguments(cuda, weights):
    prompt_check(cuda, 2, 300, 300, 4, 2, 64, weights=weights, seed=5)
    prompt_check(cuda, 2, 10, 300, 4, 2, 64, weights=weights, seed=5)


@pytest.mark.parametrize("rows,keys", [(32, 16384), (3000, 3000), (64, 5000), (65, 5000)])
def test_prompt_long(cuda, rows, keys):
    prompt_check(cuda, 1, rows, keys, 4, 2, 128, seed=6)


def test_prompt_rising_scores_move_the_reference(cuda):
    # every later key tile holds scores larger by more than 2^60 in the exponential
    rows, keys, hd = 40, 1000, 64
    q = torch.ones((1, rows, hd), device=cuda, dtype=torch.bfloat16)
    k = torch.linspace(-60.0, 60.0, keys, device=cuda).view(1, keys, 1).expand(1, keys, hd).to(torch.bfloat16).contiguous()
    w = torch.full((1, 1, keys), -3.0, device=cuda)
    ws = torch.empty(smol_b200.prefill_weights_workspace_bytes(1, rows, keys, 1, 1, hd), dtype=torch.uint8, device=cuda)
    smol_b200.prefill_attention_weights(None, w, keys, q, k, 1, rows, keys, 1, 1, hd, 1.0 / 8, ws, mask_kind=3)
    torch.cuda.synchronize()
    x = (q[0].double() @ k[0].double().T) / 8
    want = torch.softmax(x, dim=-1).sum(dim=0)
    # scores are exact multiples of bf16 steps: their size (up to 480) sets the error of x
    tol = (2 * EPS * (8 * 480 + 700)) * want + 1e-30
    assert ((w[0, 0].double() - want).abs() <= tol).all()
    no_error()


@pytest.mark.parametrize("rows,row", [(300, 5), (300, 140), (20, 7)])
def test_prompt_nan_row_reaches_the_keys_it_sees(cuda, rows, row):
    keys = 300
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn((1, rows, 4 * 64), device=cuda, generator=g).to(torch.bfloat16)
    k = torch.randn((1, keys, 2 * 64), device=cuda, generator=g).to(torch.bfloat16)
    q[0, row, 64:128] = float("nan")            # query head 1, of KV head 0
    w = torch.empty((1, 2, keys), device=cuda)
    ws = torch.empty(smol_b200.prefill_weights_workspace_bytes(1, rows, keys, 4, 2, 64), dtype=torch.uint8, device=cuda)
    smol_b200.prefill_attention_weights(None, w, keys, q, k, 1, rows, keys, 4, 2, 64, 1.0 / 8, ws, q_offset=keys - rows)
    torch.cuda.synchronize()
    seen = keys - rows + row + 1
    assert torch.isnan(w[0, 0, :seen]).all() and torch.isfinite(w[0, 0, seen:]).all() and torch.isfinite(w[0, 1]).all()


def test_prompt_nothing_to_add(cuda):
    win, wout = torch.rand((2, 3, 50), device=cuda), torch.full((2, 3, 50), -3.0, device=cuda)
    q = torch.zeros(64, device=cuda, dtype=torch.bfloat16)
    ws = torch.empty(1024, dtype=torch.uint8, device=cuda)
    smol_b200.prefill_attention_weights(win, wout, 50, q, q, 2, 0, 40, 3, 3, 64, 0.1, ws)
    torch.cuda.synchronize()
    assert torch.equal(wout[..., :40], win[..., :40]) and torch.all(wout[..., 40:] == -3.0)
    no_error()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_serving_loop(cuda):
    """Two sequences on a shared prefix: prompt, weights of its last rows, eviction, then steps that
    append (fused norm, RoPE and append), attend over the prefix and the kept rows, accumulate
    weights and evict one row each.  Every stage is checked on the state the library left."""
    from test_cache_shared_gpu import Case
    hq, hkv, hd, budget, sink, recent, steps = 4, 2, 64, 40, 2, 8, 12
    n, plen, own = 2, 150, [90, 61]
    rng = np.random.default_rng(0)
    cap_rows = 100
    c = Case(cuda, [cap_rows] * n, plens=[plen], cut=[0, n], hq=hq, hkv=hkv, hd=hd, seed=20)
    stride = cap_rows
    weights = torch.zeros((n, hkv, stride), device=cuda)
    positions = torch.full((n, hkv, stride), -1, dtype=torch.int32, device=cuda)
    kv_len = torch.tensor(own, dtype=torch.int32, device=cuda)
    seen = kv_len.clone()
    row0 = c.i64(c.first)
    # the prompt's last 16 rows weigh the own rows
    for b in range(n):
        q = torch.randn((1, 16, hq * hd), device=cuda).to(torch.bfloat16)
        k = c.k[c.first[b]:c.first[b] + own[b]]
        ws = torch.empty(smol_b200.prefill_weights_workspace_bytes(1, 16, own[b], hq, hkv, hd), dtype=torch.uint8,
                         device=cuda)
        smol_b200.prefill_attention_weights(weights[b], weights[b], stride, q, k, 1, 16, own[b], hq, hkv, hd, c.scale,
                                            ws, q_offset=own[b] - 16)
        assert abs(float(weights[b].sum()) - 16 * hq) < 1e-3      # every row hands out 1 per head
    ews = torch.empty(smol_b200.cache_evict_workspace_bytes(n, cap_rows, hkv), dtype=torch.uint8, device=cuda)
    sws = torch.empty(smol_b200.decode_shared_workspace_bytes(n, cap_rows, 1, plen, n, hq, hkv, hd), dtype=torch.uint8,
                      device=cuda)

    def evict():
        w0, p0, l0, s0 = weights.cpu().numpy(), positions.cpu().numpy(), kv_len.tolist(), seen.tolist()
        k0 = c.k.clone()
        smol_b200.cache_evict(c.k, c.v, c.rows, row0, weights, weights, positions, positions, stride, kv_len, kv_len,
                              seen, n, cap_rows, hkv, hd, budget, sink, recent, ews)
        for b in range(n):
            for h in range(hkv):
                p, holes, movers = plan(w0[b, h], p0[b, h], l0[b], s0[b], budget, sink, recent)
                got = positions[b, h, :int(kv_len[b])].cpu().numpy()
                if l0[b] > budget:
                    want = p[:budget].copy()
                    want[holes] = p[movers]
                    assert np.array_equal(got, want)
                    assert set(range(sink)) <= set(got.tolist())
                    assert set(range(s0[b] - recent, s0[b])) <= set(got.tolist())
                for d, s in zip(holes, movers):
                    sl = slice(h * hd, (h + 1) * hd)
                    assert torch.equal(c.k[c.first[b] + d, sl], k0[c.first[b] + s, sl])
        assert kv_len.tolist() == [min(x, budget) for x in l0]

    evict()
    cos = torch.from_numpy(np.cos(rng.uniform(0, 6, (200, hd))).astype(np.float32)).to(cuda)
    sin = torch.sqrt(1 - cos * cos)
    for step in range(steps):
        q, kn, vn = (torch.randn((n, m * hd), device=cuda) for m in (hq, hkv, hkv))
        qr = torch.empty_like(q)
        smol_b200.qknorm_rope_append(q, kn, vn, n, hq, hkv, hd, None, None, 1e-6, cos, sin, False, seen,
                                     row0 + kv_len, qr, None, c.k, c.v, c.rows)
        kv_len += 1
        seen += 1
        before = weights.clone()
        c.q, c.lens, c.stride, c.win = qr, kv_len.tolist(), stride, before
        c.out = torch.full((n, hq * hd), 7.0, device=cuda)
        smol_b200.decode_attention_shared(c.out, qr, c.k, c.v, c.rows, c.i64(c.pfirst), c.i32(c.plens), c.i32(c.cut), 1,
                                          plen, n, row0, kv_len, n, cap_rows, hq, hkv, hd, c.scale, sws,
                                          weights_in=weights, weights_out=weights, weights_stride=stride)
        torch.cuda.synchronize()
        c.check(weights, "in place")
        evict()
        assert max(kv_len.tolist()) <= budget
    no_error()
