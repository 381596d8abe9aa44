"""Decode over shared prefixes and with attention weights (Part 6 of smol_b200.h) against a
plain 64-bit implementation, element by element.

Tolerances are bounds derived from the arithmetic, computed from each case's inputs.  With
x the score of a key (natural units), A = sum_j p_j |v_j| and eps = 2^-23:
* score: an fp32 accumulation of hd/16 * terms + 4 partial products of size sum_d |q_d k_d|,
  three roundings of x itself, softcap's tanhf and divisions (8 eps * cap), and ex2.approx
  (2 eps on the result):  d = eps * (scale * (hd/16*3 + 4) * max sum|qk| + 3 |x| + 8 cap + 2);
* output: probabilities off by a factor 1 +- 2d, their fp16 remainder form by 2^-21, the sum
  over keys by one eps per 16 keys and per part joined:
  (2d + 2^-21 + eps * (n/16 + 64)) * A, and for a bf16 output half a bf16 step of the result
  (2^-8) and half an fp16 step of the probabilities (2^-11 * A);
* weight: 2d + eps * 64 of the added sum, and eps of the result for the addition.
Every pool row that no sequence owns holds NaN.
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


class Case:
    """A pool with `plens` shared prefixes and sequences of `lens` own rows; cut: first sequence of each prefix."""

    def __init__(self, cuda, lens, plens=(), cut=(0,), hq=16, hkv=8, hd=128, q_bf16=False, out_bf16=False, window=0,
                 cap=0.0, scale=None, seed=0, big=1.0):
        g = torch.Generator(device=cuda).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dev, self.hq, self.hkv, self.hd, self.window, self.cap = cuda, hq, hkv, hd, window, cap
        self.scale = 1.0 / math.sqrt(hd) if scale is None else scale
        self.lens, self.plens, self.cut = list(lens), list(plens), list(cut)
        sizes = self.plens + self.lens
        gaps = rng.integers(1, 9, size=len(sizes) + 1)      # NaN rows between the sequences
        first, at = [], int(gaps[0])
        for n, gap in zip(sizes, gaps[1:]):
            first.append(at)
            at += n + int(gap)
        self.rows = at
        self.k = torch.full((at, hkv * hd), float("nan"), device=cuda, dtype=torch.bfloat16)
        self.v = torch.full((at, hkv * hd), float("nan"), device=cuda, dtype=torch.float16)
        for n, r in zip(sizes, first):
            self.k[r:r + n] = torch.randn((n, hkv * hd), device=cuda, generator=g).to(torch.bfloat16)
            self.v[r:r + n] = torch.randn((n, hkv * hd), device=cuda, generator=g).to(torch.float16)
        self.pfirst, self.first = first[:len(plens)], first[len(plens):]
        n = len(self.lens)
        q = torch.randn((n, hq * hd), device=cuda, generator=g) * big
        self.q = q.to(torch.bfloat16) if q_bf16 else q
        self.out = torch.full((n, hq * hd), 7.0, device=cuda, dtype=torch.bfloat16 if out_bf16 else torch.float32)
        self.stride = max(self.lens + [1]) + 5
        self.win = torch.rand((n, hkv, self.stride), device=cuda, generator=g)
        self.wout = torch.full((n, hkv, self.stride), -3.0, device=cuda)

    def i64(self, x):
        return torch.tensor(x, dtype=torch.int64, device=self.dev)

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def run(self, weights="add", max_len=None, ws=None):
        """weights: 'add' (in and out apart), 'in place', 'zero' (no weights_in), None."""
        n, maxl = len(self.lens), max(self.lens + [0]) if max_len is None else max_len
        w_in, w_out = self.win, self.wout
        if weights == "in place":
            w_out = w_in = self.win.clone()
        elif weights == "zero":
            w_in = None
        elif weights is None:
            w_in = w_out = None
        st = 0 if w_out is None else self.stride
        self.dev_args = (self.i64(self.first), self.i32(self.lens))
        if self.plens:
            groups = [b - a for a, b in zip(self.cut, self.cut[1:])]
            need = smol_b200.decode_shared_workspace_bytes(n, maxl, len(self.plens), max(self.plens), max(groups),
                                                           self.hq, self.hkv, self.hd)
            ws = torch.full((need,), 255, dtype=torch.uint8, device=self.dev) if ws is None else ws
            smol_b200.decode_attention_shared(
                self.out, self.q, self.k, self.v, self.rows, self.i64(self.pfirst), self.i32(self.plens),
                self.i32(self.cut), len(self.plens), max(self.plens), max(groups), *self.dev_args, n, maxl, self.hq,
                self.hkv, self.hd, self.scale, ws, window=self.window, softcap=self.cap, weights_in=w_in,
                weights_out=w_out, weights_stride=st)
        else:
            need = smol_b200.decode_weights_workspace_bytes(n, maxl, self.hq, self.hkv, self.hd)
            ws = torch.full((need,), 255, dtype=torch.uint8, device=self.dev) if ws is None else ws
            smol_b200.decode_attention_weights(
                self.out, self.q, self.k, self.v, self.rows, *self.dev_args, n, maxl, self.hq, self.hkv, self.hd,
                self.scale, w_in, w_out, st, ws, window=self.window, softcap=self.cap)
        torch.cuda.synchronize()
        return w_out

    def check(self, w_out, weights="add"):
        grp, hd = self.hq // self.hkv, self.hd
        for b, n in enumerate(self.lens):
            shared, at = 0, torch.arange(self.first[b], self.first[b] + n, device=self.dev)
            for i, plen in enumerate(self.plens):
                if self.cut[i] <= b < self.cut[i + 1]:
                    shared = plen
                    at = torch.cat([torch.arange(self.pfirst[i], self.pfirst[i] + plen, device=self.dev), at])
            skip = max(0, shared + n - self.window) if self.window > 0 else 0
            at = at[skip:]
            got = self.out[b].double().view(self.hkv, grp, hd)
            add = torch.zeros((self.hkv, n), dtype=torch.float64, device=self.dev)
            if at.numel() == 0:
                assert torch.all(got == 0), b
                d = 0.0
            else:
                k, v = self.k[at].double().view(-1, self.hkv, hd), self.v[at].double().view(-1, self.hkv, hd)
                q = self.q[b].double().view(self.hkv, grp, hd)
                x = torch.einsum("hgd,jhd->hgj", q, k) * self.scale
                mag = float(torch.einsum("hgd,jhd->hgj", q.abs(), k.abs()).max()) * self.scale
                if self.cap > 0:
                    x = self.cap * torch.tanh(x / self.cap)
                d = EPS * ((hd / 16 * 3 + 4) * mag + 3 * float(x.abs().max()) + 8 * self.cap + 2)
                p = torch.softmax(x, dim=-1)
                want = torch.einsum("hgj,jhd->hgd", p, v)
                a = torch.einsum("hgj,jhd->hgd", p, v.abs())
                tol = (2 * d + 2.0 ** -21 + EPS * (at.numel() / 16 + 64)) * a
                if self.out.dtype == torch.bfloat16:
                    tol = tol + 2.0 ** -8 * want.abs() + 2.0 ** -11 * a
                assert torch.isfinite(got).all(), b
                bad = (got - want).abs() > tol
                assert not bad.any(), (b, int(bad.sum()), float(((got - want).abs() / tol).max()))
                tail = p[..., max(0, shared - skip):].sum(dim=1)
                if tail.shape[-1]:
                    add[:, n - tail.shape[-1]:] = tail
            if w_out is not None:
                base = torch.zeros_like(add) if weights == "zero" else self.win[b, :, :n].double()
                w = w_out[b, :, :n].double()
                bad = (w - base - add).abs() > (2 * d + 64 * EPS) * add + EPS * (base + add)
                assert not bad.any(), (b, float((w - base - add).abs().max()))
                rest = w_out[b, :, n:]
                assert torch.all(rest == (self.win[b, :, n:] if weights == "in place" else -3.0)), b


HEADS = [(16, 8, 128), (8, 1, 256), (12, 12, 64), (24, 2, 128), (15, 5, 64)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("q_bf16,out_bf16", [(False, False), (True, True), (True, False), (False, True)])
def test_weights_against_64_bits(cuda, hq, hkv, hd, q_bf16, out_bf16):
    c = Case(cuda, [1, 0, 63, 64, 65, 700, 130, 16], hq=hq, hkv=hkv, hd=hd, q_bf16=q_bf16, out_bf16=out_bf16, seed=1)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("q_bf16,out_bf16", [(False, False), (True, True), (True, False), (False, True)])
def test_shared_against_64_bits(cuda, hq, hkv, hd, q_bf16, out_bf16):
    # three prefixes of odd lengths (one inside a tile, one empty), a sequence before and one
    # after every range, own rows from none to several tiles
    c = Case(cuda, [5, 0, 1, 64, 33, 200, 0, 17, 9], plens=[300, 0, 77], cut=[1, 4, 6, 8], hq=hq, hkv=hkv, hd=hd,
             q_bf16=q_bf16, out_bf16=out_bf16, seed=2)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("seqs,plen,own", [(1, 1, 0), (1, 1, 1), (2, 127, 3), (70, 129, 1), (33, 1000, 40), (130, 64, 5),
                                           (3, 5000, 1500)])
def test_shared_sizes(cuda, seqs, plen, own):
    c = Case(cuda, [(own * (i + 1)) // seqs for i in range(seqs)], plens=[plen], cut=[0, seqs], q_bf16=seqs % 2 == 0,
             seed=3)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("q_bf16,out_bf16", [(True, True), (True, False), (False, False), (False, True)])
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256), (4, 2, 64)])
def test_full_query_tiles_over_several_key_tiles(cuda, hq, hkv, hd, q_bf16, out_bf16):
    # every row of a query tile in use and many key tiles to a part
    seqs = 128 * hkv // hq + 3
    c = Case(cuda, [i % 5 for i in range(seqs)], plens=[8192], cut=[0, seqs], hq=hq, hkv=hkv, hd=hd, q_bf16=q_bf16,
             out_bf16=out_bf16, seed=15)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("window", [1, 2, 10, 64, 100, 333, 5000])
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256)])
def test_window_over_prefix_and_own_rows(cuda, window, hq, hkv, hd):
    # windows that end in the own rows, in the prefix, and before both; every row differs
    c = Case(cuda, [0, 1, 9, 10, 11, 150, 64], plens=[200, 333], cut=[0, 4, 7], hq=hq, hkv=hkv, hd=hd, window=window,
             seed=4)
    c.check(c.run())
    c = Case(cuda, [0, 1, 9, 10, 11, 150, 64], hq=hq, hkv=hkv, hd=hd, window=window, seed=4)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("big,cap", [(1.0, 50.0), (20.0, 30.0), (12.0, 0.0)])
def test_large_scores_and_softcap(cuda, big, cap):
    # scores up to hundreds: the reference point of a row moves, most probabilities vanish
    c = Case(cuda, [400, 3, 90], plens=[700], cut=[0, 3], cap=cap, big=big, seed=5)
    c.check(c.run())
    no_error()


def test_rising_scores_move_the_reference(cuda):
    # keys along q with growing length: every later tile holds a larger maximum, by far more
    # than 2^15, in the prefix and in the own rows
    c = Case(cuda, [260, 100], plens=[600], cut=[0, 2], hq=2, hkv=1, hd=64, seed=6)
    q = c.q.view(2, 2, 64)
    q[:] = q[0, 0].sign()
    for r, n, lo, hi in ((c.pfirst[0], 600, -8.0, 4.0), (c.first[0], 260, 4.0, 6.0), (c.first[1], 100, -9.0, -2.0)):
        f = torch.linspace(lo, hi, n, device=cuda).view(n, 1)
        c.k[r:r + n] = (q[0, 0].view(1, 64) * f).to(torch.bfloat16)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("weights", ["in place", "zero", None])
def test_weight_arguments(cuda, weights):
    c = Case(cuda, [5, 1100, 0, 64], plens=[100], cut=[0, 3], seed=7)
    c.check(c.run(weights), weights)
    if weights is not None:
        c = Case(cuda, [5, 1100, 0, 2049], seed=8)
        c.check(c.run(weights), weights)
    no_error()


def test_infinities_past_every_length(cuda):
    c = Case(cuda, [5, 70], plens=[65], cut=[0, 2], seed=9)
    for pool in (c.k, c.v):
        pool[torch.isnan(pool[:, 0])] = float("inf")
    c.check(c.run())
    no_error()


def test_repeats_are_identical_and_longer_bounds_serve(cuda):
    c = Case(cuda, [900, 17, 300], plens=[1000], cut=[0, 3], seed=10)
    w = c.run()
    first, w1 = c.out.clone(), w.clone()
    w = c.run()
    assert torch.equal(first, c.out) and torch.equal(w1, w)
    # bounds above the real lengths change the split, not what is computed
    c.stride += 4000
    c.win, c.wout = torch.zeros((3, c.hkv, c.stride), device=cuda), torch.full((3, c.hkv, c.stride), -3.0, device=cuda)
    c.check(c.run(max_len=4000))
    # one workspace sized for the longest serves shorter calls
    need = smol_b200.decode_weights_workspace_bytes(3, 9409, 16, 8, 128)
    for n in (9409, 5000, 64, 1):
        c = Case(cuda, [n, 1, n // 2], seed=11)
        c.check(c.run(ws=torch.empty(need, dtype=torch.uint8, device=cuda)))
    no_error()


def test_device_values_beyond_the_announced_are_flagged(cuda):
    c = Case(cuda, [40, 30], seed=12)
    c.run(max_len=32)
    assert smol_b200.device_error() & (1 << 5)
    smol_b200.clear_error()
    # the sequence within the bound is right, the other one attends its first rows
    c.lens[0] = 32
    c.check(c.wout)


def test_captured_step_follows_the_device_lengths(cuda):
    c = Case(cuda, [50, 8], plens=[90], cut=[0, 2], seed=13)
    lens = c.i32([20, 8])
    args = (c.i64(c.pfirst), c.i32(c.plens), c.i32(c.cut), c.i64(c.first))
    ws = torch.empty(smol_b200.decode_shared_workspace_bytes(2, 50, 1, 90, 2, 16, 8, 128), dtype=torch.uint8,
                     device=cuda)

    def step():
        smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, args[0], args[1], args[2], 1, 90, 2, args[3],
                                          lens, 2, 50, 16, 8, 128, c.scale, ws, weights_in=c.win, weights_out=c.wout,
                                          weights_stride=c.stride)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for own in ([20, 8], [50, 0], [1, 1]):
        lens.copy_(c.i32(own))
        c.wout.fill_(-3.0)
        graph.replay()
        torch.cuda.synchronize()
        c.lens = own
        c.check(c.wout)
    no_error()


def test_pool_rows_past_32_bit_offsets(cuda):
    # own rows and a prefix whose element offsets pass 2^32 (a pool of 4.3 GB per array)
    rows = (1 << 32) // 1024 + 600
    c = Case(cuda, [300, 7], plens=[200], cut=[0, 2], seed=14)
    k = torch.empty((rows, 1024), device=cuda, dtype=torch.bfloat16)
    v = torch.empty((rows, 1024), device=cuda, dtype=torch.float16)
    k[-c.rows:], v[-c.rows:] = c.k, c.v
    off = rows - c.rows
    c.k, c.v, c.rows = k, v, rows
    c.pfirst, c.first = [x + off for x in c.pfirst], [x + off for x in c.first]
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("more", [0, 1, 9])
@pytest.mark.parametrize("window", [0, 1, 100, 420])
def test_packed_rows_around_sixteen(cuda, hq, hkv, hd, more, window):
    # sequences x group of up to 16 rows, just above, and well above; a second prefix has a
    # single sequence, and the last sequence none
    seqs = max(1, 16 * hkv // hq) + more
    lens = [(i * 37) % 150 for i in range(seqs)] + [30, 12]
    for bf16 in (False, True):
        c = Case(cuda, lens, plens=[400, 129], cut=[0, seqs, seqs + 1], hq=hq, hkv=hkv, hd=hd, q_bf16=bf16,
                 out_bf16=bf16, window=window, cap=20.0 * more, seed=16)
        c.check(c.run())
    no_error()


@pytest.mark.parametrize("per", [1, 3, 10])
@pytest.mark.parametrize("prefixes", [32, 33, 70])
def test_many_prefixes(cuda, prefixes, per):
    # lengths from none up, groups of `per` sequences and some of none
    cut = [0]
    for i in range(prefixes):
        cut.append(cut[-1] + (per if i % 5 != 3 else 0))
    c = Case(cuda, [i % 7 for i in range(cut[-1] + 1)], plens=[i * 29 % 200 for i in range(prefixes)], cut=cut, hq=4,
             hkv=2, hd=64, seed=17)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("big,cap", [(1.0, 50.0), (20.0, 30.0), (12.0, 0.0)])
def test_large_scores_of_many_sequences(cuda, big, cap):
    c = Case(cuda, [i * 13 % 90 for i in range(20)], plens=[1300], cut=[0, 20], cap=cap, big=big, seed=18)
    c.check(c.run())
    no_error()


def test_rising_scores_of_many_sequences(cuda):
    c = Case(cuda, [5] * 70, plens=[900], cut=[0, 70], hq=2, hkv=1, hd=64, seed=19)
    q = c.q.view(70, 2, 64)
    q[:] = q[0, 0].sign()
    f = torch.linspace(-8.0, 4.0, 900, device=cuda).view(900, 1)
    c.k[c.pfirst[0]:c.pfirst[0] + 900] = (q[0, 0].view(1, 64) * f).to(torch.bfloat16)
    c.check(c.run())
    no_error()


@pytest.mark.parametrize("seqs", [4, 30])
def test_prefixes_beyond_the_announced_are_flagged(cuda, seqs):
    c = Case(cuda, [3 + i % 4 for i in range(seqs)], plens=[200, 90], cut=[0, seqs - 1, seqs], seed=20)
    n, maxl = seqs, max(c.lens)
    ws = torch.empty(smol_b200.decode_shared_workspace_bytes(n, maxl, 2, 128, seqs - 1, 16, 8, 128), dtype=torch.uint8,
                     device=cuda)

    def run(plens, cut, most):
        smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, c.i64(c.pfirst), c.i32(plens), c.i32(cut), 2, 128,
                                          most, c.i64(c.first), c.i32(c.lens), n, maxl, 16, 8, 128, c.scale, ws,
                                          weights_in=c.win, weights_out=c.wout, weights_stride=c.stride)
        torch.cuda.synchronize()
        flagged = smol_b200.device_error() & (1 << 5)
        smol_b200.clear_error()
        return flagged

    assert run([200, 90], c.cut, seqs - 1)       # longer than announced: its first rows count
    c.plens = [128, 90]
    c.check(c.wout)
    assert not run([128, 90], c.cut, seqs - 1)
    c.check(c.wout)
    assert run([128, 90], [0, seqs - 1, seqs + 5], seqs - 1)   # past the last sequence
    c.check(c.wout)
    assert run([128, -4], c.cut, seqs - 1)       # counts as empty
    c.plens = [128, 0]
    c.check(c.wout)
    assert run([128, 0], c.cut, seqs - 2)        # more sequences than announced: the rest has no prefix
    c.cut = [0, seqs - 2, seqs - 2]
    c.check(c.wout)


@pytest.mark.parametrize("seqs", [3, 21])
def test_captured_step_follows_the_device_prefixes(cuda, seqs):
    c = Case(cuda, [40 + i % 9 for i in range(seqs)], plens=[700, 300], cut=[0, seqs - 1, seqs], seed=21)
    plens, cut, lens = c.i32(c.plens), c.i32(c.cut), c.i32(c.lens)
    pfirst, first = c.i64(c.pfirst), c.i64(c.first)
    maxl = max(c.lens)
    ws = torch.empty(smol_b200.decode_shared_workspace_bytes(seqs, maxl, 2, 700, seqs, 16, 8, 128), dtype=torch.uint8,
                     device=cuda)

    def step():
        smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, pfirst, plens, cut, 2, 700, seqs, first, lens,
                                          seqs, maxl, 16, 8, 128, c.scale, ws, weights_in=c.win, weights_out=c.wout,
                                          weights_stride=c.stride)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for _ in range(3):   # launches of one step after those of another, on one workspace
            step()
    for p, k in (([700, 300], [0, seqs - 1, seqs]), ([0, 1], [0, 1, seqs]), ([130, 300], [0, seqs, seqs]),
                 ([699, 2], [1, 2, 2])):
        plens.copy_(c.i32(p))
        cut.copy_(c.i32(k))
        c.plens, c.cut = p, k
        c.wout.fill_(-3.0)
        graph.replay()
        torch.cuda.synchronize()
        c.check(c.wout)
    no_error()


def test_two_streams_with_their_own_workspaces(cuda):
    cases = [Case(cuda, [100 + 13 * i for i in range(n)], plens=[900], cut=[0, n], seed=22 + n) for n in (5, 40)]
    alone = []
    for c in cases:
        w = c.run()
        alone.append((c.out.clone(), w.clone()))
        c.check(w)
    streams = [torch.cuda.Stream() for _ in cases]
    args = []
    for c in cases:
        n = len(c.lens)
        ws = torch.empty(smol_b200.decode_shared_workspace_bytes(n, max(c.lens), 1, 900, n, 16, 8, 128),
                         dtype=torch.uint8, device=cuda)
        args.append((c.out, c.q, c.k, c.v, c.rows, c.i64(c.pfirst), c.i32(c.plens), c.i32(c.cut), 1, 900, n,
                     c.i64(c.first), c.i32(c.lens), n, max(c.lens), 16, 8, 128, c.scale, ws))
        c.out.zero_()
        c.wout.fill_(-3.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for c, a, s in zip(cases, args, streams):
            with torch.cuda.stream(s):
                smol_b200.decode_attention_shared(*a, weights_in=c.win, weights_out=c.wout, weights_stride=c.stride)
    torch.cuda.synchronize()
    for c, (o, w) in zip(cases, alone):
        assert torch.equal(c.out, o) and torch.equal(c.wout, w)
    no_error()
