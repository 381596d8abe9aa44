"""Cases of Part 6 (smol_b200.h) in which timing, special values or the order of launches
decide: repeated many times, beside other work, captured, on two streams.

Comparisons are with the 64-bit forms and derived bounds of test_cache_shared_gpu.py and
test_cache_evict_gpu.py, or bit for bit with another run of the same call.
"""

import os
import subprocess
import sys

import pytest
import torch

import smol_b200
from test_cache_evict_gpu import Evict
from test_cache_shared_gpu import EPS, Case, no_error

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    smol_b200.clear_error()
    yield


def shared_call(c, weights_in=None, weights_out=None):
    """The shared decode of a Case as a call without arguments, all its buffers made."""
    n, groups = len(c.lens), [b - a for a, b in zip(c.cut, c.cut[1:])]
    maxl, maxp = max(c.lens), max(c.plens)
    ws = torch.full((smol_b200.decode_shared_workspace_bytes(n, maxl, len(c.plens), maxp, max(groups), c.hq, c.hkv, c.hd),),
                    255, dtype=torch.uint8, device=c.dev)
    args = (c.i64(c.pfirst), c.i32(c.plens), c.i32(c.cut), len(c.plens), maxp, max(groups), c.i64(c.first), c.i32(c.lens),
            n, maxl, c.hq, c.hkv, c.hd, c.scale, ws)

    def call():
        smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, *args, window=c.window, softcap=c.cap,
                                          weights_in=weights_in, weights_out=weights_out,
                                          weights_stride=0 if weights_out is None else c.stride)
    return call


# ---------------------------------------------------------------------------
# the last tile of a prefix part, whose V rows past the keys are cleared
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("plen", [33, 65, 100, 1000, 4099])
@pytest.mark.parametrize("hq,hkv,hd,bf16", [(8, 1, 256, False), (8, 1, 256, True), (16, 8, 128, False), (4, 2, 64, False)])
def test_last_tile_of_a_ragged_prefix(cuda, plen, hq, hkv, hd, bf16):
    # enough sequences for the tensor-core kernel, long own rows beside it, NaN behind the prefix:
    # a row of V cleared too early, or not at all, shows in every one of its sequences
    c = Case(cuda, [2000 + i for i in range(12)], plens=[plen], cut=[0, 12], hq=hq, hkv=hkv, hd=hd, q_bf16=bf16, seed=31)
    call = shared_call(c)
    call()
    torch.cuda.synchronize()
    c.check(None)
    first = c.out.clone()
    for _ in range(200):
        c.out.fill_(7.0)
        call()
        assert torch.equal(c.out, first)
    no_error()


# ---------------------------------------------------------------------------
# eviction by clusters
# ---------------------------------------------------------------------------
class EvictCall:
    """The eviction of an Evict case as a call without arguments, and its buffers."""

    def __init__(self, c, budget, sink=0, recent=0, in_place=True, max_len=None):
        self.c, maxl = c, c.max_len if max_len is None else max_len
        self.start = [c.k.clone(), c.v.clone(), c.dev(c.w, torch.float32), c.dev(c.pos, torch.int32),
                      c.dev(c.lens, torch.int32)]
        w, pos, lens = (x.clone() for x in self.start[2:])
        wo, po, lo = (w, pos, lens) if in_place else (torch.full_like(w, 7.0), torch.full_like(pos, 77), lens.clone())
        self.ins, self.outs = [c.k, c.v, w, pos, lens], [c.k, c.v, wo, po, lo]
        ws = torch.full((smol_b200.cache_evict_workspace_bytes(c.n, maxl, c.hkv),), 255, dtype=torch.uint8, device=c.cuda)
        self.args = (c.k, c.v, c.rows, c.dev(c.row0, torch.int64), w, wo, pos, po, c.stride, lens, lo,
                     c.dev(c.seen, torch.int32), c.n, maxl, c.hkv, c.hd, budget, sink, recent, ws)

    def reset(self):
        for x, x0 in zip(self.ins, self.start):
            x.copy_(x0)

    def __call__(self):
        smol_b200.cache_evict(*self.args)

    def results(self):
        return [x.clone() for x in self.outs]


@pytest.mark.parametrize("units,n,budget", [(1, 5000, 4000), (8, 17000, 2048), (18, 9000, 100), (40, 3000, 2999),
                                            (3, 140000, 70000)])
def test_evict_clusters_many_times(cuda, units, n, budget):
    # the CTAs of many clusters start at different times: other work holds SMs while they are launched
    c = Evict(cuda, [n], units, 8, seed=units)
    call = EvictCall(c, budget, 4, 30)
    c.run(budget, 4, 30, in_place=True)      # against the plain form; moves c's rows in place
    want = [c.k.clone(), c.v.clone()]
    other, busy = torch.cuda.Stream(), torch.randn((3001, 3001), device=cuda)
    for i in range(100):
        call.reset()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            busy * 1.5 if i % 2 else busy @ busy
        call()
        torch.cuda.synchronize()
        got = call.results()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        if i == 0:
            want += got[2:]
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, want))
    no_error()


@pytest.mark.parametrize("row0", [-1, -(1 << 63), (1 << 63) - 1, (1 << 63) - 300, 1 << 32])
def test_evict_flags_rows_anywhere_outside_the_pool(cuda, row0):
    c = Evict(cuda, [300, 200], 2, 16, seed=33)
    k0, v0 = c.k.clone(), c.v.clone()
    call = EvictCall(c, 50, 0, 4)
    call.args[3][0] = row0
    call()
    torch.cuda.synchronize()
    assert smol_b200.device_error() == 1 << 5
    smol_b200.clear_error()
    k, v, w, pos, lens = call.results()
    r1 = int(c.row0[1])
    assert torch.equal(k[:r1], k0[:r1]) and torch.equal(v[:r1], v0[:r1]) and not torch.equal(k[r1:], k0[r1:])
    assert lens.tolist() == [300, 50]
    assert torch.equal(w[0].cpu(), torch.from_numpy(c.w[0])) and torch.equal(pos[0].cpu(), torch.from_numpy(c.pos[0]))


# ---------------------------------------------------------------------------
# a step right behind the kernels that write its inputs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seqs", [3, 24])
@pytest.mark.parametrize("hq,hkv,hd", [(16, 8, 128), (8, 1, 256)])
def test_steps_read_what_the_kernels_before_them_wrote(cuda, seqs, hq, hkv, hd):
    # append (K, V and the rotated queries), the counters, the decode: once with a wait after every
    # launch, once replayed from a graph 30 steps in a row; few and many packed rows
    steps, own = 30, [1 + 7 * i % 90 for i in range(seqs)]
    g = torch.Generator(device=cuda).manual_seed(34)
    bank = [torch.randn((steps, seqs, m * hd), device=cuda, generator=g) for m in (hq, hkv, hkv)]
    angle = torch.rand((300, hd), device=cuda, generator=g) * 6
    cos, sin = angle.cos(), angle.sin()

    def run(captured):
        c = Case(cuda, [150] * seqs, plens=[500], cut=[0, seqs], hq=hq, hkv=hkv, hd=hd, seed=35)
        kv_len, step = c.i32(own), torch.zeros(1, dtype=torch.int64, device=cuda)
        row0, q = c.i64(c.first), torch.empty((seqs, hq * hd), device=cuda)
        outs = torch.zeros((steps, seqs, hq * hd), device=cuda)
        weights = torch.zeros((seqs, hkv, c.stride), device=cuda)
        ws = torch.full((smol_b200.decode_shared_workspace_bytes(seqs, 150, 1, 500, seqs, hq, hkv, hd),), 255,
                        dtype=torch.uint8, device=cuda)
        fixed = (c.i64(c.pfirst), c.i32(c.plens), c.i32(c.cut))

        def one(wait):
            x = [b.index_select(0, step)[0] for b in bank]
            slots = row0 + kv_len
            pos = kv_len.clone()
            kv_len.add_(1)
            wait()
            smol_b200.qknorm_rope_append(*x, seqs, hq, hkv, hd, None, None, 1e-6, cos, sin, False, pos, slots, q, None, c.k,
                                         c.v, c.rows)
            wait()
            smol_b200.decode_attention_shared(c.out, q, c.k, c.v, c.rows, *fixed, 1, 500, seqs, row0, kv_len, seqs, 150, hq,
                                              hkv, hd, c.scale, ws, weights_in=weights, weights_out=weights,
                                              weights_stride=c.stride)
            wait()
            outs.index_copy_(0, step, c.out[None])
            step.add_(1)

        if captured:
            s = torch.cuda.Stream()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s):
                one(lambda: None)      # first use outside the capture
            torch.cuda.synchronize()
            kv_len.copy_(c.i32(own))
            step.zero_()
            weights.zero_()
            with torch.cuda.graph(graph, stream=s):
                one(lambda: None)
            for _ in range(steps):
                graph.replay()
        else:
            for _ in range(steps):
                one(torch.cuda.synchronize)
        torch.cuda.synchronize()
        # the last step against 64 bits (its weights: what the steps before left is not known here)
        c.q, c.lens = q, kv_len.tolist()
        assert c.lens == [x + steps for x in own]
        c.check(None)
        return outs, weights, kv_len

    want = run(False)
    for _ in range(3):
        for a, b in zip(run(True), want):
            assert torch.equal(a, b)
    no_error()


# ---------------------------------------------------------------------------
# captured, repeated, on two streams, without programmatic launches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("w_in_place", [False, True])
@pytest.mark.parametrize("pos_in_place", [False, True])
@pytest.mark.parametrize("len_in_place", [False, True])
@pytest.mark.parametrize("n,budget", [(300, 70), (9000, 3000)])
def test_evict_each_output_may_be_its_input(cuda, w_in_place, pos_in_place, len_in_place, n, budget):
    c = Evict(cuda, [n, budget - 1], 2, 8, seed=36)
    whole = EvictCall(c, budget, 4, 20, in_place=True)
    whole()
    k, v, w, pos, lens = whole.results()
    whole.reset()
    call = EvictCall(c, budget, 4, 20, in_place=False)
    args, wo, po, lo = list(call.args), call.outs[2], call.outs[3], call.outs[4]
    for flag, src, dst in ((w_in_place, 4, 5), (pos_in_place, 6, 7), (len_in_place, 9, 10)):
        if flag:
            args[dst] = args[src]
    smol_b200.cache_evict(*args)
    wo, po, lo = args[5], args[7], args[10]
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v.view(torch.int16))
    assert torch.equal(lo, lens)
    for b, length in enumerate(c.lens):
        assert torch.equal(wo[b, :, :length], w[b, :, :length]) and torch.equal(po[b, :, :length], pos[b, :, :length])
        if not w_in_place:
            assert torch.all(wo[b, :, length:] == 7.0)
        if not pos_in_place:
            assert torch.all(po[b, :, length:] == 77)
    no_error()


class PromptCall:
    """Weights of prompt rows as a call without arguments (weights_in apart from weights_out)."""

    def __init__(self, cuda, batch, rows, keys, hq, hkv, hd, seed=0, **kw):
        g = torch.Generator(device=cuda).manual_seed(seed)
        q = torch.randn((batch, rows, hq * hd), device=cuda, generator=g).to(torch.bfloat16)
        k = torch.randn((batch, keys, hkv * hd), device=cuda, generator=g).to(torch.bfloat16)
        self.win = torch.rand((batch, hkv, keys), device=cuda, generator=g)
        self.out = torch.full_like(self.win, -3.0)
        ws = torch.full((smol_b200.prefill_weights_workspace_bytes(batch, rows, keys, hq, hkv, hd),), 255, dtype=torch.uint8,
                        device=cuda)
        self.args = (self.win, self.out, keys, q, k, batch, rows, keys, hq, hkv, hd, hd ** -0.5, ws)
        self.kw = dict(q_offset=keys - rows, **kw)

    def __call__(self):
        smol_b200.prefill_attention_weights(*self.args, **self.kw)


PROMPTS = [(1, 32, 5000, 16, 8, 128), (2, 600, 600, 4, 2, 128), (1, 900, 1300, 8, 1, 256), (3, 130, 400, 15, 5, 64)]


@pytest.mark.parametrize("shape", PROMPTS)
def test_prompt_weights_repeat_and_are_captured(cuda, shape):
    call = PromptCall(cuda, *shape)
    call()
    torch.cuda.synchronize()
    want = call.out.clone()
    assert torch.isfinite(want).all()
    # every row hands out 1 per head
    added = (want - call.win).double().sum(dim=(1, 2))
    assert torch.all((added / (shape[1] * shape[3]) - 1).abs() < 1e-4)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
        call()
    for i in range(20):
        call.out.fill_(-3.0)
        graph.replay() if i % 2 else call()
        assert torch.equal(call.out, want)
    no_error()


@pytest.mark.parametrize("n,budget,units", [(300, 40, 6), (20000, 6000, 3)])
def test_evict_captured(cuda, n, budget, units):
    for in_place in (False, True):
        call = EvictCall(Evict(cuda, [n, n // 2], units, 8, seed=37), budget, 4, 30, in_place=in_place)
        call()
        want = call.results()
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for _ in range(10):
            call.reset()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(call.results(), want))
    no_error()


def test_weights_decode_captured_with_eviction(cuda):
    """A step that appends, attends with weights and evicts in place, replayed, against the same step by step."""
    seqs, hq, hkv, hd, budget, steps, rows = 5, 16, 8, 128, 60, 40, 80
    g = torch.Generator(device=cuda).manual_seed(38)
    bank = [torch.randn((steps, seqs, m * hd), device=cuda, generator=g) for m in (hq, hkv, hkv)]
    cos, sin = torch.ones((300, hd), device=cuda), torch.zeros((300, hd), device=cuda)

    def run(captured):
        c = Case(cuda, [rows] * seqs, hq=hq, hkv=hkv, hd=hd, seed=39)
        kv_len = c.i32([40 + 5 * b for b in range(seqs)])
        seen, step = kv_len.clone(), torch.zeros(1, dtype=torch.int64, device=cuda)
        start = kv_len.clone()
        row0, q = c.i64(c.first), torch.empty((seqs, hq * hd), device=cuda)
        weights = torch.zeros((seqs, hkv, rows), device=cuda)
        positions = torch.full((seqs, hkv, rows), -1, dtype=torch.int32, device=cuda)
        outs = torch.zeros((steps, seqs, hq * hd), device=cuda)
        pools = c.k.clone(), c.v.clone()
        dws = torch.full((smol_b200.decode_weights_workspace_bytes(seqs, rows, hq, hkv, hd),), 255, dtype=torch.uint8, device=cuda)
        ews = torch.full((smol_b200.cache_evict_workspace_bytes(seqs, rows, hkv),), 255, dtype=torch.uint8, device=cuda)

        def one(wait):
            x = [b.index_select(0, step)[0] for b in bank]
            wait()
            smol_b200.qknorm_rope_append(*x, seqs, hq, hkv, hd, None, None, 1e-6, cos, sin, False, seen, row0 + kv_len, q, None,
                                         c.k, c.v, c.rows)
            kv_len.add_(1)
            seen.add_(1)
            wait()
            smol_b200.decode_attention_weights(c.out, q, c.k, c.v, c.rows, row0, kv_len, seqs, rows, hq, hkv, hd, c.scale,
                                               weights, weights, rows, dws)
            wait()
            smol_b200.cache_evict(c.k, c.v, c.rows, row0, weights, weights, positions, positions, rows, kv_len, kv_len, seen,
                                  seqs, rows, hkv, hd, budget, 4, 16, ews)
            wait()
            outs.index_copy_(0, step, c.out[None])
            step.add_(1)

        if captured:
            s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            with torch.cuda.stream(s):
                one(lambda: None)
            torch.cuda.synchronize()
            for x, x0 in ((kv_len, start), (seen, start), (c.k, pools[0]), (c.v, pools[1])):
                x.copy_(x0)
            step.zero_(), weights.zero_(), positions.fill_(-1)
            with torch.cuda.graph(graph, stream=s):
                one(lambda: None)
            for _ in range(steps):
                graph.replay()
        else:
            for _ in range(steps):
                one(torch.cuda.synchronize)
        torch.cuda.synchronize()
        assert max(kv_len.tolist()) == budget
        return outs, weights, positions, kv_len, c.k.view(torch.int16), c.v.view(torch.int16)

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)
    no_error()


def test_all_operators_on_two_streams(cuda):
    # each stream its own tensors and workspaces: prompt weights and eviction beside the shared decode
    shared = Case(cuda, [100 + 13 * i for i in range(40)], plens=[900], cut=[0, 40], seed=40)
    calls = [shared_call(shared, shared.win, shared.wout), PromptCall(cuda, *PROMPTS[1]), PromptCall(cuda, *PROMPTS[0], seed=1),
             EvictCall(Evict(cuda, [9000, 5000], 4, 64, seed=41), 2000, 4, 30, in_place=False)]

    def outputs():
        return [x.clone() for x in [shared.out, shared.wout, calls[1].out, calls[2].out] + calls[3].outs]

    for call in calls:
        call()
    torch.cuda.synchronize()
    want = outputs()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(30):
        calls[3].reset()
        for x in (shared.out, shared.wout, calls[1].out, calls[2].out):
            x.fill_(-3.0)
        torch.cuda.synchronize()
        for i in range(4):
            with torch.cuda.stream(streams[(i + r) % 2]):
                calls[(i + r // 2) % 4]()
        torch.cuda.synchronize()
        for a, b in zip(outputs(), want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    no_error()


@pytest.mark.parametrize("window", [0, 1, 150])
@pytest.mark.parametrize("prefixes", [31, 33, 70])
def test_many_prefixes_with_windows(cuda, prefixes, window):
    cut = [0]
    for i in range(prefixes):
        cut.append(cut[-1] + (9 if i % 5 != 3 else 0))
    c = Case(cuda, [i % 11 for i in range(cut[-1] + 1)], plens=[(i * 29 + 7) % 200 for i in range(prefixes)], cut=cut, hq=4,
             hkv=2, hd=64, window=window, seed=42)
    c.check(c.run())
    no_error()


def test_without_programmatic_launches(cuda):
    """The operators' own tests in a process whose launches are all fully ordered (SMOL_API_PDL=0)."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, SMOL_API_PDL="0")
    run = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-k",
                          "serving_loop or captured or packed_rows or two_streams or prompt_shapes or evict_small or steps_read",
                          os.path.join(here, "test_cache_shared_gpu.py"), os.path.join(here, "test_cache_evict_gpu.py"),
                          os.path.abspath(__file__)], env=env, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-1000:]
    assert " passed" in run.stdout and "skipped" not in run.stdout


@pytest.mark.parametrize("hq,hkv,hd", [(50, 1, 128), (200, 1, 64), (130, 2, 256)])
@pytest.mark.parametrize("seqs", [1, 3])
@pytest.mark.parametrize("bf16", [False, True])
def test_large_groups(cuda, hq, hkv, hd, seqs, bf16):
    # one sequence's heads fill a query tile and more, or a tile starts inside a group
    c = Case(cuda, [70, 0, 9][:seqs], plens=[300], cut=[0, seqs], hq=hq, hkv=hkv, hd=hd, q_bf16=bf16, out_bf16=bf16, seed=43)
    c.check(c.run())
    no_error()


# ---------------------------------------------------------------------------
# device values that are no ranges
# ---------------------------------------------------------------------------
LOW, HIGH = -(1 << 31), (1 << 31) - 1


@pytest.mark.parametrize("seqs", [3, 24])
@pytest.mark.parametrize("ranges", [(HIGH, LOW), (HIGH, HIGH), (LOW, LOW), (1, 0), (5000, LOW), (HIGH - 1, LOW + 1), (-1, -1)])
@pytest.mark.parametrize("prefixes", [1, 40])
def test_ranges_that_are_none_count_as_empty(cuda, seqs, ranges, prefixes):
    # one prefix (a table in registers) and 40 (found item by item), few packed rows and many
    c = Case(cuda, [3 + i % 4 for i in range(seqs)], plens=[200] + [0] * (prefixes - 1), cut=[0, seqs] + [seqs] * (prefixes - 1),
             seed=44)
    n, maxl = seqs, max(c.lens)
    ws = torch.full((smol_b200.decode_shared_workspace_bytes(n, maxl, prefixes, 200, n, 16, 8, 128),), 255, dtype=torch.uint8,
                    device=cuda)

    def run(cut):
        smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, c.i64(c.pfirst), c.i32(c.plens), c.i32(cut), prefixes,
                                          200, n, c.i64(c.first), c.i32(c.lens), n, maxl, 16, 8, 128, c.scale, ws,
                                          weights_in=c.win, weights_out=c.wout, weights_stride=c.stride)
        torch.cuda.synchronize()
        flagged = smol_b200.device_error() & (1 << 5)
        smol_b200.clear_error()
        return flagged

    assert not run(c.cut)
    c.check(c.wout)
    # the first prefix has the bad range, the others (of no rows) whatever follows from its end
    assert run(list(ranges) + [ranges[1]] * (prefixes - 1))
    c.cut, c.plens = [0] * (prefixes + 1), [0] * prefixes
    c.check(c.wout)


@pytest.mark.parametrize("max_len,max_seqs", [(0, 2), (100, 0), (0, 0)])
@pytest.mark.parametrize("plen,end", [(0, 0), (5, 2), (0, 2), (5, 0)])
def test_prefixes_announced_as_none(cuda, max_len, max_seqs, plen, end):
    # bounds of 0 are bounds: a prefix beyond them is left out and flagged
    c = Case(cuda, [70, 9], plens=[5], cut=[0, 2], seed=45)
    ws = torch.empty(smol_b200.decode_shared_workspace_bytes(2, 70, 1, max_len, max_seqs, 16, 8, 128), dtype=torch.uint8,
                     device=cuda)
    smol_b200.decode_attention_shared(c.out, c.q, c.k, c.v, c.rows, c.i64(c.pfirst), c.i32([plen]), c.i32([0, end]), 1, max_len,
                                      max_seqs, c.i64(c.first), c.i32(c.lens), 2, 70, 16, 8, 128, c.scale, ws,
                                      weights_in=c.win, weights_out=c.wout, weights_stride=c.stride)
    torch.cuda.synchronize()
    assert bool(smol_b200.device_error() & (1 << 5)) == (plen > max_len or end > max_seqs)
    smol_b200.clear_error()
    c.plens, c.cut = [0], [0, 0]
    c.check(c.wout)


def test_most_sequences(cuda):
    # as many sequences as are accepted, one of a pool's few rows each, all on one prefix
    n, hd, plen, rows = 65535, 64, 3, 40
    g = torch.Generator(device=cuda).manual_seed(46)
    k = torch.randn((rows, hd), device=cuda, generator=g).to(torch.bfloat16)
    v = torch.randn((rows, hd), device=cuda, generator=g).to(torch.float16)
    q = torch.randn((n, hd), device=cuda, generator=g)
    row0 = torch.arange(n, device=cuda) % (rows - plen) + plen
    lens = (torch.arange(n, device=cuda) % 3 > 0).to(torch.int32)
    out, w = torch.full((n, hd), 7.0, device=cuda), torch.full((n, 1, 1), -3.0, device=cuda)
    ws = torch.empty(smol_b200.decode_shared_workspace_bytes(n, 1, 1, plen, n, 1, 1, hd), dtype=torch.uint8, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    smol_b200.decode_attention_shared(out, q, k, v, rows, torch.zeros(1, dtype=torch.int64, device=cuda),
                                      torch.tensor([plen], **i32), torch.tensor([0, n], **i32), 1, plen, n, row0, lens, n, 1, 1, 1,
                                      hd, 0.125, ws, weights_out=w, weights_stride=1)
    torch.cuda.synchronize()
    x = torch.cat([q.double() @ k[:plen].double().T, (q.double() * k[row0].double()).sum(1, keepdim=True)], 1) * 0.125
    x[lens == 0, plen] = -float("inf")
    p = torch.softmax(x, dim=1)
    want = p[:, :plen] @ v[:plen].double() + p[:, plen:] * v[row0].double()
    a = p[:, :plen] @ v[:plen].double().abs() + p[:, plen:] * v[row0].double().abs()
    # the bound of test_cache_shared_gpu.py
    mag = 0.125 * float((q.double().abs() @ k.double().abs().T).max())
    d = EPS * ((hd / 16 * 3 + 4) * mag + 3 * float(x[:, :plen].abs().max()) + 2)
    assert ((out.double() - want).abs() <= (2 * d + 2.0 ** -21 + 65 * EPS) * a).all()
    seen = lens > 0
    assert ((w[seen, 0, 0].double() - p[seen, plen]).abs() <= (2 * d + 65 * EPS) * p[seen, plen]).all()
    assert torch.all(w[~seen] == -3.0)
    no_error()


@pytest.mark.parametrize("n,budget", [(262144, 100000), (262143, 262142)])
def test_evict_longest(cuda, n, budget):
    Evict(cuda, [n, 1000], 1, 8, seed=47).run(budget, 4, 100, True)
    no_error()
