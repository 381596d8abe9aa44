"""Part 6 of smol_b200.h without a GPU: what the entry points refuse (before any CUDA call),
and that the workspace of a length serves every shorter one."""
import pytest

import smol_b200

ARGS, WORKSPACE = 1, 6
P = 0x10000   # an aligned address that is never dereferenced


def shared_args(**over):
    a = dict(stream=None, out=P, out_is_bf16=0, q=P, q_is_bf16=0, k_pool=P, v_pool=P, pool_rows=1000, prefix_row0=P,
             prefix_len=P, prefix_seq0=P, n_prefixes=1, max_prefix_len=100, max_prefix_seqs=2, seq_row0=P, kv_len=P,
             n_seqs=2, max_kv_len=50, n_heads=16, n_kv_heads=8, head_dim=128, scale=0.1, window=0, softcap=0.0,
             weights_in=P, weights_out=P, weights_stride=50, workspace=P, workspace_bytes=1 << 40)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over", [
    dict(out=None), dict(q=None), dict(k_pool=None), dict(v_pool=None), dict(seq_row0=None), dict(kv_len=None),
    dict(prefix_row0=None), dict(prefix_len=None), dict(prefix_seq0=None), dict(out=P + 8), dict(q=P + 4),
    dict(k_pool=P + 2), dict(v_pool=P + 8), dict(pool_rows=0), dict(pool_rows=1 << 31), dict(head_dim=72),
    dict(head_dim=512), dict(n_heads=15), dict(n_heads=0), dict(n_kv_heads=0), dict(max_kv_len=-1),
    dict(n_seqs=65536), dict(n_prefixes=-1), dict(n_prefixes=65536), dict(max_prefix_len=-1),
    dict(max_prefix_seqs=3), dict(max_prefix_seqs=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(weights_out=None), dict(weights_stride=49),
])
def test_shared_refuses(over):
    smol_b200.clear_error()
    assert smol_b200.lib().smol_b200_decode_attention_shared(*shared_args(**over)) == ARGS
    assert smol_b200.last_error() == ARGS
    smol_b200.clear_error()


@pytest.mark.parametrize("over", [dict(workspace=None), dict(workspace_bytes=1000), dict(workspace=P + 4)])
def test_shared_refuses_workspaces(over):
    assert smol_b200.lib().smol_b200_decode_attention_shared(*shared_args(**over)) == WORKSPACE
    smol_b200.clear_error()


def test_weights_refuses():
    a = dict(stream=None, out=P, out_is_bf16=0, q=P, q_is_bf16=0, k_pool=P, v_pool=P, pool_rows=1000, seq_row0=P,
             kv_len=P, n_seqs=2, max_kv_len=50, n_heads=16, n_kv_heads=8, head_dim=128, scale=0.1, window=0,
             softcap=0.0, weights_in=None, weights_out=P, weights_stride=50, workspace=P, workspace_bytes=1 << 40)
    f = smol_b200.lib().smol_b200_decode_attention_weights
    for over in (dict(weights_out=None), dict(weights_stride=49), dict(q=None), dict(head_dim=96), dict(scale=0.0)):
        assert f(*{**a, **over}.values()) == ARGS, over
    assert f(*{**a, "workspace_bytes": 1000}.values()) == WORKSPACE
    assert f(*{**a, "n_seqs": 0}.values()) == 0     # nothing to do
    smol_b200.clear_error()


@pytest.mark.parametrize("n_seqs,hq,hkv,hd", [(1, 16, 8, 128), (1, 8, 1, 256), (3, 12, 12, 64), (200, 16, 8, 128)])
def test_workspaces_never_shrink(n_seqs, hq, hkv, hd):
    prev = 0
    for n in sorted(set(range(0, 20001, 37)) | {9409, 9472, 9600, 65536}):
        size = smol_b200.decode_weights_workspace_bytes(n_seqs, n, hq, hkv, hd)
        assert size >= prev
        prev = size
    prev = 0
    for n in sorted(set(range(0, 20001, 37)) | {9409, 9472, 65536}):
        size = smol_b200.decode_shared_workspace_bytes(n_seqs, 100, 1, n, n_seqs, hq, hkv, hd)
        assert size >= prev
        prev = size


def test_sizes_of_refused_shapes_are_zero():
    assert smol_b200.decode_weights_workspace_bytes(1, 10, 16, 8, 72) == 0
    assert smol_b200.decode_shared_workspace_bytes(0, 10, 1, 10, 1, 16, 8, 128) == 0
    assert smol_b200.decode_shared_workspace_bytes(1, 10, 1, 10, 1, 15, 8, 128) == 0


def prompt_args(**over):
    a = dict(stream=None, weights_in=None, weights_out=P, weights_stride=50, q=P, q_row_stride=2048,
             q_batch_stride=2048 * 10, k=P, k_row_stride=1024, k_batch_stride=1024 * 50, batch=2, seq_q=10, seq_k=50,
             n_heads=16, n_kv_heads=8, head_dim=128, scale=0.1, mask_kind=0, q_offset=40, prefix_len=0, window=0,
             softcap=0.0, workspace=P, workspace_bytes=1 << 40)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over", [
    dict(weights_out=None), dict(q=None), dict(k=None), dict(weights_stride=49), dict(q=P + 8), dict(k=P + 2),
    dict(q_row_stride=2044), dict(q_row_stride=1024), dict(k_row_stride=1020), dict(k_row_stride=512),
    dict(q_batch_stride=4), dict(k_batch_stride=1), dict(seq_q=-1), dict(seq_k=-1), dict(n_heads=15),
    dict(n_kv_heads=0), dict(n_heads=129, n_kv_heads=1), dict(head_dim=12), dict(head_dim=264), dict(scale=0.0),
    dict(scale=float("nan")), dict(mask_kind=2), dict(mask_kind=4), dict(mask_kind=-1), dict(batch=65536),
    dict(q_offset=1 << 30), dict(q_offset=-(1 << 30)), dict(seq_q=1 << 30), dict(seq_k=1 << 30),
])
def test_prompt_weights_refuses(over):
    assert smol_b200.lib().smol_b200_prefill_attention_weights(*prompt_args(**over)) == ARGS
    smol_b200.clear_error()


def test_prompt_weights_workspace_and_nothing_to_do():
    f = smol_b200.lib().smol_b200_prefill_attention_weights
    for over in (dict(workspace=None), dict(workspace_bytes=100), dict(workspace=P + 8)):
        assert f(*prompt_args(**over)) == WORKSPACE
    assert f(*prompt_args(batch=0)) == 0 and f(*prompt_args(seq_k=0)) == 0
    assert smol_b200.prefill_weights_workspace_bytes(1, 10, 10, 16, 8, 12) == 0
    assert smol_b200.prefill_weights_workspace_bytes(1, 10, 10, 129, 1, 64) == 0
    smol_b200.clear_error()


def evict_args(**over):
    a = dict(stream=None, k_pool=P, v_pool=P, pool_rows=1000, seq_row0=P, weights_in=P, weights_out=P, positions_in=P,
             positions_out=P, stride=200, kv_len_in=P, kv_len_out=P, seq_pos=P, n_seqs=2, max_kv_len=200, n_kv_heads=8,
             head_dim=128, budget=100, sink=4, recent=32, workspace=P, workspace_bytes=1 << 40)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over", [
    {n: None} for n in ("k_pool", "v_pool", "seq_row0", "weights_in", "weights_out", "positions_in", "positions_out",
                        "kv_len_in", "kv_len_out", "seq_pos")] + [
    dict(k_pool=P + 8), dict(v_pool=P + 2), dict(pool_rows=0), dict(stride=199), dict(n_seqs=65536),
    dict(max_kv_len=-1), dict(max_kv_len=262145, stride=262145), dict(n_kv_heads=0), dict(n_kv_heads=65536),
    dict(head_dim=4), dict(head_dim=264), dict(budget=0), dict(sink=-1), dict(recent=-1), dict(sink=69),
    dict(sink=1 << 30, recent=(1 << 31) - 1)])
def test_evict_refuses(over):
    assert smol_b200.lib().smol_b200_cache_evict(*evict_args(**over)) == ARGS
    smol_b200.clear_error()


def test_evict_workspace_and_nothing_to_do():
    f = smol_b200.lib().smol_b200_cache_evict
    for over in (dict(workspace=None), dict(workspace_bytes=100), dict(workspace=P + 8)):
        assert f(*evict_args(**over)) == WORKSPACE
    assert f(*evict_args(n_seqs=0)) == 0
    prev = 0
    for n in range(0, 3000, 7):
        size = smol_b200.cache_evict_workspace_bytes(2, n, 8)
        assert size >= prev
        prev = size
    smol_b200.clear_error()


class Recorder:
    """Stands in for the library: keeps the arguments of the last call."""

    def __getattr__(self, name):
        def call(*args):
            self.last = (name, args)
            return 0
        return call


def test_binding_passes_each_argument_to_its_parameter(monkeypatch):
    import re
    text = re.sub(r"/\*.*?\*/", "", open(smol_b200.HEADER_PATH).read(), flags=re.S)
    params = {name: [re.findall(r"\w+", a)[-1] for a in args.split(",")] for name, args in
              re.findall(r"SMOL_B200_API\s+[\w\s\*]+?\b(\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S)}
    import torch
    rec = Recorder()
    monkeypatch.setattr(smol_b200, "_lib", rec)
    t = {n: torch.zeros(8) for n in "out q k_pool v_pool prefix_row0 prefix_len prefix_seq0 seq_row0 kv_len weights_in "
         "weights_out positions_in positions_out kv_len_in kv_len_out seq_pos k".split()}
    t["out"] = torch.zeros(8, dtype=torch.bfloat16)
    ws = torch.zeros(40, dtype=torch.uint8)

    def match(name, expect):
        got, args = rec.last
        assert got == name and len(args) == len(params[name])
        bound = dict(zip(params[name], args))
        for key, want in expect.items():
            assert bound[key] == (want.data_ptr() if isinstance(want, torch.Tensor) else want), key
        assert bound["workspace"] == ws.data_ptr() and bound["workspace_bytes"] == 40 and bound["stream"] is None

    common = dict(pool_rows=11, n_seqs=3, max_kv_len=12, n_heads=16, n_kv_heads=8, head_dim=128, scale=0.5, window=13,
                  softcap=14.0, weights_stride=15)
    flags = dict(out_is_bf16=1, q_is_bf16=0)
    sel = lambda *names: {n: t[n] for n in names}  # noqa: E731
    smol_b200.decode_attention_shared(t["out"], t["q"], t["k_pool"], t["v_pool"], 11, t["prefix_row0"], t["prefix_len"],
                                      t["prefix_seq0"], 2, 21, 22, t["seq_row0"], t["kv_len"], 3, 12, 16, 8, 128, 0.5, ws,
                                      window=13, softcap=14.0, weights_in=t["weights_in"], weights_out=t["weights_out"],
                                      weights_stride=15)
    match("smol_b200_decode_attention_shared",
          {**common, **flags, "n_prefixes": 2, "max_prefix_len": 21, "max_prefix_seqs": 22,
           **sel("out", "q", "k_pool", "v_pool", "prefix_row0", "prefix_len", "prefix_seq0", "seq_row0", "kv_len",
                 "weights_in", "weights_out")})
    smol_b200.decode_attention_weights(t["out"], t["q"], t["k_pool"], t["v_pool"], 11, t["seq_row0"], t["kv_len"], 3, 12,
                                       16, 8, 128, 0.5, t["weights_in"], t["weights_out"], 15, ws, window=13, softcap=14.0)
    match("smol_b200_decode_attention_weights",
          {**common, **flags, **sel("out", "q", "k_pool", "v_pool", "seq_row0", "kv_len", "weights_in", "weights_out")})
    smol_b200.prefill_attention_weights(t["weights_in"], t["weights_out"], 15, t["q"], t["k"], 4, 5, 6, 16, 8, 128, 0.5, ws,
                                        mask_kind=1, q_offset=7, prefix_len=9, window=13, softcap=14.0,
                                        strides=((31, 32), (33, 34)))
    match("smol_b200_prefill_attention_weights",
          dict(weights_stride=15, q_row_stride=31, q_batch_stride=32, k_row_stride=33, k_batch_stride=34, batch=4, seq_q=5,
               seq_k=6, n_heads=16, n_kv_heads=8, head_dim=128, scale=0.5, mask_kind=1, q_offset=7, prefix_len=9, window=13,
               softcap=14.0, **sel("weights_in", "weights_out", "q", "k")))
    smol_b200.cache_evict(t["k_pool"], t["v_pool"], 11, t["seq_row0"], t["weights_in"], t["weights_out"],
                          t["positions_in"], t["positions_out"], 15, t["kv_len_in"], t["kv_len_out"], t["seq_pos"], 3, 12,
                          8, 128, 41, 42, 43, ws)
    match("smol_b200_cache_evict",
          dict(pool_rows=11, stride=15, n_seqs=3, max_kv_len=12, n_kv_heads=8, head_dim=128, budget=41, sink=42, recent=43,
               **sel("k_pool", "v_pool", "seq_row0", "weights_in", "weights_out", "positions_in", "positions_out",
                     "kv_len_in", "kv_len_out", "seq_pos")))


@pytest.mark.parametrize("over", [dict(max_kv_len=(1 << 29) + 1, weights_stride=1 << 30), dict(max_prefix_len=(1 << 29) + 1),
                                  dict(max_prefix_len=(1 << 31) - 1)])
def test_shared_refuses_lengths(over):
    assert smol_b200.lib().smol_b200_decode_attention_shared(*shared_args(**over)) == ARGS
    smol_b200.clear_error()


@pytest.mark.parametrize("n_prefixes,most,hq,hkv", [(1, 1, 16, 8), (1, 8, 16, 8), (1, 9, 16, 8), (40, 2, 8, 1), (40, 3, 8, 1)])
def test_shared_workspaces_never_shrink(n_prefixes, most, hq, hkv):
    prev = 0
    for n in sorted(set(range(0, 20001, 37)) | {1023, 1024, 1025, 9409, 9472, 65536, 500000}):
        size = smol_b200.decode_shared_workspace_bytes(n_prefixes * most, 100, n_prefixes, n, most, hq, hkv, 128)
        assert size >= prev
        prev = size


@pytest.mark.parametrize("which", ["out", "q"])
@pytest.mark.parametrize("dtype", ["float16", "float64", "int32", "uint8"])
@pytest.mark.parametrize("call", ["shared", "weights"])
def test_binding_refuses_types_of_queries_and_outputs(monkeypatch, which, dtype, call):
    import torch
    rec = Recorder()
    monkeypatch.setattr(smol_b200, "_lib", rec)
    t = dict(out=torch.zeros(8), q=torch.zeros(8, dtype=torch.bfloat16))
    ws = torch.zeros(40, dtype=torch.uint8)

    def run():
        if call == "shared":
            smol_b200.decode_attention_shared(t["out"], t["q"], P, P, 11, P, P, P, 2, 21, 22, P, P, 3, 12, 16, 8, 128, 0.5,
                                              ws)
        else:
            smol_b200.decode_attention_weights(t["out"], t["q"], P, P, 11, P, P, 3, 12, 16, 8, 128, 0.5, None, P, 15, ws)

    run()
    assert rec.last[1][2] == 0 and rec.last[1][4] == 1      # out fp32, q bf16
    del rec.last
    t[which] = t[which].to(getattr(torch, dtype))
    with pytest.raises(TypeError, match=which):
        run()
    assert "last" not in vars(rec)      # the library was not called


def test_binding_takes_raw_addresses(monkeypatch):
    import numpy as np
    import torch
    rec = Recorder()
    monkeypatch.setattr(smol_b200, "_lib", rec)
    ws = torch.zeros(40, dtype=torch.uint8)
    smol_b200.prefill_attention_weights(None, P, 15, P + 16, P + 32, 4, 5, 6, 16, 8, 128, 0.5, ws)
    name, args = rec.last
    assert name == "smol_b200_prefill_attention_weights" and (args[1], args[2], args[4], args[7]) == (None, P, P + 16, P + 32)
    smol_b200.cache_evict(P, P + 16, 11, P, P, P, P, P, 15, P, P, P, 3, 12, 8, 128, 41, 42, 43, ws)
    assert rec.last[1][1] == P and rec.last[1][2] == P + 16
    with pytest.raises(AttributeError):     # a host array is no device address
        smol_b200.cache_evict(np.zeros(4), P, 11, P, P, P, P, P, 15, P, P, P, 3, 12, 8, 128, 41, 42, 43, ws)
