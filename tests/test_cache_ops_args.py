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
