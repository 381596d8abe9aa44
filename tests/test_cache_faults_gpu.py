"""Cases of Part 6 (smol_b200.h) in which timing, special values or the order of launches
decide: repeated many times, beside other work, captured, on two streams.

Comparisons are with the 64-bit forms and derived bounds of test_cache_shared_gpu.py and
test_cache_evict_gpu.py, or bit for bit with another run of the same call.
"""

import pytest
import torch

import smol_b200
from test_cache_shared_gpu import Case, no_error

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
