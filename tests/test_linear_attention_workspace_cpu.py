"""Workspace that linear attention asks for (no GPU): packed documents of one piece take none."""
import ctypes

import pytest

from sorernn_b200 import _lib


def sizes(**kw):
    lib = _lib.lib()
    p = _lib.LinearAttnProblem(**{**dict(B=1, H=16, HV=16, DK=128, DV=128, cu_seqlens=16, max_seqlen=0, scale=0.1,
                                         act_dtype=_lib.BF16), **kw})
    return (lib.gdn_linear_attn_fwd_workspace_size(ctypes.byref(p)), lib.gdn_linear_attn_bwd_workspace_size(ctypes.byref(p)))


@pytest.mark.parametrize("dtype,chunk", [("BF16", 128), ("FP32", 32)])
@pytest.mark.parametrize("T", [512, 8191, 65536])
@pytest.mark.parametrize("N", [1, 2, 50, 1000, 20000])
@pytest.mark.parametrize("longest", [0, 40, 3000])  # 0: not known on the host
def test_states_of_packed_documents(dtype, chunk, T, N, longest):
    """A document of n pieces keeps n - 1 states, so however many documents there are, T tokens have T / piece states at
    most, a piece being a chunk or more: with 16 heads of 128 x 128 floats, 1 MiB each (three scans in the backward)."""
    fwd, bwd = sizes(T=T, N=N, max_seqlen=longest, act_dtype=getattr(_lib, dtype))
    assert fwd <= T // chunk << 20 and bwd <= 3 * (T // chunk) << 20


def test_many_documents():
    """65,536 tokens in 1,000 documents, lengths unknown to the host: 1.0 GB and 3.0 GB when each document kept a state."""
    fwd, bwd = sizes(T=65536, N=1000)
    assert fwd < 100e6 and bwd < 300e6
