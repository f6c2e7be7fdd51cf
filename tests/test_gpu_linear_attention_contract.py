"""GPU checks of what linear attention and the norm with rotation promise their callers, apart from the numbers."""
import ctypes

import pytest
import torch

from test_gpu_linear_attention import decays, inputs

pytestmark = pytest.mark.gpu


def error_word():
    from sorernn_b200 import _lib

    err = ctypes.c_int32(-1)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.lib().gdn_stream_kernels_error(stream, ctypes.byref(err)), "gdn_stream_kernels_error")
    return err.value


@pytest.mark.parametrize("K,V", [(128, 128), (64, 128), (64, 64)])
@pytest.mark.parametrize("B,T,cu", [(20, 300, None), (1, 2500, None), (1, 3000, [0, 7, 2100, 2100, 3000]), (2, 1, None)])
def test_no_wait_runs_out(K, V, B, T, cu):
    """bf16, forward and backward, whole and cut: no bounded wait of the tensor-memory kernel gives up."""
    from sorernn_b200 import chunk_linear_attention

    assert error_word() == 0
    N = B if cu is None else len(cu) - 1
    x = inputs(B, T, 2, 4, K, V, torch.bfloat16, N, state=True)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "h0")]
    o, ht = chunk_linear_attention(x["q"], x["k"], x["v"], decays(4), initial_state=x["h0"], output_final_state=True,
                                   cu_seqlens=None if cu is None else torch.tensor(cu, device="cuda"))
    torch.autograd.grad((o, ht), leaves, (x["do"], x["dht"]))
    assert error_word() == 0
