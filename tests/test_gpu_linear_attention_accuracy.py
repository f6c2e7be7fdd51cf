"""Accuracy of linear attention's 16-bit outputs and gradients beyond their own rounding, against the token-by-token
recurrence in 64 bits.

What is measured is |got - ref| less half a unit in the last place of the output's type at ref (a correctly rounded result
has none left), in units of RMS(ref). Bars, from the arithmetic:
  * the tensor-memory kernel (bf16, head sizes 64 and 128) splits every operand that is not exact in bf16 (in-chunk
    weights, keys times decay, the state) into two terms: 2^-18 of a value is lost, three such operands reach an output,
    each an independent error on every term of a sum whose terms have random signs: sqrt(3) 2^-18 / sqrt(3) = 3.8e-6 of
    the sum's own RMS. An element may be of a head whose RMS is 1.6 times that of all heads, late in a sequence whose RMS
    grows by sqrt(2), and five and a half standard deviations off (a million values): 5e-5; its fp32 sums add as much
    again: 2e-4 with a factor of two to spare.
  * the other kernel (fp16, and bf16 of other head sizes) is good to fp32: FP32_TOL, the bar of fp32 activations, 5e-5. The
    products in one tf32 term would leave 2^-11, ten times that.
"""
import ctypes

import numpy as np
import pytest
import torch

from helpers import CURRENT_TEST, PARITY_LOG, assert_rms_close, rms, to_np
from test_gpu_linear_attention import FP32_TOL, decays, inputs, oracle

pytestmark = pytest.mark.gpu

TC_TOL = 2e-4
DIGITS = {torch.bfloat16: (8, -126), torch.float16: (11, -14)}  # significant bits, least exponent


def excess(got, ref):
    """max(|got - ref| - half an ulp of got's type at ref) / RMS(ref)"""
    r = ref.double().cpu().numpy()
    a = got.detach().double().cpu().numpy()
    assert a.shape == r.shape and np.isfinite(a).all()
    bits, least = DIGITS[got.dtype]
    _, e = np.frexp(r)  # |r| in [2^(e-1), 2^e)
    half = np.exp2(np.maximum(e - 1, least).astype(np.float64) - bits)
    return float((np.abs(a - r) - half).max()) / max(rms(r), 1e-30)


def within(name, got, ref, tol):
    x = excess(got, ref)
    PARITY_LOG.append((name, x, x, tol, CURRENT_TEST[0]))
    assert x <= tol, f"{name}: {x:.3e} of RMS beyond the output's rounding, bar {tol}"


def run(B, T, H, HV, K, V, dtype, decay, tol, cu=None, state=True, seed=0):
    from sorernn_b200 import chunk_linear_attention

    N = B if cu is None else len(cu) - 1
    x = inputs(B, T, H, HV, K, V, dtype, N, state, seed)
    ld = decays(HV, decay)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v")]
    cu_t = None if cu is None else torch.tensor(cu, device="cuda")
    o, ht = chunk_linear_attention(x["q"], x["k"], x["v"], ld, initial_state=x["h0"], output_final_state=True,
                                   cu_seqlens=cu_t, cu_seqlens_cpu=None if cu is None else cu_t.cpu())
    outs, cots = ((o, ht), (x["do"], x["dht"])) if state else ((o,), (x["do"],))
    grads = torch.autograd.grad(outs, leaves, cots)
    ref = oracle(x["q"], x["k"], x["v"], ld, K ** -0.5, cu, x["h0"], x["do"], x["dht"])
    for n, y in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        within("lin 16-bit " + n, y, ref[n], tol)


@pytest.mark.parametrize("K,V", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("decay", ["slopes", "edges"])
def test_tensor_memory_kernel_whole_sequences(K, V, decay):
    """Many pairs, several chunks each: nothing is cut."""
    run(16, 300, 10, 10, K, V, torch.bfloat16, decay, TC_TOL, seed=11)


@pytest.mark.parametrize("K,V", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("T", [1900, 1920])
def test_tensor_memory_kernel_cut_sequences(K, V, T):
    """Pieces side by side, heads that never decay and heads that decay at once: the state enters every output."""
    run(2, T, 5, 5, K, V, torch.bfloat16, "edges", TC_TOL, seed=6)


@pytest.mark.parametrize("known", [True, False])  # the lengths, on the host
@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, TC_TOL), (torch.float32, None)])
@pytest.mark.parametrize("H,HV", [(2, 2), (1, 2)])
def test_packed_documents_cut_into_pieces(H, HV, dtype, tol, known):
    """Documents of many pieces among ones of a single piece and empty ones, with and without states, K = V = 128: the
    backward's three scans of a cut packed window in one launch. States and fp32 outputs to 5e-5 of RMS, as elsewhere."""
    from sorernn_b200 import _lib, chunk_linear_attention

    cu = [0, 0, 1, 2, 130, 1400, 1401, 1401, 1500, 3100, 3101, 3200]
    N, T = len(cu) - 1, cu[-1]
    p = _lib.LinearAttnProblem(1, T, HV, HV, 128, 128, N, 16, 1600 if known else 0, 0.1,
                               _lib.BF16 if dtype == torch.bfloat16 else _lib.FP32)
    assert _lib.lib().gdn_linear_attn_bwd_workspace_size(ctypes.byref(p)) > 0  # cut
    cu_t = torch.tensor(cu, device="cuda")
    for state in (False, True):
        x = inputs(1, T, H, HV, 128, 128, dtype, N, state, 13)
        ld = decays(HV, "-0.01")
        leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v") + (("h0",) if state else ())]
        o, ht = chunk_linear_attention(x["q"], x["k"], x["v"], ld, initial_state=x["h0"], output_final_state=True,
                                       cu_seqlens=cu_t, cu_seqlens_cpu=cu_t.cpu() if known else None)
        grads = torch.autograd.grad((o, ht) if state else (o,), leaves, (x["do"], x["dht"]) if state else (x["do"],))
        ref = oracle(x["q"], x["k"], x["v"], ld, 128 ** -0.5, cu, x["h0"], x["do"], x["dht"])
        for n, y in zip(("o", "dq", "dk", "dv", "dh0", "ht"), (o, *grads, *(() if state else (None,)), ht)):
            if y is None:
                continue
            if y.dtype == torch.float32:
                assert_rms_close(to_np(y), ref[n].cpu().numpy(), FP32_TOL, "lin packed cut " + n)
            else:
                within("lin packed cut " + n, y, ref[n], tol)


@pytest.mark.parametrize("dtype,K,V", [(torch.float16, 128, 128), (torch.float16, 64, 64), (torch.float16, 20, 33),
                                       (torch.bfloat16, 96, 128), (torch.bfloat16, 20, 33), (torch.bfloat16, 128, 7)])
@pytest.mark.parametrize("decay", ["slopes", "edges"])
def test_fp32_kernel(dtype, K, V, decay):
    """Whole (16 sequences) and cut (one long one)."""
    run(16, 100, 5, 10, K, V, dtype, decay, FP32_TOL, seed=14)
    run(1, 1500, 2, 2, K, V, dtype, decay, FP32_TOL, seed=15)
