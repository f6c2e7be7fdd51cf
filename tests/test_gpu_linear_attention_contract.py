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


def off_grid(t):
    """The values of t in contiguous memory that starts one element past a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    assert buf.data_ptr() % 16 == 0
    return buf[1:].copy_(t.flatten()).view(t.shape)


@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 20, 33), (torch.float32, 64, 64), (torch.bfloat16, 128, 128),
                                       (torch.float16, 7, 128)])
def test_memory_off_the_16_byte_grid(dtype, K, V):
    """Inputs, states and gradients of any alignment give what aligned ones do."""
    from sorernn_b200 import chunk_linear_attention

    x = inputs(2, 70, 1, 2, K, V, dtype, state=True, seed=4)
    results = []
    for move in (lambda t: t.clone(), off_grid):
        y = {n: move(t) for n, t in x.items()}
        leaves = [y[n].requires_grad_(True) for n in ("q", "k", "v", "h0")]
        o, ht = chunk_linear_attention(y["q"], y["k"], y["v"], decays(2), initial_state=y["h0"], output_final_state=True)
        results.append([o, ht, *torch.autograd.grad((o, ht), leaves, (y["do"], y["dht"]))])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_gradient_of_a_concatenation():
    """The second part's gradient is a slice of the whole's, at byte 37 x 33 x 4 of its memory."""
    from sorernn_b200 import chunk_linear_attention

    a, b = (inputs(1, T, 1, 1, 20, 33, torch.float32, seed=5) for T in (37, 22))
    leaves = [y[n].requires_grad_(True) for y in (a, b) for n in ("q", "k", "v")]
    parts = [chunk_linear_attention(y["q"], y["k"], y["v"], decays(1))[0] for y in (a, b)]
    got = torch.autograd.grad(torch.cat(parts, 1), leaves, torch.cat([a["do"], b["do"]], 1))
    want = torch.autograd.grad(parts_again(a, b), leaves, (a["do"], b["do"]))
    for u, w in zip(got, want):
        assert torch.equal(u, w)


def parts_again(a, b):
    from sorernn_b200 import chunk_linear_attention

    return [chunk_linear_attention(y["q"], y["k"], y["v"], decays(1))[0] for y in (a, b)]


def test_step_on_a_slice_of_a_pool_of_odd_states():
    """States of 3 x 3 floats: the pool's second one starts at byte 36."""
    from sorernn_b200 import linear_attention_step

    x = inputs(2, 1, 1, 1, 3, 3, torch.float32, state=True, seed=6)
    pool = torch.zeros(3, 1, 3, 3, device="cuda")
    pool[1:] = x["h0"]
    state = x["h0"].clone()
    tokens = [x[n][:, 0] for n in ("q", "k", "v")]
    want = linear_attention_step(*tokens, decays(1), state)
    got = linear_attention_step(*tokens, decays(1), pool[1:])
    assert torch.equal(got, want) and torch.equal(pool[1:], state) and not pool[0].any()


def test_backward_through_a_step_is_an_error():
    """Forward as under no_grad, an ``out`` tensor used twice too; a loss through it says that there is no backward."""
    from sorernn_b200 import linear_attention_step

    x = inputs(2, 1, 1, 2, 64, 64, torch.float32, state=True, seed=7)
    tokens = [x[n][:, 0] for n in ("q", "k", "v")]
    state = x["h0"].clone()
    want = [linear_attention_step(*tokens, decays(2), state) for _ in range(2)]
    for i in range(3):
        got_state, out = x["h0"].clone(), torch.empty_like(want[0])
        leaves = [t.detach().clone().requires_grad_(n == i) for n, t in enumerate(tokens)]
        for w in want:
            o = linear_attention_step(*leaves, decays(2), got_state, out=out)
            assert o is out and torch.equal(o, w)
            with pytest.raises(RuntimeError, match="no backward"):
                o.sum().backward()
        assert torch.equal(got_state, state)
        with torch.no_grad():
            assert not linear_attention_step(*leaves, decays(2), got_state).requires_grad


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode derivative: an input that carries a tangent is refused, others pass within dual_level."""
    import torch.autograd.forward_ad as fw

    from sorernn_b200 import chunk_linear_attention, linear_attention_step, qk_norm_rope, rotary_table

    x = inputs(1, 5, 2, 2, 64, 64, torch.float32, state=True, seed=8)
    w, table, pos = torch.ones(64, device="cuda"), rotary_table(8, 32, device="cuda"), torch.arange(5, device="cuda")[None]
    calls = [(["q", "k", "v", "h0"], lambda q, k, v, h0: chunk_linear_attention(q, k, v, decays(2), initial_state=h0)),
             (["q", "k", "v", "h0"],
              lambda q, k, v, h0: linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decays(2), h0)),
             (["q", "k", "w"], lambda q, k, w: qk_norm_rope(q, k, w, w, table, pos))]
    x["w"] = w
    with fw.dual_level():
        for names, call in calls:
            call(*(x[n].clone() for n in names))
            for m in names:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*(fw.make_dual(x[n].clone(), torch.ones_like(x[n])) if n == m else x[n].clone() for n in names))


def test_a_step_on_a_state_that_autograd_saved_is_noticed():
    """A prefill from a state, then a step on that state in place: the prefill's backward needs the old values."""
    from sorernn_b200 import chunk_linear_attention, linear_attention_step

    x = inputs(1, 5, 1, 1, 64, 64, torch.float32, state=True, seed=9)
    q = x["q"].clone().requires_grad_(True)
    o, _ = chunk_linear_attention(q, x["k"], x["v"], decays(1), initial_state=x["h0"])
    with torch.no_grad():
        linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], decays(1), x["h0"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(x["do"])
    with torch.inference_mode():
        state = x["h0"].clone()
        linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], decays(1), state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cuda_graph_capture(dtype):
    """Forward and backward (a cut sequence), a decode step and the norm with rotation, captured once and replayed on new
    inputs: the same bits as the calls outside."""
    from sorernn_b200 import chunk_linear_attention, linear_attention_step, qk_norm_rope, rotary_table

    T = 1500
    x = inputs(1, T, 2, 4, 128, 128, dtype, state=True, seed=10)
    ld, w = decays(4), torch.ones(128, device="cuda", requires_grad=True)
    table, pos = rotary_table(T, 32, device="cuda"), torch.arange(T, device="cuda")[None]
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "h0")]
    token, state = [x[n].detach()[:, 7].clone() for n in ("q", "k", "v")], x["h0"].detach().clone()

    def work():
        q, k = qk_norm_rope(x["q"], x["k"], w, w, table, pos)
        o, ht = chunk_linear_attention(q, k, x["v"], ld, initial_state=x["h0"], output_final_state=True)
        grads = torch.autograd.grad((o, ht), leaves + [w], (x["do"], x["dht"]))
        with torch.no_grad():
            return [o, ht, *grads, linear_attention_step(*token, ld, state)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    fresh = inputs(1, T, 2, 4, 128, 128, dtype, state=True, seed=11)
    with torch.no_grad():
        for n, t in fresh.items():
            x[n].copy_(t)
        start = torch.randn_like(state)
        state.copy_(start)
        graph.replay()
        got, got_state = [t.clone() for t in out], state.clone()
        state.copy_(start)
    want = work()
    assert torch.equal(got_state, state)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs in one process")
def test_tensors_on_another_device_than_the_current_one():
    from sorernn_b200 import chunk_linear_attention

    x = inputs(1, 300, 2, 2, 128, 128, torch.bfloat16, seed=12)
    ld = decays(2)
    want = chunk_linear_attention(x["q"], x["k"], x["v"], ld, output_final_state=True)
    got = chunk_linear_attention(*(x[n].to("cuda:1") for n in ("q", "k", "v")), ld.to("cuda:1"), output_final_state=True)
    for a, b in zip(want, got):
        assert b.device.index == 1 and torch.equal(a.cpu(), b.cpu())
