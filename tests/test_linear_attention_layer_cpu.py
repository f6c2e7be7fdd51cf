"""Host-side checks of the linear-attention layer (no GPU)."""
import pytest
import torch

from sorernn_b200.layer import LinearAttention

ARGS = dict(d_model=64, qk_heads=1, v_heads=2, head_dim=32, max_positions=16)


def constants(layer):
    return layer.log_decay, layer.table


@pytest.mark.parametrize("wrapped", [False, True])
@pytest.mark.parametrize("dtype", [None, torch.bfloat16])
@pytest.mark.parametrize("start", ["meta", "cpu"])
def test_constants_survive_to_empty(start, dtype, wrapped):
    """Built on the meta device, given memory and loaded from a checkpoint, which does not hold the constants; and
    emptied in place."""
    want = LinearAttention(**ARGS)
    with torch.device(start):
        layer = LinearAttention(**ARGS)
    model = torch.nn.Sequential(layer) if wrapped else layer
    if dtype is not None:
        model.to(dtype)
    model.to_empty(device="cpu")
    layer.load_state_dict(want.state_dict(), strict=True)
    for a, b in zip(constants(layer), constants(want)):
        assert a.dtype == torch.float32 and a.device.type == "cpu" and torch.equal(a, b)
    assert [n for n, _ in layer.named_buffers()] == ["log_decay", "table"] and "table" not in layer.state_dict()


def test_constants_through_casts_and_moves():
    layer = LinearAttention(**ARGS, log_decay=[-1.0, -0.25])
    want = [t.clone() for t in constants(layer)]
    table = layer.table
    layer.to("cpu")
    assert layer.table is table  # nothing to move
    for move in (lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to("meta"), lambda m: m.to_empty(device="cpu")):
        move(layer)
        assert layer.table.dtype == layer.log_decay.dtype == torch.float32
        if not layer.table.is_meta:
            assert all(torch.equal(a, b) for a, b in zip(constants(layer), want))


def test_documents_past_the_table_are_refused():
    """16 positions: longer documents are refused before any kernel; shorter ones of a longer window, lengths that only
    the device knows, and given positions go on (to the ops, which take no CPU tensors)."""
    layer = LinearAttention(**ARGS)
    x = torch.randn(1, 20, 64)
    cu = torch.tensor([0, 3, 20])
    with pytest.raises(ValueError, match="max_positions = 16"):
        layer(x)
    with pytest.raises(ValueError, match="document of 17 tokens"):
        layer(x, cu_seqlens=cu, cu_seqlens_cpu=cu)
    short = torch.tensor([0, 4, 20])
    for kw in (dict(cu_seqlens=short, cu_seqlens_cpu=short), dict(cu_seqlens=cu),
               dict(positions=torch.zeros(1, 20, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            layer(x, **kw)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer(x[:, :16])


def test_a_table_that_wants_gradients_is_refused(monkeypatch):
    """The rotation gives its table no gradient; under no_grad there is none to lose."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from sorernn_b200 import _lib, qk_norm_rope

    def called():
        raise AssertionError("the library")

    monkeypatch.setattr(_lib, "lib", called)
    with FakeTensorMode():
        q, w = torch.empty(1, 8, 2, 64, device="cuda"), torch.empty(64, device="cuda")
        table = torch.empty(9, 32, device="cuda", requires_grad=True)
        pos = torch.empty(1, 8, dtype=torch.int64, device="cuda")
        with pytest.raises(ValueError, match="table takes no gradient"):
            qk_norm_rope(q, q, w, w, table, pos)
        with torch.no_grad(), pytest.raises(Exception) as e:
            qk_norm_rope(q, q, w, w, table, pos)
        assert "no gradient" not in str(e.value)
