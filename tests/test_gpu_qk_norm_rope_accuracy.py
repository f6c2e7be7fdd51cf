"""Accuracy of the norm with rotation in 16 bits beyond the outputs' own rounding, against 64 bits.

The arithmetic is fp32 with one rounding at the end: about eight operations of 2^-24 each on a value's path, the norm's sum
included, on values of up to five RMS times weights of up to 1.8: 8 x 2^-24 x 9 = 4e-6 of RMS; 1e-5. Gradients subtract the
mean of products of as many features again: 2e-5. Measured is what is left beyond half a unit in the last place of the type,
as in test_gpu_linear_attention_accuracy.py."""
import pytest
import torch

from test_gpu_linear_attention_accuracy import within

pytestmark = pytest.mark.gpu


def reference(x, w, cos, sin, eps):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = cos.shape[-1]
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,R", [(128, 32), (128, 128), (64, 64), (256, 128), (100, 20), (128, 36)])
def test_beyond_rounding(dtype, D, R):
    from sorernn_b200 import qk_norm_rope, rotary_table

    g = torch.Generator(device="cuda").manual_seed(D + R)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    B, T, HQ, HK = 2, 301, 4, 2
    q, k = r(B, T, HQ, D).to(dtype), r(B, T, HK, D).to(dtype)
    wq, wk = 1 + 0.2 * r(D), 1 + 0.2 * r(D)
    table = rotary_table(T, R, device="cuda")
    pos = torch.arange(T, device="cuda").expand(B, T)
    leaves = [t.requires_grad_(True) for t in (q, k)]
    out = qk_norm_rope(q, k, wq, wk, table, pos)
    cots = [r(*t.shape).to(dtype) for t in out]
    grads = torch.autograd.grad(out, leaves, cots)
    cos, sin = (t.double()[pos][:, :, None] for t in (table[:, :R // 2], table[:, R // 2:]))
    x64 = [t.detach().double().requires_grad_(True) for t in (q, k)]
    ref = [reference(x, w.double(), cos, sin, 1e-6) for x, w in zip(x64, (wq, wk))]
    want = torch.autograd.grad(ref, x64, [c.double() for c in cots])
    for n, y, z in zip("qk", out, ref):
        within("rope 16-bit " + n, y, z.detach(), 1e-5)
    for n, y, z in zip("qk", grads, want):
        within("rope 16-bit d" + n, y, z, 2e-5)
