"""Products with four-bit weights that divide k: halves of a gate / up stack that begin anywhere, and the passes that add the slices, captured,
replayed and on two streams at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -23


def operands(M, N, K, dtype, seed):
    """a, w, and in 64 bits the products and the sums of their sizes"""
    from glassbox_amd import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = ops.fp4_quantize(torch.randn(N, K, generator=g, device=DEV) * 0.05)
    values = torch.empty(N, K, device=DEV)
    ops.fp4_expand(w, values)
    a = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    return a, w, a.double() @ values.double().t(), a.double().abs() @ values.double().abs().t()


@pytest.mark.parametrize("M,N,K,dtype", [(9, 4100, 4128, torch.bfloat16), (12, 2052, 8224, torch.bfloat16), (16, 5004, 8192, torch.float32),
                                         (33, 4100, 4128, torch.bfloat16), (65, 2052, 8224, torch.bfloat16), (33, 2052, 4128, torch.float32)])
def test_a_half_that_does_not_begin_at_a_word_of_four(M, N, K, dtype):
    """N / 2 is 2 more than a multiple of 4: the up half's sums begin between the 16-byte words of a slice.  A sum of K terms in 32 bits is off by
    (3 K + 16) 2^-23 of their sizes (three terms a 32-bit number); SiLU(g) u by what that makes of its factors, 8 steps and its rounding."""
    from glassbox_amd import ops
    a, w, y, size = operands(M, N, K, dtype, 3)
    floats = ops.fp4_gemm_floats(M, N, K, dtype, dtype, True)
    assert N % 8 == 4 and floats > 0
    space = torch.full((floats + 64,), 7.0, device=DEV)
    out = torch.empty(M, N // 2, dtype=dtype, device=DEV)
    ops.fp4_gemm(a, w, out, silu_mul=True, workspace=space[:floats])
    assert (space[floats:] == 7).all()
    off = (3 * K + 16) * STEP * size
    g, u, dg, du = y[:, :N // 2], y[:, N // 2:], off[:, :N // 2], off[:, N // 2:]
    want = g * torch.sigmoid(g) * u
    bound = 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + 8 * STEP * (g * u).abs() + torch.finfo(dtype).eps / 2 * 1.01 * want.abs()
    assert ((out.double() - want).abs() <= bound).all()
