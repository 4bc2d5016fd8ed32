"""The four-bit operators on neighbouring columns of one tensor: the bits that tensors of their own get."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [0, 3, 8])
def test_columns_of_one_tensor(dtype, gap):
    from glassbox_amd import ops
    H, G, D, n, page = 6, 2, 64, 37, 16
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(n, (H + 2 * G) * D, generator=g).to(dtype).to(DEV)
    angle = torch.randn(n, D // 2, generator=g).to(DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    ints = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)
    table = torch.arange(3, dtype=torch.int32, device=DEV)[None]
    w = ops.fp4_quantize(torch.randn(72, H * D, generator=g).to(DEV))

    def run(place):
        qkv = place("qkv", (H + 2 * G) * D)
        qkv.copy_(rows)
        q, k, v, att, out = place("q", H * D), place("k", G * D), place("v", G * D), place("att", H * D), place("out", 72)
        pages = torch.zeros(2, *ops.fp4_pages_shape(3, G, page, D), dtype=torch.uint8, device=DEV)
        ops.fp4_store(qkv, angle.cos(), angle.sin(), slots, pages[0], pages[1], H, G, D, q=q)
        ops.fp4_load(slots, pages[0], pages[1], k, v)
        ops.fp4_attention(q, att, ints(0), ints(n), ints(0), table, pages[0], pages[1], H, 0.125, n, n)
        ops.fp4_gemm(att, w, out)
        return qkv, q, k, v, att, out

    alone = run(lambda name, cols: torch.full((n, cols), 7.0, dtype=dtype, device=DEV))
    width = sum(t.shape[1] + gap for t in alone)
    one, at = torch.full((n, width), 7.0, dtype=dtype, device=DEV), [0]

    def place(name, cols):
        at[0] += cols + gap
        return one[:, at[0] - cols - gap:at[0] - gap]

    beside = run(place)
    for mine, other in zip(beside, alone):
        assert torch.equal(mine, other)
    first = 0
    for t in alone:      # what lies between the columns is left
        assert (one[:, first + t.shape[1]:first + t.shape[1] + gap] == 7).all()
        first += t.shape[1] + gap
