"""Four-bit attention of bfloat16 rows whose sums cancel: what a result then loses it loses where its probabilities are rounded."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("H,G,D,rows,before,window", [
    (4, 4, 64, 1, 39, 0), (8, 1, 128, 1, 47, 0), (2, 1, 256, 1, 30, 0),              # waves share out the keys
    (32, 8, 128, 16, 0, 0), (6, 2, 96, 40, 0, 0), (4, 2, 32, 40, 0, 0),              # waves of columns
    (32, 32, 64, 300, 200, 24), (32, 8, 128, 600, 0, 24), (8, 4, 256, 64, 9, 24)])
def test_probabilities_of_bfloat16_rows_are_held_in_more_than_bfloat16(H, G, D, rows, before, window):
    """Values of one size and any sign: a sum of p v is far below the sum of p |v|.  The bound: the result is rounded once (2^-8 of itself); a
    probability is off by 2^-16, which numerator and denominator share (at most twice that of the sum of p |v|); n keys are added in 32 bits
    (2 n 2^-23); a score, a sum of D exact products, is off by D 2^-23 of the sum of their sizes, and the maximum, the scale and exp2 by
    2^-21 together, which count twice.  (Probabilities of 8 bits are off by up to 2^-8 each.)"""
    from glassbox_amd import ops
    g = torch.Generator().manual_seed(7)
    T, page = before + rows, 16
    pages = -(-T // page) + 1
    kv = torch.cat([torch.randn(T, G * D, generator=g) * 0.3, torch.randint(0, 2, (T, G * D), generator=g) * 2.0 - 1.0], 1).to(DEV)
    table = torch.randperm(pages, generator=g)[:-(-T // page)].int()
    place = torch.arange(T)
    slots = (table[place // page] * page + place % page).int().to(DEV)
    kp, vp = torch.zeros(2, *ops.fp4_pages_shape(pages, G, page, D), dtype=torch.uint8, device=DEV)
    ops.fp4_store(kv, None, None, slots, kp, vp, 0, G, D)
    k, v = torch.empty(2, T, G * D, device=DEV)
    ops.fp4_load(slots, kp, vp, k, v)
    k, v = (x.double().view(T, G, D).transpose(0, 1) for x in (k, v))
    q = (torch.randn(rows, H * D, generator=g) * 0.3).bfloat16().to(DEV)
    scale = 1 / math.sqrt(D)
    ints = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)
    floats = ops.fp4_attention_floats(1, H, G, D, rows, T, window)
    out = torch.empty_like(q)
    ops.fp4_attention(q, out, ints(0), ints(rows), ints(before), table[None].to(DEV), kp, vp, H, scale, rows, T, window=window,
                      workspace=torch.empty(floats, device=DEV) if floats else None)
    qs = q.double().view(rows, G, H // G, D).permute(1, 2, 0, 3)
    position, key = before + torch.arange(rows, device=DEV)[:, None], torch.arange(T, device=DEV)
    gone = (key > position) | (key <= position - (window or T))
    p = (qs @ k[:, None].transpose(-1, -2).contiguous() * scale).masked_fill(gone, -math.inf).softmax(-1)
    want, size = p @ v[:, None], p @ v[:, None].abs()
    reach = ((qs.abs() @ k[:, None].abs().transpose(-1, -2).contiguous()) * scale).masked_fill(gone, 0).amax(-1, keepdim=True)
    seen = (~gone).sum(-1)[:, None]
    bound = want.abs() * 2 ** -8 + size * (2 * 2 ** -16 + 2 * seen * 2 ** -23 + 2 * (D * 2 ** -23 * reach + 2 ** -21))
    off = (out.double().view(rows, G, H // G, D).permute(1, 2, 0, 3) - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
