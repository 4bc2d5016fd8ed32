"""Four-bit attention of scores of any size: a softmax depends on their differences alone, however large they are or the scale makes them; a row all
of whose keys have scores of minus infinity has none and is NaN, as one with a score of plus infinity or NaN is; a row that sees no key is zeros."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,rows", [(4, 4, 64, 1), (8, 1, 128, 1), (8, 2, 32, 9), (6, 2, 96, 40), (32, 32, 64, 130), (4, 2, 256, 40)])
@pytest.mark.parametrize("keys,longest", [(1, 1), (64, 64), (70, 70), (64, 40000), (2000, 2000)])
@pytest.mark.parametrize("scale", [0.125, 8.0, 1e20])
def test_scores_of_any_size(H, G, D, rows, dtype, keys, longest, scale):
    """Scores are +-q: of a head of the last group + at key 0, - everywhere else; v is 1 to 4, which four bits hold.  The bound: the result is rounded
    once, a probability is off by 2^-16 (twice that of v), 2,000 keys are added in 32 bits (2 * 2,000 * 2^-23 of 4), exp2 is off by 2^-22."""
    from glassbox_amd import ops
    page, pages = 16, -(-keys // 16) + 1
    k, v = torch.zeros(keys, G, D), torch.arange(keys)[:, None, None].remainder(4).add(1).float().expand(keys, G, D)
    k[:, :, 3:5] = -1
    k[0, -1, 3:5] = 1
    kp, vp = torch.zeros(2, *ops.fp4_pages_shape(pages, G, page, D), dtype=torch.uint8, device=DEV)
    ops.fp4_store(torch.cat([k.flatten(1), v.flatten(1)], 1).to(DEV), None, None, torch.arange(keys, dtype=torch.int32, device=DEV), kp, vp, 0, G, D)
    q = torch.zeros(rows, H, D)
    kind = (torch.arange(rows)[:, None] + torch.arange(H)) % 6
    q[..., 3] = torch.tensor([3e38, 3e38, 1e30, 2.0, math.inf, 3e9])[kind]
    q[..., 4] = torch.tensor([3e38, 0.0, 0.0, 0.0, 0.0, 0.0])[kind]      # (whose sum with the other passes 32 bits)
    q = q.to(dtype)
    sign = torch.where((torch.arange(H) // (H // G) == G - 1)[:, None] & (torch.arange(keys) == 0), 1.0, -1.0)
    score = (q[..., 3].float() + q[..., 4].float())[..., None] * sign
    score = torch.where((kind == 4)[..., None], math.nan, score)         # (infinity times the zeros of the other channels)
    want = (torch.softmax(score.double() * scale, -1) * v[:, 0, 0].double()).sum(-1)
    lost = want.isnan()
    assert torch.equal(lost, (kind == 0) | (kind == 4))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None].expand(rows, pages).contiguous()
    # requests of one row each; and rows of one request whose later rows see the same keys, since its table ends there
    calls = [(ints(list(range(rows))), ints([1] * rows), ints([keys - 1] * rows), table, 1, rows)]
    if keys % page == 0:
        calls.append((ints([0]), ints([rows]), ints([keys - 1]), table[:1, :keys // page].contiguous(), rows, 1))
    for q_start, q_len, pos0, tables, most, seqs in calls:
        floats = ops.fp4_attention_floats(seqs, H, G, D, most, longest, 0, dtype)
        out = torch.full((rows, H * D), 9.0, dtype=dtype, device=DEV)
        ops.fp4_attention(q.flatten(1).to(DEV), out, q_start, q_len, pos0, tables, kp, vp, H, scale, most, longest,
                          workspace=torch.empty(floats, device=DEV) if floats else None)
        got = out.cpu().double().view(rows, H, D)
        assert torch.equal(got.isnan(), lost[..., None].expand_as(got)), (most, got[0, :, 0], want[0])
        bound = (torch.finfo(dtype).eps / 2 * want.abs() + 4 * (2 * 2 ** -16 + 2 * keys * 2 ** -23 + 2 ** -21))[..., None].expand_as(got)
        assert ((got - want[..., None])[~lost[..., None].expand_as(got)].abs() <= bound[~lost[..., None].expand_as(got)]).all(), most


def test_rows_that_see_no_key_are_zeros_whatever_their_queries():
    from glassbox_amd import ops
    kp = torch.zeros(ops.fp4_pages_shape(2, 2, 16, 64), dtype=torch.uint8, device=DEV)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for rows in (1, 40):
        q = torch.full((rows, 4 * 64), -math.inf, device=DEV)
        q[:, 1] = math.nan
        out = torch.full_like(q, 5.0)
        ops.fp4_attention(q, out, ints([0]), ints([rows]), ints([-rows]), ints([[0, 1]]), kp, kp.clone(), 4, 0.125, rows, 64)
        assert (out == 0).all()
        ops.fp4_attention(q, out.fill_(5.0), ints([0]), ints([rows]), ints([0]), ints([[-1, 7]]), kp, kp.clone(), 4, 0.125, rows, 64)
        assert (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,rows", [(4, 4, 64, 1), (8, 1, 128, 1), (8, 2, 32, 40), (32, 32, 64, 130), (32, 8, 128, 200), (4, 2, 256, 40)])
@pytest.mark.parametrize("step,scale", [(2.0 ** -10, 1e3), (2.0 ** -20, 1e6), (2.0 ** -23, 1e7)])
@pytest.mark.parametrize("longest", [256, 20000])
def test_differences_that_are_small_beside_the_scores(H, G, D, rows, dtype, step, scale, longest):
    """Scores of 1 and, every other run of 64 keys, 1 + step, exactly; their difference, scaled, is about 1, the scores themselves 10^3 to 10^7: what
    a tile's maximum loses by a rounding, the next tile's does not.  The bound is that of the test above; the scaled difference is off by 2^-23
    of itself, at most 2."""
    from glassbox_amd import ops
    keys, page = 256, 16
    k, v = torch.zeros(keys, G, D), torch.zeros(keys, G, D)
    upper = torch.arange(keys) // 64 % 2 == 1
    k[..., 3] = 1
    k[upper, :, 4] = 1
    v[...], v[upper] = 1, 3
    kp, vp = torch.zeros(2, *ops.fp4_pages_shape(keys // page, G, page, D), dtype=torch.uint8, device=DEV)
    ops.fp4_store(torch.cat([k.flatten(1), v.flatten(1)], 1).to(DEV), None, None, torch.arange(keys, dtype=torch.int32, device=DEV), kp, vp, 0, G, D)
    q = torch.zeros(rows, H, D)
    q[..., 3], q[..., 4] = 1, step
    table = torch.arange(keys // page, dtype=torch.int32, device=DEV)[None]
    ints = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)
    floats = ops.fp4_attention_floats(1, H, G, D, rows, longest, 0, dtype)
    out = torch.empty(rows, H * D, dtype=dtype, device=DEV)
    ops.fp4_attention(q.to(dtype).flatten(1).to(DEV), out, ints(0), ints(rows), ints(keys - 1), table, kp, vp, H, scale, rows, longest,
                      workspace=torch.empty(floats, device=DEV) if floats else None)
    weight = math.exp(step * scale)
    want = (1 + 3 * weight) / (1 + weight)
    bound = torch.finfo(dtype).eps / 2 * want + 3 * (2 * 2 ** -16 + 2 * keys * 2 ** -23 + 2 ** -21)
    assert (out.double() - want).abs().max().item() <= bound
