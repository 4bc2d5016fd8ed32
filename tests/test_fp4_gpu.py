"""Four-bit pages and matrices on the GPU against plain 64-bit operations (``fp4_plain``): stores, loads, attention, products, and all of them
together.

Tolerances are bounds, not fits.  A stored number is the nearest of its block, equal to the bit.  A sum of n terms in 32 bits is off by at
most n 2^-23 times the sum of their magnitudes (2^-24 a rounding, twice for what a matrix core may cut); a result in bfloat16 by 2^-8 of
itself; bfloat16 probabilities by 2^-8 each; a score that is off by d makes a probability off by a factor e^d and the softmax's result by
at most 2 (e^d - 1) of the sum of p |v|."""
import math

import pytest
import torch

import fp4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -23


def normal(*shape, seed=0, scale=1.0, wide=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g, dtype=torch.float64) * scale
    if wide:
        x = x * torch.where(torch.rand(shape[-1], generator=g) < 0.1, wide, 1.0)
    return x.float()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def blank(pages, G, page, D):
    from glassbox_amd import ops
    return torch.zeros(ops.fp4_pages_shape(pages, G, page, D), dtype=torch.uint8)


# ---------------------------------------------------------------------------------------------------------------- the format
SPECIAL = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.2500001, 0.7499999, 5.0000005, 4.9999995]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (17, 96), (5, 544), (130, 1024)])
def test_quantize_takes_the_nearest_number_and_expand_gives_it_back(rows, cols, dtype):
    from glassbox_amd import ops
    x = normal(rows, cols, seed=1, wide=6.0).to(dtype)
    # ties, both signs, blocks of zeros, tiny and huge blocks, largest magnitudes on both sides of 7 units
    x[0, :len(SPECIAL)] = torch.tensor(SPECIAL).to(dtype)
    if rows > 2:
        x[1, :32] = 0
        x[2, :32] = (x[2, :32].float() * 2.0 ** -130).to(dtype)
        x[2, 32:64] = (x[2, 32:64].float().clamp(-2, 2) * 2.0 ** 126).to(dtype)
        x[0, 32:64] = torch.tensor([-v for v in SPECIAL] + [8.0] * (32 - len(SPECIAL))).to(dtype)
    wide = torch.zeros(rows, cols + 3, dtype=dtype)      # rows that do not begin at 16-byte words
    wide[:, :cols] = x
    codes, scales = plain.quantized(x)
    for given in (x.to(DEV), wide.to(DEV)[:, :cols]):
        m = ops.fp4_quantize(given)
        assert m.shape == (rows, cols)
        assert torch.equal(m.codes.cpu(), (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(-2))
        assert torch.equal(m.scales.cpu()[:, :cols // 32], scales) and not m.scales[:, cols // 32:].any()
        for out in (torch.bfloat16, torch.float32):
            back = torch.empty(rows, cols, dtype=out, device=DEV)
            ops.fp4_expand(m, back)
            assert torch.equal(back.cpu().double(), plain.values(codes, scales))


def test_blocks_that_are_not_finite_read_as_nan_and_no_others():
    from glassbox_amd import ops
    x = normal(4, 128, seed=2)
    x[0, 5], x[1, 40], x[2, 100] = math.inf, -math.inf, math.nan
    m = ops.fp4_quantize(x.to(DEV))
    back = torch.empty(4, 128, device=DEV)
    ops.fp4_expand(m, back)
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(back.cpu().isnan().view(4, 4, 32).all(-1), bad) and torch.equal(back.cpu().isnan().view(4, 4, 32).any(-1), bad)


# -------------------------------------------------------------------------------------------------------------- store and load
STORES = [  # heads, kv heads, head size, page, rows
    (1, 1, 32, 16, 1), (9, 3, 64, 16, 5), (4, 4, 96, 32, 33), (8, 2, 128, 16, 70), (2, 1, 256, 48, 17), (0, 2, 64, 16, 4), (32, 32, 64, 16, 8),
    # many rows: four heads a lane, the last group not full; values in words and, behind slots out of order, in bytes
    (9, 5, 64, 16, 1400), (6, 3, 96, 32, 900), (3, 2, 128, 16, 2000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,page,n", STORES)
@pytest.mark.parametrize("rotate", [True, False])
def test_store_and_load(H, G, D, page, n, dtype, rotate):
    from glassbox_amd import ops
    pages = -(-n // page) + 3
    wide = (H + 2 * G) * D + 5                                       # rows of odd strides
    rows = normal(n, wide, seed=3, wide=5.0).to(dtype)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 37 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    cos, sin = angle.cos().float(), angle.sin().float()
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(pages * page, generator=g)[:n].int()
    if n > 100:                                                      # whole pages in no order, and rows out of order among them
        slots = (torch.randperm(pages, generator=g)[:-(-n // page), None] * page + torch.arange(page)).flatten()[:n].int()
        slots[500:520] = slots[500:520].flip(0)
    if n > 3:
        slots[1], slots[2] = -1, pages * page                        # rows that are not stored
    k0 = torch.randint(0, 256, blank(pages, G, page, D).shape, generator=g, dtype=torch.uint8)
    v0 = torch.randint(0, 256, k0.shape, generator=g, dtype=torch.uint8)
    heads = rows[:, :(H + 2 * G) * D].reshape(n, H + 2 * G, D)
    k32 = plain.turned(heads[:, H:H + G], cos, sin) if rotate else heads[:, H:H + G].float()
    kc, ks = plain.quantized(k32)
    vc, vs = plain.quantized(heads[:, H + G:])
    want_k, want_v = k0.clone(), v0.clone()
    kept_rows = [i for i in range(n) if 0 <= slots[i] < pages * page]
    for i in kept_rows:
        plain.put(want_k, want_v, int(slots[i]), kc[i], ks[i], vc[i], vs[i])
    want_k_rows, want_v_rows = torch.full((2, n, G * D), 9.0, dtype=torch.float64)
    want_k_rows[kept_rows] = plain.values(kc, ks).flatten(1)[kept_rows]
    want_v_rows[kept_rows] = plain.values(vc, vs).flatten(1)[kept_rows]
    q32 = plain.turned(heads[:, :H], cos, sin) if rotate else heads[:, :H].float()
    want_q = q32.to(dtype).reshape(n, H * D)
    angles = (cos.to(DEV), sin.to(DEV)) if rotate else (None, None)
    for place in ("own", "in place", "none stored"):
        qkv = rows.to(DEV)
        kp, vp = k0.to(DEV), v0.to(DEV)
        q = torch.full((n, H * D + 1), 7.0, dtype=dtype, device=DEV)[:, :H * D] if place == "own" else None
        ops.fp4_store(qkv, *angles, slots.to(DEV) if place != "none stored" else None, kp, vp, H, G, D, q=q)
        if place == "none stored":
            assert torch.equal(kp.cpu(), k0) and torch.equal(vp.cpu(), v0)
        else:
            assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)
        got = (qkv[:, :H * D] if q is None else q).cpu()
        assert torch.equal(got, want_q)
        kept = rows[:, H * D:] if q is None else rows
        assert torch.equal((qkv[:, H * D:] if q is None else qkv).cpu(), kept)
        if place == "own":
            k = torch.full((n, G * D + 3), 9.0, dtype=dtype, device=DEV)[:, :G * D]
            v = torch.full((n, G * D), 9.0, dtype=dtype, device=DEV)
            ops.fp4_load(slots.to(DEV), kp, vp, k, v)
            assert torch.equal(k.cpu().double(), want_k_rows) and torch.equal(v.cpu().double(), want_v_rows)


def test_store_without_rows():
    from glassbox_amd import ops
    kp, vp = blank(2, 2, 16, 64).to(DEV), blank(2, 2, 16, 64).to(DEV)
    none = torch.empty(0, 6 * 64, dtype=torch.bfloat16, device=DEV)
    slots = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.fp4_store(none, None, None, slots, kp, vp, 2, 2, 64)
    ops.fp4_load(slots, kp, vp, none[:, :128], none.new_empty(0, 128))
    assert not kp.any() and not vp.any()


# ------------------------------------------------------------------------------------------------------------------ attention
def cached(lengths, G, D, page, seed, spare=2):
    """Pages that hold normal keys and values for requests of these lengths, their tables, all in no order; what no request holds is noise."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-l // page) for l in lengths]
    pages = sum(held) + spare
    kp = torch.randint(0, 256, blank(pages, G, page, D).shape, generator=g, dtype=torch.uint8)
    vp = torch.randint(0, 256, kp.shape, generator=g, dtype=torch.uint8)
    order = torch.randperm(pages, generator=g)
    tables = torch.full((len(lengths), max(held + [1])), -1, dtype=torch.int32)
    at = 0
    for i, (h, l) in enumerate(zip(held, lengths)):
        tables[i, :h] = order[at:at + h]
        at += h
        kc, ks = plain.quantized(torch.randn(l, G, D, generator=g) * torch.where(torch.rand(D, generator=g) < 0.1, 4.0, 1.0))
        vc, vs = plain.quantized(torch.randn(l, G, D, generator=g))
        for t in range(l):
            plain.put(kp, vp, int(tables[i, t // page]) * page + t % page, kc[t], ks[t], vc[t], vs[t])
    return kp, vp, tables


def attend(q, q_start, q_len, pos0, tables, kp, vp, H, scale, window=0, max_context=None, out=None, keep=None):
    from glassbox_amd import ops
    P, G, nb, _, page = kp.shape
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    most = max(q_len)
    longest = max_context or max(1, max(p + l for p, l in zip(pos0, q_len)))
    out = torch.full_like(q, 5.0, device=DEV) if out is None else out
    floats = ops.fp4_attention_floats(len(q_len), H, G, nb * 32, most, longest, window, q.dtype)
    ws = torch.full((floats,), math.nan, device=DEV) if floats else None
    args = [q.to(DEV), out, ints(q_start), ints(q_len), ints(pos0), tables.to(DEV), kp.to(DEV), vp.to(DEV), H, scale, most, longest]
    if keep is not None:
        keep += [args, ws]
    ops.fp4_attention(*args, window=window, workspace=ws)
    return out


def check(got, q, q_start, q_len, pos0, tables, kp, vp, H, scale, window=0):
    D = 32 * kp.shape[2]
    want, size, reach = plain.attention(q, q_start, q_len, pos0, tables, kp, vp, H, scale, window)
    got = got.cpu().double().view(want.shape)
    none = want.isnan()
    keys = max([p + l for p, l in zip(pos0, q_len)] + [1])
    for row in range(q.shape[0]):
        mine = any(s <= row < s + l for s, l in zip(q_start, q_len))
        if not mine:
            assert (got[row] == 5).all(), row
            continue
        assert torch.equal(none[row], got[row].isnan()), row
        off = (3 * D + 8) * STEP * reach[row] + 4 * STEP * reach[row]                    # of a score: its sum, its scaling and the exponent's
        off = 2 * (torch.exp(off) - 1)[:, None] * size[row] + (3 * keys + 80) * STEP * size[row]   # probabilities; sums and joins
        if q.dtype == torch.bfloat16:
            off = off + half_step(q.dtype) * size[row]
        off = off + half_step(q.dtype) * want[row].abs() + 1e-30
        bad = ((got[row] - want[row]).abs() > off) & ~none[row]
        assert not bad.any(), (row, (got[row] - want[row]).abs()[bad].max(), off[bad].max())


ATTENDS = [  # heads, kv heads, head size, page, rows of each request, tokens before them, window
    (1, 1, 32, 16, [1], [0], 0),
    (3, 1, 64, 16, [1], [300], 0),
    (9, 3, 64, 16, [1, 1, 1], [0, 63, 64], 0),
    (8, 2, 128, 32, [1, 1], [15, 700], 0),
    (24, 1, 64, 16, [1, 1], [5, 129], 0),                # more heads than one tile of columns
    (4, 4, 96, 48, [1, 1], [47, 200], 0),
    (2, 1, 256, 16, [1, 2], [90, 300], 0),
    (2, 2, 64, 16, [1], [2600], 0),                      # a context in runs
    (2, 1, 128, 16, [1, 1], [1500, 3], 40),              # a window that ends inside tiles and pages
    (6, 2, 64, 16, [3, 0, 1, 20], [0, 7, 65, 100], 0),   # portions of all lengths, none among them
    (4, 1, 128, 16, [70], [33], 0),
    (5, 5, 32, 64, [130, 40], [0, 300], 17),
    (15, 5, 64, 16, [33], [0], 0),
    (2, 2, 96, 16, [40], [10], 100),
    (2, 1, 256, 16, [50], [40], 0),
    (16, 16, 64, 16, [40, 0, 33], [960, 0, 100], 0),     # three tiles of columns a wave, of which some rows fill one and a half
    (16, 16, 64, 32, [131, 5, 17], [1400, 20, 0], 1100),
    (32, 32, 32, 16, [40], [1963], 0),
    (24, 8, 32, 48, [90, 7], [1905, 0], 0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,page,rows,before,window", ATTENDS)
def test_attention(H, G, D, page, rows, before, window, dtype):
    lengths = [r + b if r else 0 for r, b in zip(rows, before)]
    kp, vp, tables = cached(lengths, G, D, page, seed=7)
    n = sum(rows) + 2                                    # two rows of no request, before and behind the others
    q = normal(n, H * D, seed=8, scale=1.3).to(dtype)
    start, at = [], 1
    for r in rows:
        start.append(at)
        at += r
    args = (q, start, rows, before, tables, kp, vp, H, 1 / math.sqrt(D), window)
    check(attend(*args), *args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 90])
def test_attention_rows_that_see_nothing_give_zeros(rows, dtype):
    """Positions below 0, tables of pages that are none of the pool's, tables that end before the row's position."""
    kp, vp, tables = cached([100, 100, 100], 1, 64, 16, seed=9)
    tables[1] = torch.tensor([-1, kp.shape[0], -5, 1 << 30, -1, -1, 99999][:tables.shape[1]], dtype=torch.int32)
    tables[2, 3] = 12345                                 # a hole: its keys are not seen
    q = normal(3 * rows, 2 * 64, seed=10).to(dtype)
    pos0 = [-rows // 2 if rows > 1 else -3, 40, 95 if rows == 1 else 10]
    args = (q, [0, rows, 2 * rows], [rows] * 3, pos0, tables, kp, vp, 2, 0.125)
    got = attend(*args)
    check(got, *args)
    assert (got[rows:2 * rows] == 0).all() and (got[0] == 0).all()
    # positions behind the end of the table
    args = (q[:rows], [0], [rows], [100], tables[:1, :4], kp, vp, 2, 0.125)
    check(attend(*args), *args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_leaves_what_is_masked_alone(rows, dtype):
    """Keys and values that are not finite behind the row's position, before its window or in the rest of its last page change nothing;
    seen ones make their rows NaN, values only the block's channels."""
    D, window = 128, 64
    kp, vp, tables = cached([200], 1, D, 16, seed=11)
    pos0 = 140 - rows
    q = normal(rows, 2 * D, seed=12).to(dtype)
    args = (q, [0], [rows], [pos0], tables, kp, vp, 2, 0.1, window)
    clean = attend(*args)
    check(clean, *args)
    bad_k, bad_v = kp.clone(), vp.clone()
    for t in list(range(0, pos0 - window + 1)) + list(range(pos0 + rows, 200)):
        pg, off = int(tables[0, t // 16]), t % 16
        bad_k.view(kp.shape[0], 1, 4, 17 * 16)[pg, :, :, 16 * 16 + plain.key_place(off)] = 255
        bad_v[pg, :, :, 16, off] = 255
    args = (q, [0], [rows], [pos0], tables, bad_k, bad_v, 2, 0.1, window)
    assert torch.equal(attend(*args), clean)
    # one that the last rows alone see, in one block of the values
    t = pos0 + rows - 1
    bad_v[int(tables[0, t // 16]), 0, 2, 16, t % 16] = 255
    got = attend(*args).view(rows, 2, D).cpu()
    assert got[-1, :, 64:96].isnan().all() and torch.equal(got[-1, :, :64], clean.view(rows, 2, D).cpu()[-1, :, :64])
    if rows > 1:
        assert torch.equal(got[:-1], clean.view(rows, 2, D).cpu()[:-1])


def test_attention_takes_strides_and_writes_in_place():
    H, G, D = 4, 2, 64
    kp, vp, tables = cached([90, 40], G, D, 16, seed=13)
    wide = normal(5, H * D + 9, seed=14).bfloat16()
    q = wide[:, 3:3 + H * D]                              # rows that begin anywhere
    rows, start, before = [1, 3], [0, 2], [80, 30]
    table = torch.full((2, 20), -7, dtype=torch.int32)
    table[:, :tables.shape[1]] = tables
    args = (q, start, rows, before, table, kp, vp, H, 0.125)
    dev = wide.to(DEV)
    out = torch.full((5, H * D + 2), 5.0, dtype=torch.bfloat16, device=DEV)[:, 1:1 + H * D]
    from glassbox_amd import ops
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    rest = (ints(start), ints(rows), ints(before), table.to(DEV)[:, :tables.shape[1]], kp.to(DEV), vp.to(DEV), H, 0.125, 3, 200)
    assert ops.fp4_attention_floats(2, H, G, D, 3, 200) == 0
    ops.fp4_attention(dev[:, 3:3 + H * D], out, *rest)
    check(out, *args)
    ops.fp4_attention(dev[:, 3:3 + H * D], dev[:, 3:3 + H * D], *rest)
    assert torch.equal(dev[[0, 2, 3, 4], 3:3 + H * D], out[[0, 2, 3, 4]]) and torch.equal(dev[1].cpu(), wide[1])


def test_attention_and_store_reach_pages_beyond_four_gigabytes():
    from glassbox_amd import ops
    G, D, page = 2, 128, 16
    pages = (1 << 32) // (G * 4 * 17 * page) + 40
    kp, vp = (torch.zeros(ops.fp4_pages_shape(pages, G, page, D), dtype=torch.uint8, device=DEV) for _ in range(2))
    n = 20
    table = torch.tensor([[pages - 1, pages - 30]], dtype=torch.int32)
    slots = torch.tensor([int(table[0, i // page]) * page + i % page for i in range(n)], dtype=torch.int32)
    rows = normal(n, 6 * D, seed=15).bfloat16()
    q = torch.empty(n, 2 * D, dtype=torch.bfloat16, device=DEV)
    ops.fp4_store(rows.to(DEV), None, None, slots.to(DEV), kp, vp, 2, G, D, q=q)
    few_k, few_v = kp[pages - 30:].cpu(), vp[pages - 30:].cpu()
    k, v = (torch.empty(n, G * D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.fp4_load(slots.to(DEV), kp, vp, k, v)
    heads = rows.view(n, 6, D)
    assert torch.equal(k.cpu().double().view(n, G, D), plain.rounded(heads[:, 2:4])) and torch.equal(v.cpu().double().view(n, G, D), plain.rounded(heads[:, 4:]))
    out = torch.empty(1, 2 * D, dtype=torch.bfloat16, device=DEV)
    ints = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)
    ops.fp4_attention(q[-1:], out, ints(0), ints(1), ints(n - 1), table.to(DEV), kp, vp, 2, 0.1, 1, n)
    few = table - (pages - 30)
    check(out, q[-1:].cpu(), [0], [1], [n - 1], few, few_k, few_v, 2, 0.1)


# ------------------------------------------------------------------------------------------------------------------- products
GEMMS = [(1, 1, 32), (1, 40, 64), (3, 17, 96), (16, 64, 512), (17, 130, 544), (5, 2563, 992), (33, 300, 2048), (64, 96, 4128), (65, 48, 160),
         (130, 1040, 256), (16, 17000, 96), (9, 520, 4128), (1, 8200, 1056), (2, 33000, 128), (20, 16500, 160), (300, 70, 992),
         # (each of the kernels' forms, with k whole and divided, one tile of rows and several)
         (9, 4100, 544), (9, 8200, 544), (17, 4100, 544), (9, 2050, 8224), (30, 1040, 8224), (17, 520, 8224), (9, 4100, 4128), (700, 70, 4128),
         (8, 16400, 96), (5, 24600, 544), (3, 20000, 1056), (1, 25000, 2080),
         (33, 6150, 2080), (65, 12300, 96), (65, 6150, 4128), (33, 6150, 8224), (130, 1000, 960)]


@pytest.mark.parametrize("M,N,K", GEMMS)
@pytest.mark.parametrize("dtype,out_dtype,how", [(torch.bfloat16, torch.bfloat16, "store"), (torch.bfloat16, torch.float32, "add"),
                                                 (torch.bfloat16, torch.bfloat16, "silu"), (torch.float32, torch.float32, "store"),
                                                 (torch.float32, torch.float32, "silu"), (torch.float32, torch.bfloat16, "store"),
                                                 (torch.bfloat16, torch.float32, "silu")])
def test_gemm(M, N, K, dtype, out_dtype, how):
    from glassbox_amd import ops
    if how == "silu":
        N += N % 2
    w = ops.fp4_quantize(normal(N, K, seed=20, scale=0.05).to(DEV))
    wd = torch.empty(N, K, device=DEV)
    ops.fp4_expand(w, wd)
    a = normal(M, K, seed=21, wide=4.0).to(dtype)
    a64, w64 = a.to(DEV).double(), wd.double()
    y, size = a64 @ w64.t(), a64.abs() @ w64.abs().t()
    off = (3 * K + 16) * STEP * size
    cols = N // 2 if how == "silu" else N
    first = normal(M, cols, seed=22)
    if how == "silu":
        g, u, dg, du = y[:, :cols], y[:, cols:], off[:, :cols], off[:, cols:]
        y = g * torch.sigmoid(g) * u
        off = 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + 8 * STEP * (g * u).abs()
    if how == "add":
        y = y + first.to(DEV).double()
        off = off + STEP * y.abs()
    off = off + half_step(out_dtype) * (y.abs() + off) + 1e-30
    for odd in (0, 3):                                    # whole rows, and rows of odd strides that begin anywhere
        given = torch.zeros(M, K + 2 * odd, dtype=dtype, device=DEV)[:, odd:odd + K]
        given.copy_(a)
        out = torch.full((M, cols + 2 * odd), 3.0, dtype=out_dtype, device=DEV)
        mine = out[:, odd:odd + cols]
        if how == "add":
            mine.copy_(first)
        floats = ops.fp4_gemm_floats(M, N, K, dtype, out_dtype, how == "silu")
        ops.fp4_gemm(given, w, mine, accumulate=how == "add", silu_mul=how == "silu",
                     workspace=torch.full((floats,), math.nan, device=DEV) if floats else None)
        far = (mine.double() - y).abs() > off
        assert not far.any(), (float((mine.double() - y).abs()[far].max()), float(off[far].max()))
        if odd:
            assert (out[:, :odd] == 3).all() and (out[:, odd + cols:] == 3).all()


@pytest.mark.parametrize("M,N,K,how", [(1540, 8208, 8192, "silu"), (1600, 8200, 8192, "add"), (1536, 2064, 2048, "silu"), (770, 4100, 4128, "store"), (1537, 2051, 2080, "store"), (771, 4099, 4128, "add"), (700, 8300, 640, "store"), (260, 28672, 96, "silu")])
def test_gemm_of_many_rows(M, N, K, how):
    """Through the weights' values and in tiles, with the workspace and without it: of one size within rounding."""
    from glassbox_amd import ops
    w = ops.fp4_quantize((torch.randn(N, K, generator=torch.Generator().manual_seed(27)) * 0.05).to(DEV))
    wd = torch.empty(N, K, device=DEV)
    ops.fp4_expand(w, wd)
    a = normal(M, K, seed=28).bfloat16().to(DEV)
    out_dtype, cols = (torch.float32, N) if how == "add" else (torch.bfloat16, N // 2 if how == "silu" else N)
    y, size = a.double() @ wd.double().t(), a.double().abs() @ wd.double().abs().t()
    off = (3 * K + 16) * STEP * size
    if how == "silu":
        g, u, dg, du = y[:, :cols], y[:, cols:], off[:, :cols], off[:, cols:]
        y, off = g * torch.sigmoid(g) * u, 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + 8 * STEP * (g * u).abs()
    off = off + half_step(out_dtype) * (y.abs() + off) + 1e-30
    floats = ops.fp4_gemm_floats(M, N, K, torch.bfloat16, out_dtype, how == "silu")
    for ws in ([None] if floats == 0 else [None, torch.full((floats,), math.nan, device=DEV)]):
        out = torch.zeros(M, cols, dtype=out_dtype, device=DEV)
        ops.fp4_gemm(a, w, out, accumulate=how == "add", silu_mul=how == "silu", workspace=ws)
        assert ((out.double() - y).abs() <= off).all()


def test_gemm_of_rows_and_weights_that_are_not_finite():
    from glassbox_amd import ops
    w = normal(40, 64, seed=23)
    w[7, 40] = math.inf
    m = ops.fp4_quantize(w.to(DEV))
    for dtype in (torch.float32, torch.bfloat16):
        a = normal(3, 64, seed=24).to(dtype)
        a[1, 3] = math.nan
        out = torch.empty(3, 40, dtype=dtype, device=DEV)
        ops.fp4_gemm(a.to(DEV), m, out)
        bad = out.cpu().isnan()
        assert bad[1].all() and bad[:, 7].all() and not bad[0, :7].any() and not bad[2, 8:].any()


def test_gemm_gives_a_row_the_same_bits_each_time():
    from glassbox_amd import ops
    m = ops.fp4_quantize(normal(700, 2048, seed=25, scale=0.05).to(DEV))
    a = normal(16, 2048, seed=26).bfloat16().to(DEV)
    outs = []
    for _ in range(3):
        out = torch.empty(16, 700, dtype=torch.float32, device=DEV)
        ops.fp4_gemm(a, m, out)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# --------------------------------------------------------------------------------------------------------------- together
def layer(ops, state, out, ws):
    """What a layer does of it: query, key and value heads from the rows, stored and attended to, and the output's product."""
    s = state
    ops.fp4_gemm(s["h"], s["w_qkv"], s["qkv"])
    ops.fp4_store(s["qkv"], s["cos"], s["sin"], s["slots"], s["k"], s["v"], s["H"], s["G"], s["D"], q=s["q"])
    ops.fp4_attention(s["q"], s["att"], s["q_start"], s["q_len"], s["pos0"], s["tables"], s["k"], s["v"], s["H"], s["scale"], s["most"], s["longest"],
                      workspace=ws)
    ops.fp4_gemm(s["att"], s["w_o"], out, accumulate=True)


def a_layer(dtype, seed=30, rows=(1, 1, 9), before=(0, 0, 0), longest=None):
    from glassbox_amd import ops
    H, G, D, page, width = 8, 2, 64, 16, 256
    n, lengths = sum(rows), [r + b for r, b in zip(rows, before)]
    kp, vp, tables = cached(lengths, G, D, page, seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    start = [sum(rows[:i]) for i in range(len(rows))]
    positions = [b + i for r, b in zip(rows, before) for i in range(r)]
    seqs = [s for s, r in enumerate(rows) for _ in range(r)]
    angle = torch.tensor(positions, dtype=torch.float64)[:, None] / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    w_qkv, w_o = normal((H + 2 * G) * D, width, seed=seed + 1, scale=0.06), normal(width, H * D, seed=seed + 2, scale=0.06)
    s = dict(H=H, G=G, D=D, scale=D ** -0.5, most=max(rows), longest=longest or max(lengths), k=kp.to(DEV), v=vp.to(DEV), tables=tables.to(DEV),
             q_start=ints(start), q_len=ints(list(rows)), pos0=ints(list(before)), cos=angle.cos().float().to(DEV), sin=angle.sin().float().to(DEV),
             slots=ints([int(tables[q, p // page]) * page + p % page for q, p in zip(seqs, positions)]),
             h=normal(n, width, seed=seed + 3).to(dtype).to(DEV), w_qkv=ops.fp4_quantize(w_qkv.to(DEV)), w_o=ops.fp4_quantize(w_o.to(DEV)),
             qkv=torch.empty(n, (H + 2 * G) * D, dtype=dtype, device=DEV), q=torch.empty(n, H * D, dtype=dtype, device=DEV),
             att=torch.empty(n, H * D, dtype=dtype, device=DEV))
    floats = ops.fp4_attention_floats(len(rows), H, G, D, s["most"], s["longest"], 0, dtype)
    return s, torch.empty(floats, device=DEV) if floats else None, (w_qkv, w_o, start, rows, before, tables)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layer_of_them(dtype):
    from glassbox_amd import ops
    s, ws, (w_qkv, w_o, start, rows, before, tables) = a_layer(dtype)
    out = torch.zeros(sum(rows), 256, device=DEV)
    layer(ops, s, out, ws)
    H, G, D = s["H"], s["G"], s["D"]
    heads = s["qkv"].cpu().view(-1, H + 2 * G, D)          # each step from what the step before gave
    qkv64 = s["h"].cpu().double() @ plain.rounded(w_qkv).t()
    size = s["h"].cpu().double().abs() @ plain.rounded(w_qkv).abs().t()
    assert ((heads.double().flatten(1) - qkv64).abs() <= 800 * STEP * size + half_step(dtype) * qkv64.abs() * 1.01).all()
    assert torch.equal(s["q"].cpu(), plain.turned(heads[:, :H], s["cos"].cpu(), s["sin"].cpu()).to(dtype).flatten(1))
    check(s["att"], s["q"].cpu(), start, rows, before, tables, s["k"].cpu(), s["v"].cpu(), H, s["scale"])
    att = s["att"].cpu().double()
    want, size = att @ plain.rounded(w_o).t(), att.abs() @ plain.rounded(w_o).abs().t()
    assert ((out.cpu().double() - want).abs() <= (3 * H * D + 16) * STEP * size).all()


def test_a_captured_layer_gives_what_it_gives_eagerly():
    """Two graphs of one layer each, of different steps, with the program's own work between their replays."""
    from glassbox_amd import ops
    cases = []
    for seed, rows, before, longest in ((40, (1, 1), (700, 30), 2000), (50, (5, 40), (3, 60), 300)):
        s, ws, _ = a_layer(torch.bfloat16, seed, rows, before, longest)
        out = torch.zeros(sum(rows), 256, device=DEV)
        layer(ops, s, out, ws)                              # kernels are loaded
        torch.cuda.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer(ops, s, out, ws)
        cases.append((graph, s, out, want, ws))
    for turn in range(3):
        for graph, s, out, want, ws in cases:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn
            eager = torch.zeros_like(out)
            layer(ops, s, eager, ws)
            assert torch.equal(eager, want), turn


def test_two_streams_at_once():
    from glassbox_amd import ops
    works = [a_layer(torch.bfloat16, 60 + 10 * i, (1, 30), (900, 5)) for i in range(2)]
    wants = []
    for s, ws, _ in works:
        out = torch.zeros(31, 256, device=DEV)
        layer(ops, s, out, ws)
        wants.append(out)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in works], [torch.zeros(31, 256, device=DEV) for _ in works]
    torch.cuda.synchronize()
    for _ in range(5):
        for (s, ws, _), stream, out in zip(works, streams, outs):
            with torch.cuda.stream(stream):
                out.zero_()
                layer(ops, s, out, ws)
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_with_the_loosest_bound_of_the_contexts(dtype, rows, window):
    """``max_context`` as large as it may be: more runs than there are keys, the answer of any other bound."""
    kp, vp, tables = cached([rows + 130, rows + 7], 2, 64, 16, 50)
    q = normal(2 * rows, 4 * 64, seed=51).to(dtype)
    for many in (1, 300):                                  # few requests, whose contexts are divided, and more than compute units
        start, length, pos0 = [0, rows] + [0] * (2 * many - 2), [rows, rows] + [0] * (2 * many - 2), [130, 7] + [0] * (2 * many - 2)
        table = tables.repeat(many, 1)
        got = attend(q.to(DEV), start, length, pos0, table.to(DEV), kp.to(DEV), vp.to(DEV), 4, 0.1, window, max_context=2 ** 31 - 1)
        check(got, q, [0, rows], [rows, rows], [130, 7], tables, kp, vp, 4, 0.1, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_at_positions_that_no_table_has(dtype, rows):
    """Positions at the ends of 32 bits: with a window such rows see nothing and give zeros, without one all that the table has, from behind; those
    before the first key see nothing."""
    kp, vp, tables = cached([64], 2, 64, 16, 52)
    q = normal(rows, 4 * 64, seed=53).to(dtype)
    k, v, t = kp.to(DEV), vp.to(DEV), tables.to(DEV)
    every = attend(q.to(DEV), [0], [rows], [64], t, k, v, 4, 0.1, max_context=200)
    check(every, q, [0], [rows], [64], tables, kp, vp, 4, 0.1)
    for pos0 in (2 ** 31 - 1, 2 ** 31 - 60, 2 ** 30):
        far = attend(q.to(DEV), [0], [rows], [pos0], t, k, v, 4, 0.1, max_context=200)
        assert torch.equal(far, every)
        for window in (1, 64, 2 ** 31 - 1 - 2 ** 30 - 100):
            assert (attend(q.to(DEV), [0], [rows], [pos0], t, k, v, 4, 0.1, window, max_context=200) == 0).all()
    for pos0 in (-rows, -(2 ** 31) + rows):
        for window in (0, 1, 2 ** 31 - 1):
            assert (attend(q.to(DEV), [0], [rows], [pos0], t, k, v, 4, 0.1, window, max_context=200) == 0).all()


@pytest.mark.parametrize("how", ["silu", "add", "store"])
def test_gemm_through_the_values_into_rows_that_begin_anywhere(how):
    from glassbox_amd import ops
    M, N, K = 1537, 2064, 2048
    w = ops.fp4_quantize(normal(N, K, seed=54, scale=0.05).to(DEV))
    a = normal(M, K, seed=55).bfloat16().to(DEV)
    dtype, cols = (torch.float32, N) if how == "add" else (torch.bfloat16, N // 2 if how == "silu" else N)
    floats = ops.fp4_gemm_floats(M, N, K, torch.bfloat16, dtype, how == "silu")
    assert floats >= N * K // 2
    outs = []
    for odd in (0, 3):
        out = torch.full((M, cols + 2 * odd), 2.0, dtype=dtype, device=DEV)
        ops.fp4_gemm(a, w, out[:, odd:odd + cols], accumulate=how == "add", silu_mul=how == "silu", workspace=torch.empty(floats, device=DEV))
        assert not odd or ((out[:, :odd] == 2).all() and (out[:, odd + cols:] == 2).all())
        outs.append(out[:, odd:odd + cols])
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("M,N,K", [(1, 64, 96), (8, 2048, 544), (3, 2592, 160), (7, 6176, 64), (5, 40, 32), (8, 4096, 4128), (2, 4128, 64), (3, 16416, 32), (8, 16416, 32),
                                   (4, 24608, 4128), (2, 24608, 4128)])
@pytest.mark.parametrize("gamma_dtype", [torch.float32, torch.bfloat16])
def test_a_product_prepares_a_norm_and_the_next_takes_it(M, N, K, gamma_dtype):
    from glassbox_amd import ops
    w = ops.fp4_quantize(normal(N, K, seed=60, scale=0.05).to(DEV))
    wd = torch.empty(N, K, device=DEV)
    ops.fp4_expand(w, wd)
    a, first = normal(M, K, seed=61, wide=4.0).bfloat16().to(DEV), normal(M, N, seed=62, wide=3.0).to(DEV)
    gamma = (normal(N, seed=63) + 1).to(gamma_dtype).to(DEV)
    tiles, eps = ops.fp4_gemm_emit_parts(M, N), 1e-5
    assert tiles > 0
    x, plain_x = first.clone(), first.clone()
    h = torch.full((M, N + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    parts = torch.full((tiles + 1, ops.parts_stride(M)), 7.0, device=DEV)
    ops.fp4_gemm(a, w, x, accumulate=True, emit=(gamma, h[:, :N], parts))
    ops.fp4_gemm(a, w, plain_x, accumulate=True)
    assert torch.equal(x, plain_x)                                   # the residual is what it is without
    assert torch.equal(h[:, :N], (gamma.float() * x).bfloat16()) and (h[:, N:] == 3).all() and (parts[tiles:] == 7).all()
    with pytest.raises(ops.KernelError, match="each of"):
        ops.fp4_gemm(a, w, plain_x, accumulate=True, emit=(gamma, h[:, :N], parts.flatten()[:tiles * 8 - 1]))
    squares = (x.double() ** 2).sum(-1)
    assert ((parts[:tiles, :M].double().sum(0) - squares).abs() <= (N / 2 + 8) * STEP * squares).all()   # (half a step for each addition)
    if N % 32:
        return
    C = 98 if N > 2592 else 16402
    w2 = ops.fp4_quantize(normal(C, N, seed=64, scale=0.05).to(DEV))
    wd2 = torch.empty(C, N, device=DEV)
    ops.fp4_expand(w2, wd2)
    root = 1 / torch.sqrt(squares / N + eps)
    rows = h[:, :N].double()
    y, size = rows @ wd2.double().t() * root[:, None], rows.abs() @ wd2.double().abs().t() * root[:, None]
    off = (3 * N + 16 + N / 2 + 16) * STEP * size                    # the sums; the root of a sum of N squares and of as many partial sums
    for out_dtype in (torch.bfloat16, torch.float32):
        out = torch.empty(M, C, dtype=out_dtype, device=DEV)
        ops.fp4_gemm(h[:, :N], w2, out, rms_parts=(parts, tiles, eps))
        assert ((out.double() - y).abs() <= off + half_step(out_dtype) * (y.abs() + off)).all()
        out = torch.empty(M, C // 2, dtype=out_dtype, device=DEV)
        ops.fp4_gemm(h[:, :N], w2, out, silu_mul=True, rms_parts=(parts, tiles, eps))
        g, u, dg, du = y[:, :C // 2], y[:, C // 2:], off[:, :C // 2], off[:, C // 2:]
        z, dz = g * torch.sigmoid(g) * u, 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + 8 * STEP * (g * u).abs()
        assert ((out.double() - z).abs() <= dz + half_step(out_dtype) * (z.abs() + dz) + 1e-30).all()


@pytest.mark.parametrize("M,N,K", [(30, 1040, 8224), (64, 4100, 4128), (65, 6148, 4128), (700, 68, 4128), (9, 2052, 8224), (520, 260, 8224), (12, 8192, 8192)])
@pytest.mark.parametrize("gamma_dtype", [torch.float32, torch.bfloat16])
def test_a_product_that_divides_k_does_the_norm(M, N, K, gamma_dtype):
    from glassbox_amd import ops
    assert ops.fp4_gemm_emit_mode(M, N, K) == 2
    w = ops.fp4_quantize(normal(N, K, seed=70, scale=0.05).to(DEV))
    a, first = normal(M, K, seed=71, wide=4.0).bfloat16().to(DEV), normal(M, N, seed=72, wide=3.0).to(DEV)
    gamma, eps = (normal(N, seed=73) + 1).to(gamma_dtype).to(DEV), 1e-5
    x, plain_x = torch.full((M, N + 4), 5.0, device=DEV), first.clone()
    x[:, :N] = first
    h = torch.full((M, N + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    ws = torch.full((ops.fp4_gemm_floats(M, N, K, torch.bfloat16, torch.float32) + 16,), math.nan, device=DEV)
    for few in (None, ws[:-17]):
        with pytest.raises(ops.KernelError, match="divide k"):
            ops.fp4_gemm(a, w, x[:, :N], accumulate=True, emit=(gamma, h[:, :N], eps), workspace=few)
    ops.fp4_gemm(a, w, x[:, :N], accumulate=True, emit=(gamma, h[:, :N], eps), workspace=ws[:-16])
    ops.fp4_gemm(a, w, plain_x, accumulate=True, workspace=ws[:-16])
    assert torch.equal(x[:, :N], plain_x) and (x[:, N:] == 5).all() and (h[:, N:] == 3).all() and ws[-16:].isnan().all()
    rows = plain_x.double()
    want = gamma.double() * rows / torch.sqrt((rows ** 2).mean(-1, keepdim=True) + eps)
    # up to 8 numbers a thread, 6 exchanges and 16 waves make a row's sum, each a rounding of what is positive: half of that in its root; and a quotient, two
    # roots' and quotients' roundings, two products
    off = (15 + 8) * STEP * want.abs()
    assert ((h[:, :N].double() - want).abs() <= off + half_step(torch.bfloat16) * (want.abs() + off) + 1e-30).all()


def test_a_norm_is_refused_where_a_product_does_not_divide_k():
    from glassbox_amd import ops
    M, N, K = 33, 36, 4128
    assert ops.fp4_gemm_emit_mode(M, N, K) == 0 and ops.fp4_gemm_emit_mode(0, N, K) == 0 and ops.fp4_gemm_emit_mode(12, 8196, 8192) == 0
    w, x = ops.fp4_quantize(torch.ones(N, K, device=DEV)), torch.zeros(M, N, device=DEV)
    with pytest.raises(ops.KernelError, match="divide k"):
        ops.fp4_gemm(torch.ones(M, K, dtype=torch.bfloat16, device=DEV), w, x, accumulate=True, workspace=torch.zeros(1 << 20, device=DEV),
                     emit=(torch.ones(N, device=DEV), torch.zeros(M, N, dtype=torch.bfloat16, device=DEV), 1e-5))
    assert (x == 0).all()
