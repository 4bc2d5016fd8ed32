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


# rows, rows of w, k, how: divided lines, divided tiles, both with the norm behind them done, the weights' values first
WORKS = [(12, 2048, 8192, torch.bfloat16, "store"), (12, 4100, 8192, torch.bfloat16, "silu"), (40, 2048, 8192, torch.bfloat16, "add"),
         (33, 2052, 4128, torch.float32, "store"), (12, 2048, 8192, torch.bfloat16, "norm"), (64, 4096, 8192, torch.bfloat16, "norm"),
         (1600, 2048, 2048, torch.bfloat16, "silu"), (1600, 2048, 2048, torch.bfloat16, "add")]


def work(M, N, K, dtype, how, seed, space=None):
    """A call of one product with the workspace that it asks for, and what it writes"""
    from glassbox_amd import ops
    a, w, _, _ = operands(M, N, K, dtype, seed)
    out_dtype = torch.float32 if how in ("add", "norm") else dtype
    floats = ops.fp4_gemm_floats(M, N, K, dtype, out_dtype, how == "silu")
    assert 0 < floats <= (1 << 23) and (how != "norm" or ops.fp4_gemm_emit_mode(M, N, K) == 2)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    space = torch.empty(floats, device=DEV) if space is None else space
    base = torch.randn(M, N, generator=g, device=DEV)
    out = torch.empty(M, N // 2 if how == "silu" else N, dtype=out_dtype, device=DEV)
    h, gamma = torch.empty(M, N, dtype=torch.bfloat16, device=DEV), torch.rand(N, generator=g, device=DEV) + 0.5

    def call():
        if how in ("add", "norm"):
            out.copy_(base)
        else:
            out.fill_(7)
        h.fill_(7)
        ops.fp4_gemm(a, w, out, accumulate=how in ("add", "norm"), silu_mul=how == "silu", workspace=space,
                     emit=(gamma, h, 1e-5) if how == "norm" else None)

    return call, (out, h), space


def made(call, outs):
    call()
    torch.cuda.synchronize()
    return [t.clone() for t in outs]


def test_captured_products_with_their_workspaces_give_what_they_give_eagerly():
    """A graph of each and one of all of them, with one workspace for all, and the program's own work on it between the replays."""
    one = torch.empty(1 << 23, device=DEV)
    works = [work(*w, 20 + 2 * i, one) for i, w in enumerate(WORKS)]
    wants = [made(call, outs) for call, outs, _ in works]
    graphs = []
    for calls in [[w] for w in works] + [works]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for call, _, _ in calls:
                call()
        graphs.append((graph, calls))
    for turn in range(3):
        for graph, calls in graphs:
            for _, outs, space in calls:
                space.fill_(float("nan"))
                for t in outs:
                    t.fill_(3)
            graph.replay()
            torch.cuda.synchronize()
            for w in calls:
                which = works.index(w)
                assert all(torch.equal(t, want) for t, want in zip(w[1], wants[which])), (turn, WORKS[which])
            call, outs, _ = calls[0]
            assert all(torch.equal(t, want) for t, want in zip(made(call, outs), wants[works.index(calls[0])])), turn


@pytest.mark.parametrize("first,second", [(0, 4), (1, 2), (3, 5), (6, 7)])
def test_products_with_workspaces_of_their_own_on_two_streams_at_once(first, second):
    works = [work(*WORKS[i], 60 + i) for i in (first, second)]
    wants = [made(call, outs) for call, outs, _ in works]
    streams = [torch.cuda.Stream() for _ in works]
    torch.cuda.synchronize()
    for _ in range(6):
        for (call, _, _), stream in zip(works, streams):
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    for (_, outs, _), want, i in zip(works, wants, (first, second)):
        assert all(torch.equal(t, w) for t, w in zip(outs, want)), WORKS[i]


@pytest.mark.parametrize("requests", [12, 16, 40])
def test_steps_of_many_requests_replayed(requests):
    """An engine's steps of single tokens whose products divide k and do the norms behind them: replayed, the bits of the same steps launched one by one."""
    import helpers
    from glassbox_amd import ops
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.engine import Engine
    from glassbox_amd.engine.decode_graphs import padded_rows
    from glassbox_amd.weights import build_model
    from glassbox_amd.weights.loader import random_tensors
    d, inter, vocab = 2048, 8192, 90
    model = build_model(config_from_dict(dict(helpers.TINY_B, hidden_size=d, intermediate_size=inter, num_hidden_layers=2, num_attention_heads=4,
                                              num_key_value_heads=2, head_dim=64, vocab_size=vocab)))
    model.load_tree(random_tensors(model, 7, 0.03, "uniform", torch.bfloat16, "cuda:0"))
    rows = padded_rows(requests)
    assert ops.fp4_gemm_floats(rows, d, inter) > 0 and ops.fp4_gemm_emit_mode(rows, d, inter) == 2
    got = []
    for replayed in (True, False):
        eng = Engine(model, dtype="bfloat16", max_tokens=48 * 64, max_seqs=48, kv_cache="fp4", weights="fp4")
        eng.step([(i, helpers.random_tokens(vocab, 3 + i % 7, i), []) for i in range(requests)])
        steps = []
        for t in range(7):
            if not replayed:
                for shape in eng.decode_graphs.shapes.values():
                    shape.runs = 0
            steps.append(eng.step([(i, [(5 * t + 3 * i) % vocab], [0]) for i in range(requests)])[:, :vocab].clone())
        assert eng.decode_graphs.replays == (5 if replayed else 0)
        got.append(steps)
        del eng
    for t, (mine, other) in enumerate(zip(*got)):
        assert mine.isfinite().all() and torch.equal(mine, other), t
