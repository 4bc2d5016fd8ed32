"""Operands of the four-bit operators that are columns of one tensor, without a GPU: taken where they share no memory, refused where they do."""
import random

import pytest
import torch

from glassbox_amd import ops
from test_fp4 import attention, gemm, pages, store

BF, I32 = torch.bfloat16, torch.int32


def test_rows_that_share_no_memory_are_found_by_their_bytes():
    rng = random.Random(3)
    seen = set()
    for _ in range(4000):
        both = rng.random() < 0.5
        a_bytes, b_bytes = rng.randint(1, 6), rng.randint(1, 6)
        a_step = a_bytes + rng.randint(0, 9)
        b_step = max(b_bytes, a_step) if both else b_bytes + rng.randint(0, 9)
        a0, b0, a_rows, b_rows = rng.randint(0, 40), rng.randint(0, 40), rng.randint(1, 5), rng.randint(1, 5)
        held = lambda at, rows, size, step: {at + i * step + j for i in range(rows) for j in range(size)}
        apart = held(a0, a_rows, a_bytes, a_step).isdisjoint(held(b0, b_rows, b_bytes, b_step))
        assert ops._apart(a0, a_rows, a_bytes, a_step, b0, b_rows, b_bytes, b_step) == apart, (a0, a_rows, a_bytes, a_step, b0, b_rows, b_bytes, b_step)
        seen.add((apart, a_step == b_step))
    assert len(seen) == 4
    assert ops._apart(0, 1, 4, 0, 4, 1, 4, 0) and not ops._apart(0, 1, 4, 0, 3, 1, 4, 0)


ROWS = torch.zeros(5, 1024, dtype=BF)


@pytest.mark.parametrize("call", [
    lambda: ops.fp4_load(torch.zeros(5, dtype=I32), pages(), pages(), ROWS[:, :128], ROWS[:, 128:256]),      # (as a stacked row has them)
    lambda: store(qkv=ROWS[:, :512], q=ROWS[:, 512:768]),
    lambda: attention(q=ROWS[:, :256], out=ROWS[:, 256:512]),
    lambda: gemm(a=ROWS[:3, :64], out=ROWS[:3, 64:74]),
    lambda: gemm(a=ROWS[:3, :64], out=torch.as_strided(ROWS, (3, 10), (512, 1), 64)),                        # (rows closer together)
])
def test_neighbouring_columns_are_taken(call):
    with pytest.raises(ops.KernelError, match="current GPU"):       # (everything before has been checked)
        call()


@pytest.mark.parametrize("call", [
    lambda: ops.fp4_load(torch.zeros(5, dtype=I32), pages(), pages(), ROWS[:, :128], ROWS[:, 127:255]),
    lambda: store(qkv=ROWS[:, :512], q=ROWS[:, 511:767]),
    lambda: attention(q=ROWS[:, :256], out=ROWS[:, 255:511]),
    lambda: gemm(a=ROWS[:3, :64], out=ROWS[:3, 63:73]),
    lambda: gemm(a=ROWS[:3, :64], out=torch.as_strided(ROWS, (3, 10), (480, 1), 64)),                        # (its third row reaches into a's second)
])
def test_columns_that_overlap_are_refused(call):
    with pytest.raises(ops.KernelError, match="memory|other columns|other rows"):
        call()
