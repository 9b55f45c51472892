"""The paged cache's operators at edges that test_gpu_paged.py leaves out: query blocks that are partly filled, on every
page size; rows that are not finite; values and queries of any magnitude; what unused memory holds; calls that do not fit
together; captured steps; a cache's state after a call that fails.

Bounds are those of test_gpu_paged.py's docstring.
"""
import math

import numpy as np
import pytest

from test_gpu_paged import FORMATS, Case, queries_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("tokens", [65, 100, 127, 129, 193])
def test_chunks_that_fill_a_query_block_in_part(cuda, bits, dtype, dim, group, page, tokens):
    """Chunks of odd lengths, whose last block of 128 query rows has rows to spare, over slots that end anywhere in a
    page and in a tile; one slot is shorter than the chunk, so that its first queries see nothing."""
    case = Case(cuda, bits, dtype, dim, group, page, 2, [tokens + 3 * page + 5, 37, 2, 400], seed=tokens)
    counts = [tokens, tokens - 40]
    queries = queries_of(case, counts, 1)
    out, lse = case.attend(queries, counts)
    case.check(queries, counts, out, lse)


# Every key of these rows is NaN; formats with 16-bit and 4-bit rows.
SOME = [(16, "f16", 128, 0), (16, "bf16", 64, 0), (4, "bf16", 128, 64), (4, "f16", 64, 32)]


def poison_keys(case, slot, rows):
    pool = case.pages.keys if case.bits == 16 else case.pages.key_scales
    rows = np.asarray(rows)
    pool[case.host_table[slot, rows // case.page].tolist(), (rows % case.page).tolist()] = float("nan")


@pytest.mark.parametrize("bits,dtype,dim,group", SOME)
@pytest.mark.parametrize("groups", [2, 12, 30, 70])
def test_lse_of_keys_that_are_not_numbers(cuda, bits, dtype, dim, group, groups):
    """A slot's only row, the only row of its last tile, and all of its rows: out and lse are both NaN."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [1, 33, 65, 40, 150], seed=8)
    for slot, rows in ((0, [0]), (1, [32]), (2, [64]), (3, range(40))):
        poison_keys(case, slot, list(rows))
    out, lse = case.attend(queries_of(case, [1] * 5, groups), [1] * 5)
    assert torch.isnan(out[:4]).all() and torch.isnan(lse[:4]).all()
    assert torch.isfinite(out[4]).all() and torch.isfinite(lse[4]).all()


@pytest.mark.parametrize("bits,dtype,dim,group", SOME)
@pytest.mark.parametrize("groups", [1, 14, 32, 70])
def test_lse_of_a_split_slot_with_keys_that_are_not_numbers(cuda, bits, dtype, dim, group, groups):
    """So many NaN rows that whole blocks and warps meet nothing else."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 64, 1, [6000, 6000], seed=8)
    poison_keys(case, 0, np.arange(2000, 4500))
    out, lse = case.attend(queries_of(case, [1, 1], groups), [1, 1])
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isfinite(out[1]).all() and torch.isfinite(lse[1]).all()


@pytest.mark.parametrize("bits,dtype,dim,group", SOME)
@pytest.mark.parametrize("groups", [3, 70])
def test_lse_of_queries_that_are_not_numbers(cuda, bits, dtype, dim, group, groups):
    import torch

    case = Case(cuda, bits, dtype, dim, group, 64, 1, [500, 20], seed=8)
    queries = queries_of(case, [1, 1], groups)
    queries[0, 1, 7] = float("nan")
    queries[1, 0] = float("nan")
    out, lse = case.attend(queries, [1, 1])
    bad = torch.zeros(2, groups, dtype=torch.bool, device=cuda)
    bad[0, 1] = bad[1, 0] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.isfinite(out[~bad]).all() and torch.isfinite(lse[~bad]).all()
