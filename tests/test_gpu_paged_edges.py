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
