"""The paged cache's operators at edges that test_gpu_paged.py leaves out: query blocks that are partly filled, on every
page size; rows that are not finite; values and queries of any magnitude; what unused memory holds; calls that do not fit
together; captured steps; a cache's state after a call that fails.

Bounds are those of test_gpu_paged.py's docstring.
"""
import math

import numpy as np
import pytest

from test_gpu_paged import APPEND, FORMATS, UNIT, Case, check_append, queries_of, run_append

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


def compare(case, queries, counts, out, lse, scale=None, absent=None, flag=0):
    """Case.check's bound, with what weights below f16's normal range lose (2^-22 of the largest) taken of the slot's
    largest value in the channel instead of 1; a weight times a scale below f16's normal range loses 2^-25 (its codes
    eight times that) beside a largest weight of 2^8.  absent: slot -> rows that are left out."""
    dim, heads = case.dim, case.heads
    groups = queries.shape[1] // heads
    scale = dim ** -0.5 if scale is None else scale
    q = queries.double().cpu().numpy()
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    name = "bf16" if str(out.dtype).endswith("bfloat16") else "f16"
    unit = UNIT["f16"] if case.bits == 4 else UNIT[name]
    lengths = case.lengths.cpu().tolist()
    t = 0
    for s, n in enumerate(counts):
        for i in range(n):
            for h in range(heads):
                slot = s * heads + h
                keep = np.arange(max(0, lengths[slot] - n + i + 1))
                if absent and slot in absent:
                    keep = np.setdiff1d(keep, absent[slot])
                at = slice(h * groups, (h + 1) * groups)
                if keep.size == 0:
                    assert (got[t, at] == 0).all() and np.isneginf(got_lse[t, at]).all(), (s, i, h)
                    continue
                keys, values, sizes = case.rows[slot][0][keep], case.rows[slot][1][keep], case.sizes[slot][keep]
                scores = scale * q[t, at] @ keys.T
                top = scores.max(-1, keepdims=True)
                weight = np.exp(scores - top)
                total = weight.sum(-1, keepdims=True)
                want, want_lse = weight @ values / total, (top + np.log(total))[:, 0]
                d = (dim + 16) * 2.0 ** -23 * abs(scale) * (np.abs(q[t, at]) @ np.abs(keys).T).max()
                bound = ((2 * unit + 4 * d + 2.0 ** -16) * (weight @ sizes / total) + UNIT[name] * np.abs(want) +
                         keep.size / total * (2.0 ** -22 * case.sizes[slot].max(0) + (2.0 ** -30 if case.bits == 4 else 0)) +
                         (2.0 ** -25 if name == "f16" else 0))
                off = np.abs(got[t, at] - want)
                assert (off <= bound).all(), (s, i, h, off.max(), bound.min())
                assert (np.abs(got_lse[t, at] - want_lse) <= 2 * d + 2.0 ** -20 * (1 + np.abs(want_lse))).all(), (s, i, h)
            t += 1
    assert int(case.flag.item()) == flag


def fill_unused(case, scale, offset):
    """(scale, offset) in every row of the pages that no slot holds."""
    import torch

    used = np.zeros(tuple(case.pages.positions.shape), dtype=bool)
    for slot, n in enumerate(case.lengths.tolist()):
        row = np.arange(n)
        used[case.host_table[slot, row // case.page], row % case.page] = True
    unused = torch.from_numpy(~used).to(case.device)
    pair = torch.tensor([scale, offset], dtype=torch.float16, device=case.device)
    for scales in (case.pages.key_scales, case.pages.value_scales):
        scales[unused] = pair


@pytest.mark.parametrize("dim,group", [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("tokens,groups", [(1, 4), (3, 4), (7, 4), (1, 70)])
def test_scales_beyond_a_slot_are_not_used(cuda, dim, group, page, tokens, groups):
    """The same bits whatever the unused rows' scales hold, in pages (and, where a page of 16 rows ends a tile, in what
    an earlier call left in shared memory), for values so small that their weights' precision would show it."""
    import torch

    lengths = [37, 7, 16, 100]
    case = Case(cuda, 4, "bf16", dim, group, page, 1, lengths, seed=3, value_spread=lambda n: np.full(n, 1e-3))
    large = Case(cuda, 4, "bf16", dim, group, page, 1, [1024] * 32, seed=4, value_spread=lambda n: np.full(n, 60000.0))
    counts = [tokens] * 4
    queries = queries_of(case, counts, groups)
    fill_unused(case, 0.0, 0.0)
    want, want_lse = case.attend(queries, counts)
    compare(case, queries, counts, want, want_lse)
    for scale, offset in ((float("nan"), float("nan")), (65504.0, 0.0), (-65504.0, 1.0), (float("inf"), float("-inf")), (0.0, 0.0)):
        fill_unused(case, scale, offset)
        large.attend(queries_of(large, [1] * 32, groups), [1] * 32)
        out, lse = case.attend(queries, counts)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), scale


def refill(case, make):
    """New rows in every slot, appended (so quantised) as a user's are: make(n) gives float32 keys and values [n, D]."""
    import torch

    from code_for_iclr27_b200.paged import paged_append, paged_read

    zero = torch.zeros(1, dtype=torch.int32, device=case.device)
    for slot, n in enumerate(case.lengths.tolist()):
        if n == 0:
            continue
        new = [torch.from_numpy(x.astype(np.float32)).to(case.dtype).to(case.device)[:, None] for x in make(n)]
        at = slice(slot, slot + 1)
        paged_append(case.pages, case.table[at], case.lengths[at], *new, torch.zeros(n, dtype=torch.int64, device=case.device),
                     case.starts([n]), case.flag)
        keys, values, _ = paged_read(case.pages, case.table[at], zero, case.starts([n]), n, torch.float32, case.flag)
        case.rows[slot] = (keys.double().cpu().numpy(), values.double().cpu().numpy())
        if case.bits == 16:
            case.sizes[slot] = np.abs(case.rows[slot][1])
        else:
            row = np.arange(n)
            held = case.pages.value_scales.double().cpu().numpy()[case.host_table[slot, row // case.page], row % case.page]
            case.sizes[slot] = np.repeat(8 * held[..., 0] + np.abs(held[..., 1]), case.group, -1)
    assert int(case.flag.item()) == 0


FOUR_BITS = [(4, "bf16", 128, 32), (4, "bf16", 128, 64), (4, "bf16", 128, 128), (4, "bf16", 64, 32), (4, "bf16", 64, 64)]


@pytest.mark.parametrize("bits,dtype,dim,group", FOUR_BITS)
@pytest.mark.parametrize("groups", [4, 14, 30, 70])
@pytest.mark.parametrize("kind", ["huge", "tiny", "rising", "falling", "mixed"])
def test_values_of_any_magnitude(cuda, bits, dtype, dim, group, groups, kind):
    """Values up to what a group's float16 scale and offset can name (some 500,000, far beyond float16), down to
    1e-6, and both in one slot.  The ends of every group's range are set so that its offset stays in float16's range."""
    rng = np.random.default_rng(5)
    size = {"huge": lambda n: np.full(n, 5e5), "tiny": lambda n: np.full(n, 1e-6),
            "rising": lambda n: np.geomspace(1e-6, 5e5, n), "falling": lambda n: np.geomspace(5e5, 1e-6, n),
            "mixed": lambda n: np.where(np.arange(n) % 97 == 50, 3e5, 1e-3)}[kind]

    def make(n):
        values = rng.uniform(-0.9, 0.9, (n, dim))
        values[:, 0::group], values[:, 1::group] = -1.0, 0.96
        return rng.standard_normal((n, dim)), values * size(n)[:, None]

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [700, 40], seed=13)
    refill(case, make)
    queries = queries_of(case, [1, 1], groups)
    out, lse = case.attend(queries, [1, 1])
    assert np.isfinite(out.float().cpu().numpy()).all()
    compare(case, queries, [1, 1], out, lse)


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_steps_of_a_cache(cuda, bits):
    """Two graphs of a PagedCache's step, captured one after the other: the second may be replayed first, on streams of
    their own, beside the cache's own calls, and each gives the bits of a direct call."""
    import torch

    from code_for_iclr27_b200.paged import PagedCache, attention_workspace
    from test_gpu_arena import make_packed

    cache = PagedCache(3, 1, 4, 128, 200, cuda, bits=bits, page_size=64, max_rows=2048)
    cache.load(0, make_packed(cuda, seed=1))
    cache.advance([1])
    for layer in range(3):
        cache.append(layer, *(queries_of_shape((1, 4, 128), seed, cuda) for seed in (3, 4)), torch.tensor([900], device=cuda))
    queries = [queries_of_shape((1, 8, 128), seed, cuda) for seed in (1, 2)]
    kept = attention_workspace(cuda)

    def step(query, **more):
        return [cache.attend(layer, query, **more) for layer in range(3)]

    want = [step(q) for q in queries]
    torch.cuda.synchronize()
    graphs, held = [], []
    junk = torch.full((256 << 20,), 0x5a, dtype=torch.uint8, device=cuda)
    del junk
    torch.cuda.empty_cache()  # memory that a graph's pool is given from here on may hold anything
    for query in queries:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(query))
    for workspace in getattr(cache, "_workspaces", {}).values():
        assert int(workspace[:4 * 4096].count_nonzero()) == 0  # a direct call finds its counters at zero
    for order in ((1, 0), (0, 1), (1, 1)):
        for tensors in held:
            for out, lse in tensors:
                out.fill_(float("nan"))
                lse.fill_(float("nan"))
        for number in order:
            graphs[number].replay()
        torch.cuda.synchronize()
        for number in order:
            for (out, lse), (want_out, want_lse) in zip(held[number], want[number]):
                assert torch.equal(out, want_out) and torch.equal(lse, want_lse)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        step(queries[0])
    torch.cuda.synchronize()
    for number in range(2):
        for (out, lse), (want_out, want_lse) in zip(held[number], want[number]):
            assert torch.equal(out, want_out) and torch.equal(lse, want_lse)
    for out, want_out in zip(step(queries[1], workspace=kept), want[1]):
        assert torch.equal(out[0], want_out[0]) and torch.equal(out[1], want_out[1])
    cache.check_flags()


def queries_of_shape(shape, seed, device):
    import torch

    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(device)


@pytest.mark.parametrize("bits", [16, 4])
def test_load_that_fails_changes_nothing(cuda, bits):
    """Too many rows for the pages or for a slot, another dimension, type, number of heads or of layers: the sequence
    keeps what it held."""
    import torch

    from code_for_iclr27_b200.kvcache import PackedCache
    from code_for_iclr27_b200.paged import PagedCache
    from test_gpu_arena import make_packed

    packed = make_packed(cuda, seed=1)
    cache = PagedCache(3, 2, 4, 128, 170, cuda, bits=bits, page_size=64, max_rows=1024)
    cache.load(1, packed)

    def state():
        back = cache.to_packed(1)
        return ([t for layer in back.layers for t in (layer.keys, layer.values, layer.positions, layer.cumulative)],
                [(layer.head_lens, layer.prompt_lens) for layer in back.layers], cache.rows.tolist(),
                cache.prompt_rows.tolist(), cache.free_pages(), cache.lengths.tolist())

    before = state()

    def made(rows=64, dim=128, dtype=torch.bfloat16, heads=4, layers=3, values=None):
        other = PackedCache()
        for _ in range(layers):
            keys = torch.zeros(heads * rows, dim, dtype=dtype, device=cuda)
            other.add_layer(keys, keys.clone() if values is None else values(keys), torch.zeros(heads * rows, device=cuda),
                            [rows] * heads, [0] * heads)
        return other

    wrong = [(MemoryError, made(rows=1000)), (MemoryError, made(rows=1100)), (ValueError, made(dim=64)), (ValueError, made(heads=3)),
             (ValueError, made(layers=2)), (ValueError, made(dtype=torch.float32)), (ValueError, PackedCache()),
             (ValueError, made(values=lambda k: k[:-1])), (ValueError, made(values=lambda k: k.half()))]
    elsewhere = made()
    elsewhere.layers[2].values = elsewhere.layers[2].values.cpu()
    wrong.append((ValueError, elsewhere))
    if bits == 16:
        wrong.append((ValueError, made(dtype=torch.float16)))
    for error, other in wrong:
        with pytest.raises(error):
            cache.load(1, other)
        now = state()
        assert now[1:] == before[1:]
        assert all(torch.equal(a, b) for a, b in zip(now[0], before[0]))
    for sequence in (-1, 2):
        for call in (lambda: cache.load(sequence, packed), lambda: cache.release(sequence), lambda: cache.to_packed(sequence)):
            with pytest.raises(ValueError):
                call()
    # What the sequence holds counts as free: a request that fits only in its place is taken.
    taken = cache.free_pages()
    cache.load(1, made(rows=64 * ((170 - 2) // 12)))
    assert taken < 170 // 2 + 60 and cache.free_pages() == 170 - 12 * ((170 - 2) // 12)
    cache.check_flags()


def test_load_of_a_type_that_4_bit_rows_take(cuda):
    """float16 rows into the 4-bit pages of a bfloat16 cache, as before."""
    import torch

    from code_for_iclr27_b200.kvcache import PackedCache
    from code_for_iclr27_b200.paged import PagedCache

    packed = PackedCache()
    rows = torch.randn(2 * 50, 64, generator=torch.Generator().manual_seed(0)).half().to(cuda)
    packed.add_layer(rows, rows * 2, torch.arange(100, dtype=torch.float32, device=cuda), [50, 50], [10, 20])
    cache = PagedCache(1, 1, 2, 64, 8, cuda, bits=4, group=32, page_size=16)
    cache.load(0, packed)
    back = cache.to_packed(0, torch.float32).layers[0]
    step = (rows.float().unflatten(-1, (2, 32)).amax(-1) - rows.float().unflatten(-1, (2, 32)).amin(-1)) / 15
    assert ((back.keys - rows.float()).abs().unflatten(-1, (2, 32)).amax(-1) <= 0.6 * step).all()
    cache.check_flags()


def test_tokens_seen_come_back(cuda):
    """A request's count of seen tokens goes into the pages and back with it, a step's tokens added."""
    from code_for_iclr27_b200.arena import ArenaCache
    from code_for_iclr27_b200.paged import PagedCache
    from test_gpu_arena import make_packed

    packed = [make_packed(cuda, seed=s) for s in (1, 2)]
    packed[1].seen_tokens = 5000
    cache = PagedCache(3, 2, 4, 128, 400, cuda, bits=4, page_size=64, max_rows=2048)
    for s in range(2):
        cache.load(s, packed[s])
    assert [cache.to_packed(s).seen_tokens for s in range(2)] == [packed[0].seen_tokens, 5000]
    cache.advance([1, 7])
    assert [cache.to_packed(s).seen_tokens for s in range(2)] == [packed[0].seen_tokens + 1, 5007]
    assert ArenaCache.from_packed(cache.to_packed(1), margin=8).seen_tokens == 5007
    cache.release(1)
    assert cache.to_packed(1).seen_tokens == 0 and cache.to_packed(0).seen_tokens == packed[0].seen_tokens + 1


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("tokens,groups", [(1, 4), (3, 4), (5, 6), (70, 1)])
def test_rows_whose_page_does_not_exist_are_left_out(cuda, bits, dtype, dim, group, page, tokens, groups):
    """A page id outside the pages takes that page's rows out of the slot, and nothing else; the flag says so."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, page, 2, [300, 75, 150, 16, 40, 600], seed=page)
    counts = [tokens] * 3
    queries = queries_of(case, counts, groups)
    good, good_lse = case.attend(queries, counts)
    compare(case, queries, counts, good, good_lse)
    absent = {}
    for slot, at, entry in ((0, 0, -1), (0, 1, 2 ** 30), (1, 75 // page, -2 ** 31), (2, 1, 2 ** 31 - 1), (3, 0, -5),
                            (5, 300 // page, 2 ** 20), (5, 599 // page, -1)):
        case.table[slot, at] = entry
        rows = np.arange(at * page, (at + 1) * page)
        absent[slot] = np.union1d(absent.get(slot, np.zeros(0, dtype=int)), rows)
    out, lse = case.attend(queries, counts)
    compare(case, queries, counts, out, lse, absent=absent, flag=1)
    again, again_lse = case.attend(queries, counts)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)
    case.flag.zero_()
    # The untouched slot of the last sequence is as it was.
    at = slice(2 * tokens, 3 * tokens)
    assert torch.allclose(out[at, :groups].float(), good[at, :groups].float(), rtol=2 ** -7, atol=1e-6)


def fill_free_memory(device, sizes):
    """NaN in the memory that outputs of these sizes (bytes) are given next."""
    import torch

    torch.cuda.synchronize()
    held = [torch.full((size,), 0xff, dtype=torch.uint8, device=device) for size in sizes for _ in range(4)]
    del held


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "bf16", 128, 0), (4, "f16", 128, 64), (4, "bf16", 64, 32)])
@pytest.mark.parametrize("groups", [1, 5, 40])
@pytest.mark.parametrize("starts", [[2, 3, 5], [0, 0, 0], [8, 8, 8], [0, 4, 6], [1, 1, 8], [-3, 2, 8], [0, 3, 100]])
def test_tokens_of_no_sequence(cuda, bits, dtype, dim, group, groups, starts):
    """Eight tokens, some of them in no sequence: those see nothing (0 and -inf), the flag is set, the others are
    computed."""
    import torch

    from code_for_iclr27_b200.paged import attention_workspace, paged_attention

    case = Case(cuda, bits, dtype, dim, group, 32, 2, [100, 40, 64, 9], seed=3)
    queries = queries_of(case, [8], groups)
    fill_free_memory(cuda, [queries.numel() * 2, queries.shape[0] * queries.shape[1] * 4])
    out, lse = paged_attention(case.pages, case.table, case.lengths, queries,
                               torch.tensor(starts, dtype=torch.int32, device=cuda), attention_workspace(cuda), case.flag)
    assert int(case.flag.item()) == 1
    case.flag.zero_()
    inside = [min(max(x, 0), 8) for x in starts]
    lost = [t for t in range(8) if not inside[0] <= t < inside[2]]
    assert (out[lost] == 0).all() and torch.isneginf(lse[lost]).all()
    counts = [inside[1] - inside[0], inside[2] - inside[1]]
    at = slice(inside[0], inside[2])
    compare(case, queries[at], counts, out[at], lse[at])


def test_starts_that_descend_and_negative_lengths_are_flagged(cuda):
    import torch

    from code_for_iclr27_b200.paged import attention_workspace, paged_attention

    for groups in (4, 40):
        case = Case(cuda, 4, "bf16", 128, 64, 32, 1, [100, 40, 64], seed=3)
        queries = queries_of(case, [8], groups)
        workspace = attention_workspace(cuda)
        starts = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        out, lse = paged_attention(case.pages, case.table, case.lengths, queries, starts(0, 5, 3, 8), workspace, case.flag)
        assert int(case.flag.item()) == 1 and torch.isfinite(out).all() and torch.isfinite(lse).all()
        case.flag.zero_()
        case.lengths[1] = -1
        out, lse = paged_attention(case.pages, case.table, case.lengths, queries, starts(0, 3, 5, 8), workspace, case.flag)
        assert int(case.flag.item()) == 1
        assert (out[3:5] == 0).all() and (lse[3:5] == -math.inf).all() and torch.isfinite(lse[5:]).all()


def test_inputs_that_want_a_gradient_are_refused(cuda):
    """The operators have no backward: an input that requires a gradient would lose it without a word."""
    import torch

    from code_for_iclr27_b200.paged import attention_workspace, paged_append, paged_attention, rotary_table

    case = Case(cuda, 16, "bf16", 128, 0, 16, 2, [20, 20])
    starts, workspace = case.starts([1]), attention_workspace(cuda)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device=cuda)
    position = torch.zeros(1, dtype=torch.int64, device=cuda)
    rotary = rotary_table(4, 128, 10000.0, cuda)
    wants = lambda x: x.clone().requires_grad_(True)  # noqa: E731
    attend = lambda q=q: paged_attention(case.pages, case.table, case.lengths, q, starts, workspace, case.flag)  # noqa: E731
    append = lambda k=k, v=k, q=q, r=rotary: paged_append(case.pages, case.table, case.lengths, k, v, position, starts, case.flag, r, False, q)  # noqa: E731
    for call in (lambda: attend(wants(q)), lambda: append(k=wants(k)), lambda: append(v=wants(k)), lambda: append(q=wants(q)),
                 lambda: append(r=wants(rotary))):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
    attend(wants(q).detach())
    append(wants(k).detach())


@pytest.mark.parametrize("bits,dtype,dim,group", FOUR_BITS)
@pytest.mark.parametrize("tokens", [1, 70])
def test_queries_at_the_ends_of_their_type(cuda, bits, dtype, dim, group, tokens):
    """bfloat16 queries up to 2^128 and down to its subnormals, with scales that bring their scores back."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [200], seed=3)
    for exponent in (127, 126, 100, -100, -125, -126, -130):
        queries = queries_of(case, [tokens], 2).double().clamp(-1.9, 1.9)
        queries[:, :, 0] = 1.75
        queries = (queries * 2.0 ** exponent).to(torch.bfloat16)
        assert torch.isfinite(queries).all()
        scale = case.dim ** -0.5 * 2.0 ** -exponent
        if scale >= 2.0 ** 100:  # what a scale in float32 holds beside the kernels' own factors
            scale = 2.0 ** 100
        out, lse = case.attend(queries, [tokens], scale=scale)
        compare(case, queries, [tokens], out, lse, scale=float(np.float32(scale)))


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "bf16", 128, 0), (4, "f16", 64, 32)])
@pytest.mark.parametrize("tokens", [3, 1500])
def test_queries_without_a_rotation_are_not_numbers(cuda, bits, dtype, dim, group, tokens):
    """A position outside the rotary table: the token's rotated queries are NaN, not what their memory held."""
    import torch

    from code_for_iclr27_b200.paged import paged_append, rotary_table

    case = Case(cuda, bits, dtype, dim, group, 64, 1, [tokens], seed=2)
    rows = queries_of(case, [tokens], 3)
    position = torch.arange(tokens, device=cuda) % 50
    position[1], position[2] = 50, -1
    for rotary_dim in (dim, 32):
        fill_free_memory(cuda, [rows.numel() * 2])
        turned = paged_append(case.pages, case.table, case.lengths, rows[:, :1], rows[:, :1], position, case.starts([tokens]),
                              case.flag, rotary_table(50, rotary_dim, 10000.0, cuda), False, rows)
        assert int(case.flag.item()) == 2
        case.flag.zero_()
        assert torch.isnan(turned[1:3]).all()
        assert torch.isfinite(turned[0]).all() and torch.isfinite(turned[3:]).all()


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "bf16", 128, 0), (4, "f16", 64, 32)])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_rows_read_from_no_page_are_not_numbers(cuda, bits, dtype, dim, group, out):
    import torch

    from code_for_iclr27_b200.paged import paged_read

    kind = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[out]
    case = Case(cuda, bits, dtype, dim, group, 32, 1, [70, 64], seed=2)
    case.table[0, 1] = -1
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    # Slot 0's rows 0..69 (32..63 have no page), slot 1's rows -2..61, and three rows of no slot.
    read = lambda: paged_read(case.pages, case.table, ints(0, -2), ints(0, 70, 134), 137, kind, case.flag)  # noqa: E731
    fill_free_memory(cuda, [137 * dim * kind.itemsize, 137 * 4])
    keys, values, positions = read()
    assert int(case.flag.item()) == 1
    lost = torch.zeros(137, dtype=torch.bool, device=cuda)
    lost[32:64] = lost[70:72] = lost[134:] = True
    for got in (keys, values, positions):
        assert torch.isnan(got[lost]).all() and torch.isfinite(got[~lost]).all()


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (16, True), (32, False), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("counts,heads,query_heads", [([1000, 0, 37], 3, 5), ([1024], 1, 0), ([7, 1030], 2, 4)])
def test_append_of_many_tokens(cuda, bits, dtype, dim, group, rotary, interleaved, counts, heads, query_heads):
    """Over a thousand tokens, not a multiple of what a block takes, with rows (2 heads + query heads) that fill the
    last four of a block in part: every rotation, bit for bit."""
    if rotary > dim:
        pytest.skip("rotates more channels than the head has")
    before = [(53 * i) % 130 for i in range(len(counts) * heads)]
    args = run_append(cuda, bits, dtype, dim, group, 32, counts, before, heads, query_heads, rotary, interleaved, rotary != 32)
    check_append(*args, counts, heads, query_heads, interleaved)


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
@pytest.mark.parametrize("rotary", [32, 64])
def test_append_of_many_tokens_flags_what_has_no_place(cuda, bits, dtype, dim, group, rotary):
    """Rows beyond the table or in pages that do not exist, and positions outside the rotary table, among 1,100 tokens:
    their rows stay as they were, the others are written."""
    import torch

    from code_for_iclr27_b200.paged import paged_append, rotary_table

    tokens = 1100
    case = Case(cuda, bits, dtype, dim, group, 64, 2, [tokens, tokens - 3], seed=5)
    case.table[0, 2] = -1
    case.table[1, 16] = 2 ** 30
    rows = queries_of(case, [tokens], 1)
    positions = torch.arange(tokens, device=cuda) % 50
    positions[700], positions[701], positions[9] = 50, -1, 2 ** 40
    before = case.pages.positions.clone()
    # (The second head's first three rows are negative.)
    paged_append(case.pages, case.table, case.lengths, rows, rows, positions, case.starts([tokens]), case.flag,
                 rotary_table(50, rotary, 10000.0, cuda), False, None)
    assert int(case.flag.item()) == 3
    want = before.cpu()
    for head, shift in ((0, 0), (1, 3)):
        for t in range(tokens):
            row = t - shift
            if row < 0 or t in (700, 701, 9):
                continue
            page = int(case.host_table[head, row // 64])
            if (head, row // 64) in ((0, 2), (1, 16)):
                continue
            want[page, row % 64] = float(t % 50)
    assert torch.equal(case.pages.positions.cpu(), want)


MANY = [(16, "bf16", 128, 0), (16, "f16", 64, 0), (4, "bf16", 128, 32), (4, "f16", 128, 64), (4, "bf16", 128, 128), (4, "f16", 64, 32),
        (4, "bf16", 64, 64)]


@pytest.mark.parametrize("bits,dtype,dim,group", MANY)
@pytest.mark.parametrize("page", [16, 128])
def test_chunks_with_peaked_and_large_scores(cuda, bits, dtype, dim, group, page):
    """Scores of some hundreds: the running maximum moves all the time; a scale of their sign turned round, and zero."""
    case = Case(cuda, bits, dtype, dim, group, page, 1, [500, 77], seed=2, key_spread=8.0)
    queries = queries_of(case, [70, 70], 1, spread=8.0)
    for scale in (None, -0.5, 0.0):
        out, lse = case.attend(queries, [70, 70], scale=scale)
        case.check(queries, [70, 70], out, lse, scale=scale)


@pytest.mark.parametrize("bits,dtype,dim,group", MANY)
@pytest.mark.parametrize("large", [60.0, 4000.0, 15000.0])
def test_chunks_over_values_of_all_magnitudes(cuda, bits, dtype, dim, group, large):
    for spread in (lambda n: large * (np.arange(n) + 1.0) / max(n, 1), lambda n: np.where(np.arange(n) % 97 == 50, large, 1e-3)):
        case = Case(cuda, bits, dtype, dim, group, 32, 1, [700, 40], seed=13, value_spread=spread)
        queries = queries_of(case, [70, 70], 1)
        out, lse = case.attend(queries, [70, 70])
        case.check(queries, [70, 70], out, lse)


@pytest.mark.parametrize("bits,dtype,dim,group", MANY)
def test_chunks_of_tiny_and_huge_queries(cuda, bits, dtype, dim, group):
    case = Case(cuda, bits, dtype, dim, group, 32, 1, [200], seed=3)
    for factor in (1e-6, 1e-3, 3e4, 0.0) + ((1e30, 1e-30) if dtype == "bf16" else ()):
        queries = ((queries_of(case, [70], 2).float()).clamp(-2, 2) * factor).to(case.dtype)
        scale = case.dim ** -0.5 if factor < 1 else case.dim ** -0.5 / factor
        out, lse = case.attend(queries, [70], scale=scale)
        case.check(queries, [70], out, lse, scale=scale)


@pytest.mark.parametrize("bits,dtype,dim,group", MANY)
@pytest.mark.parametrize("page", [16, 64])
def test_chunks_strided_split_and_captured(cuda, bits, dtype, dim, group, page):
    """Queries as views of a joint projection and of a wider row; slots split over many blocks; a captured call."""
    import torch

    from code_for_iclr27_b200.paged import attention_workspace, paged_attention

    case = Case(cuda, bits, dtype, dim, group, page, 1, [9001, 300], seed=6)
    counts = [33, 40]
    queries = queries_of(case, counts, 4)
    workspace = attention_workspace(cuda)
    want, want_lse = case.attend(queries, counts, workspace=workspace)
    case.check(queries, counts, want, want_lse)
    joint = torch.zeros(73, 9, dim, dtype=queries.dtype, device=cuda)
    joint[:, 2:6] = queries
    odd = torch.zeros(73, 4, dim + 3, dtype=queries.dtype, device=cuda)
    odd[:, :, 1:1 + dim] = queries
    for view in (joint[:, 2:6], odd[:, :, 1:1 + dim], queries.transpose(0, 1).contiguous().transpose(0, 1)):
        out, lse = case.attend(view, counts, workspace=workspace)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    starts = case.starts(counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged_attention(case.pages, case.table, case.lengths, queries, starts, workspace, case.flag)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("bits,dtype,dim,group", MANY)
def test_a_chunk_over_a_key_that_is_not_a_number(cuda, bits, dtype, dim, group):
    """It reaches the queries that see its row and no other."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 16, 1, [150, 150], seed=8)
    poison_keys(case, 0, [149 - 20])
    out, lse = case.attend(queries_of(case, [70, 70], 1), [70, 70])
    sees = torch.zeros(140, dtype=torch.bool, device=cuda)
    sees[49:70] = True  # token i of 70 sees rows up to 80 + i
    assert torch.isnan(out[sees]).all() and torch.isnan(lse[sees]).all()
    assert torch.isfinite(out[~sees]).all() and torch.isfinite(lse[~sees]).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_step_serves_later_steps(cuda, bits):
    """A graph of a step's appends and attentions, replayed after each advance (counts shifting between the sequences,
    new pages among them), gives the bits of the same steps called directly on another cache."""
    import torch

    from code_for_iclr27_b200.paged import PagedCache, rotary_table
    from test_gpu_arena import make_packed

    packed = [make_packed(cuda, seed=s) for s in (1, 2)]
    page_size = 16 if bits == 4 else 64
    caches = [PagedCache(3, 2, 4, 128, 24 * 1024 // page_size, cuda, bits=bits, page_size=page_size, max_rows=1024)
              for _ in range(2)]
    rotary = rotary_table(2000, 128, 10000.0, cuda)
    joint = torch.zeros(3, 5, 16, 128, dtype=torch.bfloat16, device=cuda)
    position = torch.zeros(5, dtype=torch.int64, device=cuda)

    def step(cache):
        outs = []
        for layer in range(3):
            q, k, v = joint[layer].split([8, 4, 4], 1)
            outs.append(cache.attend(layer, cache.append(layer, k, v, position, rotary, queries=q)))
        return outs

    for cache in caches:
        for s in range(2):
            cache.load(s, packed[s])
    graph = held = None
    for number, counts in enumerate(([2, 3], [1, 4], [5, 0], [0, 5], [3, 2], [4, 1], [2, 3])):
        joint.copy_(torch.randn(joint.shape, generator=torch.Generator().manual_seed(number)))
        position.fill_(900 + number)
        for cache in caches:
            cache.advance(counts)
        want = step(caches[0])
        if graph is None:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = step(caches[1])
        fill_free_memory(cuda, [(3 + 8) * 4, 256, 512])  # what a step has let go of is used again
        graph.replay()
        torch.cuda.synchronize()
        for (out, lse), (want_out, want_lse) in zip(held, want):
            assert torch.isfinite(want_out).all()
            assert torch.equal(out, want_out) and torch.equal(lse, want_lse)
    for cache in caches:
        cache.check_flags()
    for s in range(2):
        for a, b in zip(caches[0].to_packed(s).layers, caches[1].to_packed(s).layers):
            assert torch.equal(a.keys, b.keys) and torch.equal(a.values, b.values) and torch.equal(a.positions, b.positions)


@pytest.mark.parametrize("dim,group", [(128, 32), (128, 64), (64, 32)])
@pytest.mark.parametrize("groups", [4, 14, 30, 70])
@pytest.mark.parametrize("size", [1.0, 1e-6])
@pytest.mark.parametrize("bad", [0, 1])
def test_a_value_group_that_is_not_a_number_leaves_the_others_alone(cuda, dim, group, groups, size, bad):
    """Rows with a group of channels that append held as NaN: those channels are NaN, the others keep compare's bound."""
    import torch

    rng = np.random.default_rng(7)
    case = Case(cuda, 4, "bf16", dim, group, 32, 1, [700, 40], seed=13)
    refill(case, lambda n: (rng.standard_normal((n, dim)), size * rng.standard_normal((n, dim))))
    queries = queries_of(case, [1, 1], groups)
    for slot, row in ((0, 3), (0, 650), (1, 39)):
        case.pages.value_scales[int(case.host_table[slot, row // 32]), row % 32, bad] = float("nan")
    out, lse = case.attend(queries, [1, 1])
    at = slice(bad * group, (bad + 1) * group)
    assert torch.isnan(out[:, :, at]).all() and torch.isfinite(lse).all()
    out[:, :, at] = 0
    for slot in range(2):
        case.rows[slot][1][:, at] = 0
    compare(case, queries, [1, 1], out, lse)
