"""The paged cache's operators (paged.py, csrc/paged_append.cu, csrc/paged_attention.cu) against plain forms.

Appended rows are compared bit for bit with the same float32 steps in numpy (each product and sum rounded once), and the
4-bit values with the nearest of their sixteen levels in 64 bits.  Attention is compared with float64: with u the unit of
the type that the weights p are held in (2^-11 f16, 2^-8 bf16; 4-bit rows always take f16) and d a bound of a float32
score's error, an output may be off by (2 u + 4 d) sum p |v| plus its own rounding; for a 4-bit row |v| is taken as
8 scale + |offset|, which its code and offset contribute apart.  Every row and page that a call may not use holds NaN.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def torch_dtype(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def quantise(x, group):
    """float32 [..., D] -> codes uint8 [..., D] (unpacked), scale and offset float16 [..., D / group]."""
    x = np.asarray(x, dtype=np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        scale = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
        step = scale.astype(np.float32)
        offset = (lo + np.float32(8) * step).astype(np.float16)
        fine = np.isfinite(scale) & np.isfinite(offset)
        inverse = np.where(step > 0, np.float32(1) / np.where(step > 0, step, np.float32(1)), np.float32(0))
        level = np.rint((g - offset.astype(np.float32)[..., None]) * inverse[..., None]) + np.float32(8)
        code = np.where(fine[..., None], np.clip(level, 0, 15), 0).astype(np.uint8)
    nan = np.float16(np.nan)
    return code.reshape(x.shape), np.where(fine, scale, nan), np.where(fine, offset, nan)


def rotate(x, table, positions, interleaved):
    """float32 [tokens, heads, D], every product and sum rounded once."""
    x = np.array(x, dtype=np.float32)
    R = table.shape[1]
    cos, sin = table[positions][:, None, :R // 2], table[positions][:, None, R // 2:]
    first = np.arange(R // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first] = a * cos - b * sin
    x[..., second] = b * cos + a * sin
    return x


class Case:
    """Pages with every unused byte poisoned, a shuffled page table (a strided view), and the rows' float64 values."""

    def __init__(self, device, bits, dtype, dim, group, page, heads, lengths, seed=0, spare=3, key_spread=1.0,
                 value_spread=None):
        import torch

        from code_for_iclr27_b200.paged import Pages

        self.device, self.bits, self.dim, self.group, self.page, self.heads = device, bits, dim, group, page, heads
        self.dtype = torch_dtype(dtype)
        self.rng = np.random.default_rng(seed)
        self.slots = len(lengths)
        need = [-(-n // page) for n in lengths]
        total = sum(need) + spare
        order = self.rng.permutation(total)
        width = max(need, default=0) + 1
        table = np.full((self.slots, width + 2), 2 ** 30, dtype=np.int32)  # unused entries name no page
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.host_table = table
        self.table = torch.from_numpy(table).to(device)[:, :width]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.flag = torch.zeros(1, dtype=torch.int32, device=device)
        if bits == 16:
            keys = torch.full((total, page, dim), float("nan"), dtype=self.dtype)
            values = keys.clone()
            scales = (None, None)
        else:
            keys = torch.full((total, page, dim // 2), 0xff, dtype=torch.uint8)
            values = keys.clone()
            scales = tuple(torch.full((total, page, dim // group, 2), float("nan"), dtype=torch.float16) for _ in range(2))
        positions = torch.full((total, page), -7.0)
        self.rows, self.sizes = [], []  # per slot: float64 keys, values; and the sizes that bound a value's error
        for s, n in enumerate(lengths):
            held = []
            for side, pool in enumerate((keys, values)):
                x = self.rng.standard_normal((n, dim)).astype(np.float32) * (key_spread if side == 0 else 1.0)
                if side == 1 and value_spread is not None:
                    x = np.clip(x * value_spread(n)[:, None].astype(np.float32), -65000, 65000)  # finite in float16
                pages, lines = table[s, np.arange(n) // page], np.arange(n) % page
                if bits == 16:
                    x = torch.from_numpy(x).to(self.dtype)
                    pool[pages, lines] = x
                    held.append((x.double().numpy(), np.abs(x.double().numpy())))
                    continue
                code, scale, offset = quantise(x, group)
                pool[pages, lines] = torch.from_numpy(code[:, 0::2] | (code[:, 1::2] << 4))
                scales[side][pages, lines] = torch.from_numpy(np.stack((scale, offset), -1))
                wide = [np.repeat(v.astype(np.float64), group, -1) for v in (scale, offset)]
                held.append((wide[1] + wide[0] * (code.astype(np.float64) - 8), 8 * wide[0] + np.abs(wide[1])))
            self.rows.append((held[0][0], held[1][0]))
            self.sizes.append(held[1][1])
        self.pages = Pages(keys.to(device), values.to(device), positions.to(device),
                           *(None if t is None else t.to(device) for t in scales))

    def starts(self, counts):
        import torch

        return torch.from_numpy(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)).to(self.device)

    def attend(self, queries, counts, causal=True, scale=None, workspace=None):
        from code_for_iclr27_b200.paged import attention_workspace, paged_attention

        workspace = attention_workspace(self.device) if workspace is None else workspace
        return paged_attention(self.pages, self.table, self.lengths, queries, self.starts(counts), workspace, self.flag,
                               scale, causal)

    def check(self, queries, counts, out, lse, causal=True, scale=None):
        """Compare with float64 at the bound in the module's docstring."""
        dim, heads = self.dim, self.heads
        groups = queries.shape[1] // heads
        scale = dim ** -0.5 if scale is None else scale
        q = queries.double().cpu().numpy()
        got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        name = "f16" if out.dtype == torch_dtype("f16") else "bf16"
        unit = UNIT["f16"] if self.bits == 4 else UNIT[name]
        lengths = self.lengths.cpu().tolist()
        t = 0
        for s, n in enumerate(counts):
            for i in range(n):
                for h in range(heads):
                    slot = s * heads + h
                    keys, values = self.rows[slot]
                    seen = max(0, lengths[slot] - n + i + 1) if causal else lengths[slot]
                    at = slice(h * groups, (h + 1) * groups)
                    if seen == 0:
                        assert (got[t, at] == 0).all() and np.isneginf(got_lse[t, at]).all(), (s, i, h)
                        continue
                    scores = scale * q[t, at] @ keys[:seen].T
                    top = scores.max(-1, keepdims=True)
                    weight = np.exp(scores - top)
                    total = weight.sum(-1, keepdims=True)
                    want, want_lse = weight @ values[:seen] / total, (top + np.log(total))[:, 0]
                    d = (dim + 16) * 2.0 ** -23 * abs(scale) * (np.abs(q[t, at]) @ np.abs(keys[:seen]).T).max()
                    mass = weight @ self.sizes[slot][:seen] / total
                    # Weights below f16's normal range keep 2^-25 of the running maximum.
                    small = 2.0 ** -22 * seen / total
                    bound = (2 * unit + 4 * d + 2.0 ** -16) * mass + small + UNIT[name] * np.abs(want) + 1e-7
                    assert (np.abs(got[t, at] - want) <= bound).all(), (s, i, h, np.abs(got[t, at] - want).max(), bound.min())
                    assert (np.abs(got_lse[t, at] - want_lse) <= 2 * d + 2.0 ** -20 * (1 + np.abs(want_lse))).all(), (s, i, h)
                t += 1
        assert int(self.flag.item()) == 0


def queries_of(case, counts, groups, spread=1.0, seed=5):
    import torch

    g = torch.Generator().manual_seed(seed)
    total = sum(counts)
    return (spread * torch.randn(total, case.heads * groups, case.dim, generator=g)).to(case.dtype).to(case.device)


FORMATS = [(16, "bf16", 128, 0), (16, "f16", 128, 0), (16, "bf16", 64, 0), (16, "f16", 64, 0), (4, "bf16", 128, 32),
           (4, "f16", 128, 64), (4, "bf16", 128, 128), (4, "bf16", 64, 32), (4, "f16", 64, 64)]
# Zero, one, and both sides of a page's, a tile's and several tiles' end.
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300, 511, 513, 1024]


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_decode_lengths(cuda, bits, dtype, dim, group, page):
    """One token a sequence, every length, 4 query heads a KV head."""
    case = Case(cuda, bits, dtype, dim, group, page, 2, LENGTHS, seed=page)
    counts = [1] * (len(LENGTHS) // 2)
    queries = queries_of(case, counts, 4, spread=2.0)
    out, lse = case.attend(queries, counts)
    case.check(queries, counts, out, lse)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("groups", [1, 3, 7, 8, 12, 33])
def test_attention_query_groups(cuda, bits, dtype, dim, group, groups):
    case = Case(cuda, bits, dtype, dim, group, 32, 1, [70, 0, 333], seed=groups)
    queries = queries_of(case, [1, 1, 1], groups)
    out, lse = case.attend(queries, [1, 1, 1])
    case.check(queries, [1, 1, 1], out, lse)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("counts", [[2, 0, 5], [7, 1, 3], [33, 40, 1], [130, 0, 64], [1, 257, 2]])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_several_tokens(cuda, bits, dtype, dim, group, counts, causal):
    """Ragged token counts, none among them; slots shorter than the step's tokens, whose first queries see nothing."""
    lengths = [90, 3, 64, 1, 350, 200]
    case = Case(cuda, bits, dtype, dim, group, 64, 2, lengths, seed=sum(counts))
    queries = queries_of(case, counts, 3)
    out, lse = case.attend(queries, counts, causal=causal)
    case.check(queries, counts, out, lse, causal=causal)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
def test_attention_long_and_ragged(cuda, bits, dtype, dim, group):
    """Slots long enough to be split over many blocks beside short ones; the same call twice gives the same bits."""
    import torch

    from code_for_iclr27_b200.paged import attention_workspace

    lengths = [20011, 5, 0, 7000, 1, 12345]
    case = Case(cuda, bits, dtype, dim, group, 128, 2, lengths, seed=9)
    queries = queries_of(case, [1, 1, 1], 5, spread=3.0)
    workspace = attention_workspace(cuda)
    out, lse = case.attend(queries, [1, 1, 1], workspace=workspace)
    case.check(queries, [1, 1, 1], out, lse)
    for _ in range(3):
        again, again_lse = case.attend(queries, [1, 1, 1], workspace=workspace)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("page,groups", [(16, 2), (64, 12), (128, 30)])
def test_attention_many_tiles_a_block(cuda, bits, dtype, dim, group, page, groups):
    """Enough rows that every block's ring of tiles goes round many times, over ends of slots."""
    lengths = [3000 + 997 * (i % 5) + i for i in range(64)]
    lengths[7], lengths[20], lengths[21] = 0, 1, 40000
    case = Case(cuda, bits, dtype, dim, group, page, 4, lengths, seed=page)
    queries = queries_of(case, [1] * 16, groups)
    out, lse = case.attend(queries, [1] * 16)
    case.check(queries, [1] * 16, out, lse)


@pytest.mark.parametrize("bits,dim,group", [(16, 128, 0), (4, 128, 32), (4, 128, 64), (4, 128, 128), (4, 64, 64)])
@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_attention_long_sums_keep_precision(cuda, bits, dim, group, tokens):
    """Nearly even weights over 33,000 rows: the output is a small rest of large sums.  In the 2-norm it may be off by
    the output's rounding (2^-9) and the weights' (2^-9 more for bf16 weights, 2^-12 for f16)."""
    case = Case(cuda, bits, "bf16", dim, group, 128, 1, [33000], seed=17)
    queries = queries_of(case, [tokens], 4, spread=0.25)
    out, _ = case.attend(queries, [tokens])
    keys, values = case.rows[0]
    q = queries.double().cpu().numpy()
    want = np.empty(q.shape)
    for i in range(tokens):
        seen = 33000 - tokens + i + 1
        scores = dim ** -0.5 * q[i] @ keys[:seen].T
        weight = np.exp(scores - scores.max(-1, keepdims=True))
        want[i] = weight @ values[:seen] / weight.sum(-1, keepdims=True)
    off = np.linalg.norm(out.double().cpu().numpy() - want) / np.linalg.norm(want)
    assert off <= 2.0 ** -9 + (2.0 ** -12 if bits == 4 else 2.0 ** -9), off


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
def test_attention_window_of_queries(cuda, bits, dtype, dim, group):
    """A chunk of 250 tokens at the end of a longer slot."""
    case = Case(cuda, bits, dtype, dim, group, 64, 1, [1500], seed=4)
    queries = queries_of(case, [250], 4, spread=2.0)
    out, lse = case.attend(queries, [250])
    case.check(queries, [250], out, lse)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
def test_attention_peaked_and_large_scores(cuda, bits, dtype, dim, group):
    """Scores of some hundreds, increasing and decreasing along the rows: the running maximum moves all the time; and a
    scale of their sign turned round, and of zero."""
    case = Case(cuda, bits, dtype, dim, group, 32, 2, [500, 77], seed=2, key_spread=8.0)
    queries = queries_of(case, [1], 6, spread=8.0)
    for scale in (None, -0.5, 0.0):
        out, lse = case.attend(queries, [1], scale=scale)
        case.check(queries, [1], out, lse, scale=scale)


@pytest.mark.parametrize("bits,dtype,dim,group", FORMATS)
@pytest.mark.parametrize("large", [60.0, 4000.0, 15000.0])
def test_attention_value_magnitudes(cuda, bits, dtype, dim, group, large):
    """Values whose 4-bit scales grow along the rows, up to near float16's largest; few large ones among small ones."""
    rising = lambda n: large * (np.arange(n) + 1.0) / max(n, 1)  # noqa: E731
    some = lambda n: np.where(np.arange(n) % 97 == 50, large, 1e-3)  # noqa: E731
    for spread in (rising, some):
        case = Case(cuda, bits, dtype, dim, group, 32, 1, [700, 40], seed=13, value_spread=spread)
        queries = queries_of(case, [1, 1], 4)
        out, lse = case.attend(queries, [1, 1])
        case.check(queries, [1, 1], out, lse)


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "f16", 128, 0), (16, "bf16", 64, 0), (4, "bf16", 128, 64), (4, "f16", 64, 32)])
def test_attention_query_magnitudes(cuda, bits, dtype, dim, group):
    """Tiny and huge queries (subnormal float16, beyond float16 in bfloat16), zero ones, and one large channel."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [200], seed=3)
    for factor in (1e-6, 1e-3, 3e4, 0.0) + ((1e30, 1e-30) if dtype == "bf16" else ()):
        queries = (queries_of(case, [2], 4).float() * 1.0).clamp(-2, 2) * factor
        queries[:, :, 3] *= 0.5
        queries = queries.to(case.dtype)
        scale = case.dim ** -0.5 if factor == 0 or factor < 1 else case.dim ** -0.5 / factor
        out, lse = case.attend(queries, [2], scale=scale)
        case.check(queries, [2], out, lse, scale=scale)
    queries = queries_of(case, [2], 4)
    queries[:, :, 5] = 64.0
    out, lse = case.attend(queries, [2])
    case.check(queries, [2], out, lse)
    assert not torch.isnan(out).any()


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "bf16", 128, 0), (4, "bf16", 128, 64)])
def test_attention_strides_and_streams(cuda, bits, dtype, dim, group):
    """Queries as a view of a joint projection, as an unaligned view, with a padded last dimension; on a stream of its own."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 64, 2, [100, 40, 257, 9], seed=6)
    counts = [2, 3]
    queries = queries_of(case, counts, 4)
    want, want_lse = case.attend(queries, counts)
    case.check(queries, counts, want, want_lse)
    joint = torch.zeros(5, 13, dim, dtype=queries.dtype, device=cuda)
    joint[:, 2:10] = queries
    odd = torch.zeros(5, 8, dim + 3, dtype=queries.dtype, device=cuda)
    odd[:, :, 1:1 + dim] = queries
    apart = torch.zeros(5, 8, dim, 2, dtype=queries.dtype, device=cuda)
    apart[..., 1] = queries
    for view in (joint[:, 2:10], odd[:, :, 1:1 + dim], apart[..., 1], queries.transpose(0, 1).contiguous().transpose(0, 1)):
        out, lse = case.attend(view, counts)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = case.attend(queries, counts)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "f16", 128, 0), (4, "f16", 128, 64), (4, "f16", 64, 32)])
def test_attention_rows_that_are_not_finite(cuda, bits, dtype, dim, group):
    """A NaN key or value row reaches the queries that see it and no other."""
    import torch

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [150, 150], seed=8)
    pool = case.pages.keys if bits == 16 else case.pages.key_scales
    page, line = int(case.host_table[0, 149 // 32]), 149 % 32
    pool[page, line] = float("nan")
    counts = [3, 3]
    queries = queries_of(case, counts, 2)
    out, lse = case.attend(queries, counts)
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    others = [0, 1, 3, 4, 5]
    assert torch.isfinite(out[others]).all() and torch.isfinite(lse[others]).all()


@pytest.mark.parametrize("bits,dtype,dim,group", [(16, "bf16", 128, 0), (4, "bf16", 128, 64)])
def test_attention_flags_rows_without_pages(cuda, bits, dtype, dim, group):
    """A page id outside the pages, or a length beyond the table, sets the flag; other slots are computed."""
    case = Case(cuda, bits, dtype, dim, group, 32, 1, [100, 60, 64], seed=8)
    queries = queries_of(case, [1, 1, 1], 4)
    good, good_lse = case.attend(queries, [1, 1, 1])
    for entry in (-1, 2 ** 30, -2 ** 31):
        case.table[1, 1] = entry
        out, lse = case.attend(queries, [1, 1, 1])
        assert int(case.flag.item()) == 1
        case.flag.zero_()
        assert (out[0] == good[0]).all() and (out[2] == good[2]).all()
    case.table[1, 1] = int(case.host_table[1, 1])
    for length in (case.table.shape[1] * 32 + 1, 2 ** 31 - 1):
        case.lengths[1] = length
        out, lse = case.attend(queries, [1, 1, 1])
        assert int(case.flag.item()) == 1
        case.flag.zero_()
        assert (out[0] == good[0]).all() and (out[2] == good[2]).all()
    case.lengths[1] = -5
    out, lse = case.attend(queries, [1, 1, 1])
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_offsets_beyond_32_bits(cuda):
    """Pages whose byte and element offsets pass 2^32 and 2^31: append, attention and (4-bit) read back."""
    import torch

    from code_for_iclr27_b200.paged import Pages, attention_workspace, paged_append, paged_attention, paged_read

    for bits, pages in ((16, 140_000), (4, 540_000)):
        pool = Pages.empty(pages, 128, 128, cuda, torch.bfloat16, bits, 128)
        page_ids = [pages - 1, pages // 2 + 1, 0]
        table = torch.tensor([page_ids], dtype=torch.int32, device=cuda)
        n = 300
        g = torch.Generator().manual_seed(1)
        keys, values = (torch.randn(n, 1, 128, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
        lengths = torch.tensor([n], dtype=torch.int32, device=cuda)
        starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        flag = torch.zeros(1, dtype=torch.int32, device=cuda)
        paged_append(pool, table, lengths, keys, values, torch.arange(n, device=cuda), starts, flag)
        row_starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        back_k, back_v, where = paged_read(pool, table, torch.zeros(1, dtype=torch.int32, device=cuda), row_starts, n,
                                           torch.float32, flag)
        assert torch.equal(where, torch.arange(n, device=cuda).float())
        if bits == 16:
            assert torch.equal(back_k, keys[:, 0].float()) and torch.equal(back_v, values[:, 0].float())
        query = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16).to(cuda)
        one = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
        out, lse = paged_attention(pool, table, lengths, query, one, attention_workspace(cuda), flag)
        scores = query[0].double() @ back_k.double().T / 128 ** 0.5
        want = scores.softmax(-1) @ back_v.double()
        assert (out[0].double() - want).abs().max() <= 2 ** -7 * back_v.abs().max().item()
        assert (lse[0].double() - scores.logsumexp(-1)).abs().max() <= 1e-4
        assert int(flag.item()) == 0
        del pool


# ------------------------------------------------------------------- append

APPEND = [(16, "bf16", 128, 0), (16, "f16", 64, 0), (4, "bf16", 128, 32), (4, "f16", 128, 64), (4, "bf16", 128, 128),
          (4, "f16", 64, 32), (4, "bf16", 64, 64)]


def run_append(cuda, bits, dtype, dim, group, page, counts, before, heads, query_heads, rotary_dim, interleaved, fused,
               scale=1.0, seed=0, edit=None):
    """Append random rows; returns (case, host inputs, the pages' host copies before, rotated queries)."""
    import torch

    from code_for_iclr27_b200.paged import paged_append, rotary_table

    lengths = [b + counts[s // heads] for s, b in enumerate(before)]
    case = Case(cuda, bits, dtype, dim, group, page, heads, lengths, seed=seed)
    total = sum(counts)
    g = torch.Generator().manual_seed(seed + 1)
    wide = query_heads + 2 * heads
    joint = (scale * torch.randn(total, wide, dim, generator=g)).to(case.dtype)
    if edit is not None:
        edit(joint, query_heads, heads)
    positions = torch.randint(0, 50, (total,), generator=g)
    rotary = rotary_table(50, rotary_dim, 10000.0, cuda) if rotary_dim else None
    on_gpu = joint.to(cuda)
    parts = [on_gpu[:, :query_heads], on_gpu[:, query_heads:query_heads + heads], on_gpu[:, query_heads + heads:]]
    if not fused:
        parts = [p.contiguous() for p in parts]
    old = [t.clone() for t in (case.pages.keys, case.pages.values, case.pages.positions) +
           ((case.pages.key_scales, case.pages.value_scales) if bits == 4 else ())]
    turned = paged_append(case.pages, case.table, case.lengths, parts[1], parts[2], positions.to(cuda), case.starts(counts),
                          case.flag, rotary, interleaved, parts[0] if query_heads else None)
    return case, joint, positions.numpy(), None if rotary is None else rotary.cpu().numpy(), old, turned


def check_append(case, joint, positions, rotary, old, turned, counts, heads, query_heads, interleaved):
    """The whole pages, bit for bit: new rows as the float32 steps give them, everything else as it was."""
    import torch

    rows = joint.float().numpy()
    q, k, v = rows[:, :query_heads], rows[:, query_heads:query_heads + heads], rows[:, query_heads + heads:]
    if rotary is not None:
        with np.errstate(all="ignore"):
            q, k = rotate(q, rotary, positions, interleaved), rotate(k, rotary, positions, interleaved)
    want = [t.cpu() for t in old]
    lengths = case.lengths.cpu().tolist()
    t = 0
    for s, n in enumerate(counts):
        for i in range(n):
            for h in range(heads):
                row = lengths[s * heads + h] - n + i
                at = (int(case.host_table[s * heads + h, row // case.page]), row % case.page)
                want[2][at] = float(positions[t])
                for side, x in enumerate((k[t, h], v[t, h])):
                    if case.bits == 16:
                        want[side][at] = torch.from_numpy(x).to(case.dtype)
                        continue
                    code, scale, offset = quantise(x, case.group)
                    want[side][at] = torch.from_numpy(code[0::2] | (code[1::2] << 4))
                    want[3 + side][at] = torch.from_numpy(np.stack((scale, offset), -1))
            t += 1
    got = [x.cpu() for x in (case.pages.keys, case.pages.values, case.pages.positions) +
           ((case.pages.key_scales, case.pages.value_scales) if case.bits == 4 else ())]
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0)), i
    if query_heads:
        b = torch.from_numpy(q).to(case.dtype)
        assert torch.equal(torch.nan_to_num(turned.cpu().float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))
    else:
        assert turned is None
    assert int(case.flag.item()) == 0


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (16, False), (16, True), (64, False), (64, True), (32, False), (128, True), (128, False)])
@pytest.mark.parametrize("fused", [True, False])
def test_append_rotations(cuda, bits, dtype, dim, group, rotary, interleaved, fused):
    if rotary > dim:
        pytest.skip("rotates more channels than the head has")
    counts, heads = [3, 0, 1, 18], 2
    before = [0, 5, 1, 1, 63, 64, 14, 100]
    args = run_append(cuda, bits, dtype, dim, group, 16, counts, before, heads, 5, rotary, interleaved, fused)
    check_append(*args, counts, heads, 5, interleaved)


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("counts,heads,query_heads", [([1] * 9, 3, 0), ([200, 1], 1, 1), ([1], 8, 32), ([0, 0, 77], 4, 28)])
def test_append_sizes(cuda, bits, dtype, dim, group, page, counts, heads, query_heads):
    before = [(37 * i) % 150 for i in range(len(counts) * heads)]
    args = run_append(cuda, bits, dtype, dim, group, page, counts, before, heads, query_heads, 64, False, True, seed=page)
    check_append(*args, counts, heads, query_heads, False)


@pytest.mark.parametrize("bits,dtype,dim,group", [a for a in APPEND if a[0] == 4])
def test_append_values_that_quantise_badly(cuda, bits, dtype, dim, group):
    """Constant and zero groups, NaN, infinities, the type's largest and smallest values, and values far from zero."""
    import torch

    def edit(joint, query_heads, heads):
        k = joint[:, query_heads:]
        k[0] = 0
        k[1] = 1.5
        k[2, :, 3] = float("nan")
        k[3, :, 5] = float("inf")
        k[4, :, 5] = -float("inf")
        k[5] = float("inf")
        k[6] = torch.finfo(joint.dtype).max
        k[7] = torch.finfo(joint.dtype).tiny
        k[8] = 1000 + 0.01 * k[8]
        k[9] = -k[8]
        k[10, :, 0] = 60000.0
        k[11, :, 0] = -60000.0
        k[12] *= 1e-6
        k[13, :, ::2] = -0.0
        k[13, :, 1::2] = 0.0

    args = run_append(cuda, bits, dtype, dim, group, 16, [16], [3, 3], 2, 2, 0, False, True, edit=edit)
    check_append(*args, [16], 2, 2, False)


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
def test_append_flags_what_has_no_place(cuda, bits, dtype, dim, group):
    """Rows without a page and positions outside the table leave the pages as they were and set their bits."""
    import torch

    from code_for_iclr27_b200.paged import paged_append, rotary_table

    case = Case(cuda, bits, dtype, dim, group, 16, 1, [20, 20, 20])
    before = [case.pages.keys.clone(), case.pages.positions.clone()]
    rows = torch.randn(3, 1, dim).to(case.dtype).to(cuda)
    rotary = rotary_table(50, 32, 10000.0, cuda)
    starts = case.starts([1, 1, 1])
    same = lambda a, b: torch.equal(torch.nan_to_num(a.float(), nan=9.0), torch.nan_to_num(b.float(), nan=9.0))  # noqa: E731

    def append(lengths, positions, expected):
        paged_append(case.pages, case.table, torch.tensor(lengths, dtype=torch.int32, device=cuda), rows, rows,
                     torch.tensor(positions, device=cuda), starts, case.flag, rotary, False, rows)
        assert int(case.flag.item()) == expected
        case.flag.zero_()
        assert same(case.pages.keys, before[0]) and same(case.pages.positions, before[1])

    append([0, -1, 1000], [0, 1, 2], 1)  # no row, a negative one, one beyond the table
    append([40, 2 ** 31 - 1, -2 ** 31], [0, 1, 2], 1)  # an entry that names no page
    append([20, 20, 20], [50, -1, 2 ** 40], 2)
    append([20, 0, 20], [50, 3, -9], 3)


@pytest.mark.parametrize("bits,dtype,dim,group", APPEND)
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_read_rows(cuda, bits, dtype, dim, group, out):
    """Slots from any first row, empty ones among them; float32 values are the held ones, others rounded once."""
    import torch

    from code_for_iclr27_b200.paged import paged_read

    case = Case(cuda, bits, dtype, dim, group, 32, 1, [70, 0, 1, 300, 33, 32], seed=11)
    case.pages.positions.copy_(torch.arange(case.pages.positions.numel(), device=cuda).view_as(case.pages.positions))
    first, take = [10, 0, 0, 299, 31, 0], [60, 0, 1, 1, 2, 32]
    starts = np.concatenate(([0], np.cumsum(take)))
    kind = torch.float32 if out == "f32" else torch_dtype(out)
    keys, values, positions = paged_read(case.pages, case.table, torch.tensor(first, dtype=torch.int32, device=cuda),
                                         torch.from_numpy(starts.astype(np.int32)).to(cuda), int(starts[-1]), kind, case.flag)
    assert keys.dtype == kind and values.dtype == kind and int(case.flag.item()) == 0
    for side, got in enumerate((keys, values)):
        want = np.concatenate([case.rows[s][side][a:a + n] for s, (a, n) in enumerate(zip(first, take))])
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(kind))
    where = np.concatenate([case.host_table[s, np.arange(a, a + n) // 32].astype(np.int64) * 32 + np.arange(a, a + n) % 32
                            for s, (a, n) in enumerate(zip(first, take))])
    assert torch.equal(positions.cpu(), torch.from_numpy(where).float())
    keys, _, _ = paged_read(case.pages, case.table, torch.tensor(first, dtype=torch.int32, device=cuda),
                            torch.zeros(7, dtype=torch.int32, device=cuda), 0, kind, case.flag)
    assert keys.shape == (0, dim)
    first[3] = 320  # beyond the slot's pages
    paged_read(case.pages, case.table, torch.tensor(first, dtype=torch.int32, device=cuda),
               torch.from_numpy(starts.astype(np.int32)).to(cuda), int(starts[-1]), kind, case.flag)
    assert int(case.flag.item()) == 1


def test_refusals(cuda):
    """Arguments that do not fit raise before anything is launched, with the operator's message."""
    import torch

    from code_for_iclr27_b200.paged import Pages, attention_workspace, paged_append, paged_attention, paged_read

    case = Case(cuda, 4, "bf16", 128, 64, 16, 2, [20, 20])
    p, starts, flag, ws = case.pages, case.starts([1]), case.flag, attention_workspace(cuda)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device=cuda)
    pos = torch.zeros(1, dtype=torch.int64, device=cuda)

    def refused(match, call):
        with pytest.raises(RuntimeError, match=match):
            call()

    attend = lambda pages=p, table=case.table, lengths=case.lengths, q=q, s=starts, w=ws, f=flag, **k: paged_attention(pages, table, lengths, q, s, w, f, **k)  # noqa: E731
    append = lambda pages=p, table=case.table, lengths=case.lengths, k=k, v=k, pos=pos, s=starts, f=flag, r=None, q=None: paged_append(pages, table, lengths, k, v, pos, s, f, r, False, q)  # noqa: E731
    refused("contiguous CUDA", lambda: attend(lengths=case.lengths.cpu()))
    refused("int32", lambda: attend(lengths=case.lengths.long()))
    refused("int32", lambda: attend(table=case.table.long()))
    refused("multiple", lambda: attend(q=q[:, :3]))
    refused("multiple", lambda: attend(q=q[:, :1]))
    refused("queries must be", lambda: attend(q=q.float()))
    refused("queries must be", lambda: attend(q=q[:, :, :64]))
    refused("workspace", lambda: attend(w=ws[:1000]))
    refused("scale", lambda: attend(scale=float("nan")))
    refused("heads rows", lambda: attend(s=case.starts([1, 0, 0])))
    refused("flag", lambda: attend(f=flag.float()))
    refused("uint8", lambda: attend(pages=Pages(p.keys.to(torch.int8), p.values.to(torch.int8), p.positions, p.key_scales, p.value_scales)))
    refused("both", lambda: attend(pages=Pages(p.keys, p.values, p.positions, p.key_scales, None)))
    refused("16-bit|float16 or bfloat16", lambda: attend(pages=Pages(p.keys, p.values, p.positions)))
    refused("page size", lambda: attend(pages=Pages(p.keys[:, :8].contiguous(), p.values[:, :8].contiguous(), p.positions[:, :8].contiguous(),
                                                    p.key_scales[:, :8].contiguous(), p.value_scales[:, :8].contiguous())))
    sixteen = Case(cuda, 16, "f16", 128, 0, 16, 2, [20, 20])
    refused("pages' type", lambda: paged_attention(sixteen.pages, sixteen.table, sixteen.lengths, q, starts, ws, flag))
    refused("pages' type", lambda: paged_append(sixteen.pages, sixteen.table, sixteen.lengths, k, k, pos, starts, flag))
    refused("differ", lambda: append(v=k[:, :1]))
    refused("new rows", lambda: append(k=k.float(), v=k.float()))
    refused("positions must be", lambda: append(pos=pos.int()))
    refused("rotary", lambda: append(r=torch.zeros(4, 24, device=cuda)))
    refused("rotary", lambda: append(r=torch.zeros(4, 144, device=cuda)))
    refused("rotary", lambda: append(r=torch.zeros(4, 64, device=cuda, dtype=torch.float64)))
    refused("tokens and dtype", lambda: append(q=q.half()))
    refused("token starts", lambda: append(s=case.starts([1, 1])))
    refused("f16, bf16 or f32", lambda: paged_read(p, case.table, case.lengths, torch.zeros(3, dtype=torch.int32, device=cuda), 4, torch.float64, flag))
    refused("row starts", lambda: paged_read(p, case.table, case.lengths, torch.zeros(2, dtype=torch.int32, device=cuda), 4, torch.bfloat16, flag))
    assert int(flag.item()) == 0


def test_nothing_to_do(cuda):
    """No tokens, no sequences, no pages."""
    import torch

    from code_for_iclr27_b200.paged import Pages, attention_workspace, paged_append, paged_attention

    case = Case(cuda, 4, "bf16", 128, 64, 16, 2, [20, 20])
    empty = torch.zeros(0, 4, 128, dtype=torch.bfloat16, device=cuda)
    ws = attention_workspace(cuda)
    out, lse = paged_attention(case.pages, case.table, case.lengths, empty, case.starts([0]), ws, case.flag)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    turned = paged_append(case.pages, case.table, case.lengths, empty[:, :2], empty[:, :2],
                          torch.zeros(0, dtype=torch.int64, device=cuda), case.starts([0]), case.flag, None, False, empty)
    assert turned.shape == (0, 4, 128)
    none = torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    out, lse = paged_attention(case.pages, none, none[:, 0].contiguous(), empty, case.starts([]), ws, case.flag)
    assert out.shape == (0, 4, 128)
    pages = Pages.empty(0, 16, 128, cuda, torch.bfloat16, 4, 64)
    table = torch.zeros(2, 0, dtype=torch.int32, device=cuda)
    query = torch.ones(1, 4, 128, dtype=torch.bfloat16, device=cuda)
    out, lse = paged_attention(pages, table, torch.zeros(2, dtype=torch.int32, device=cuda), query, case.starts([1]), ws, case.flag)
    assert (out == 0).all() and torch.isneginf(lse).all() and int(case.flag.item()) == 0


# -------------------------------------------------------------------- cache

@pytest.mark.parametrize("bits", [16, 4])
def test_paged_cache_through_its_life(cuda, bits):
    """Load two requests, decode steps with evictions between, release: rows, positions and attention as in the packed
    layout; the pages all come back."""
    import torch

    from code_for_iclr27_b200.paged import PagedCache, rotary_table
    from test_gpu_arena import make_packed

    packed = [make_packed(cuda, seed=s) for s in (1, 2)]
    cache = PagedCache(3, 2, 4, 128, 400, cuda, bits=bits, page_size=64, max_rows=2048)
    for s in range(2):
        cache.load(s, packed[s])
    rotary = rotary_table(2000, 128, 10000.0, cuda)
    g = torch.Generator().manual_seed(0)
    for step in range(5):
        counts = [1, 0] if step == 2 else [1, 3]
        cache.advance(counts)
        total = sum(counts)
        position = torch.full((total,), 1200 + step, device=cuda)
        for layer in range(3):
            rows = torch.randn(total, 16, 128, generator=g).to(torch.bfloat16).to(cuda)
            turned = cache.append(layer, rows[:, 8:12], rows[:, 12:], position, rotary, queries=rows[:, :8])
            out, lse = cache.attend(layer, turned)
            back = cache.to_packed(0, torch.float32).layers[layer]
            ends = np.cumsum(back.head_lens)
            for h in range(4):
                span = slice(ends[h] - back.head_lens[h], ends[h])
                k, v = back.keys[span].double(), back.values[span].double()
                scores = turned[0, 2 * h:2 * h + 2].double() @ k.T / 128 ** 0.5
                want = scores.softmax(-1) @ v
                assert (out[0, 2 * h:2 * h + 2].double() - want).abs().max() <= 2 ** -6 * v.abs().max().item()
    cache.check_flags()
    assert cache.lengths.cpu().numpy().tolist() == cache.rows.tolist()
    back = cache.to_packed(1)
    for layer in range(3):
        old, new = packed[1].layers[layer], back.layers[layer]
        assert new.head_lens == [n + 12 for n in old.head_lens] and new.prompt_lens == old.prompt_lens
        a, b = old.bounds(), new.bounds()
        for h in range(4):
            new_rows, old_rows = slice(b[h], b[h] + old.head_lens[h]), slice(a[h], a[h + 1])
            assert torch.equal(new.positions[new_rows], old.positions[old_rows])
            if bits == 16:
                assert torch.equal(new.keys[new_rows], old.keys[old_rows]) and torch.equal(new.values[new_rows], old.values[old_rows])
            else:  # half a step of a range of 16 levels, and the offset's and the output's rounding
                step = (old.keys[old_rows].float().unflatten(-1, (2, 64)).amax(-1) - old.keys[old_rows].float().unflatten(-1, (2, 64)).amin(-1)) / 15
                off = (new.keys[new_rows].float() - old.keys[old_rows].float()).abs().unflatten(-1, (2, 64)).amax(-1)
                assert (off <= 0.52 * step + 2 ** -7 * 5).all()
    # The audit's eviction on the packed rows, then back into pages.
    back.remove_positions({(0, 1): list(range(40)), (2, 3): [5, 9]})
    cache.load(1, back)
    again = cache.to_packed(1)
    for layer in range(3):
        assert again.layers[layer].head_lens == back.layers[layer].head_lens
        assert torch.equal(again.layers[layer].positions, back.layers[layer].positions)
        if bits == 16:
            assert torch.equal(again.layers[layer].keys, back.layers[layer].keys)
    for s in range(2):
        cache.release(s)
    assert cache.free_pages() == 400
    with pytest.raises(MemoryError):
        cache.advance([100000, 0])
    with pytest.raises(ValueError):
        cache.advance([1])
    assert cache.free_pages() == 400 and not cache.rows.any()


@pytest.mark.parametrize("bits,group", [(16, 64), (4, 32), (4, 128)])
def test_example(cuda, bits, group):
    """The example's whole path: audit, pages, decode steps, audit.  16-bit pages against themselves differ by nothing;
    4-bit rows, half a step of sixteen levels off each, by a tenth of the outputs' norm or so (a step is some 5 sigma /
    15, its error a step / sqrt(12): 0.1 sigma, in keys and values both)."""
    from code_for_iclr27_b200.paged_example import run

    result = run(layers=2, rows=1024, steps=4, bits=bits, group=group)
    assert result["rows"] == 2 * 8 * (1024 + 4) - result["evicted"]
    assert result["rows_after_audit"] == result["rows"] - 2 * 8
    assert result["relative_error"] == 0 if bits == 16 else 0 < result["relative_error"] < 0.3


def test_attention_in_a_cuda_graph(cuda):
    """A captured step (append and attention) replays on new inputs in place."""
    import torch

    from code_for_iclr27_b200.paged import attention_workspace, paged_append, paged_attention, rotary_table

    case = Case(cuda, 4, "bf16", 128, 64, 64, 2, [700, 650], seed=21)
    rotary, workspace, starts = rotary_table(1000, 128, 10000.0, cuda), attention_workspace(cuda), case.starts([1])
    joint = torch.zeros(1, 12, 128, dtype=torch.bfloat16, device=cuda)
    position = torch.tensor([699], device=cuda)

    def step():
        turned = paged_append(case.pages, case.table, case.lengths, joint[:, 8:10], joint[:, 10:], position, starts, case.flag,
                              rotary, False, joint[:, :8])
        return paged_attention(case.pages, case.table, case.lengths, turned, starts, workspace, case.flag)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        joint.copy_(torch.randn(1, 12, 128, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        direct = step()
        assert torch.equal(replayed[0], direct[0]) and torch.equal(replayed[1], direct[1])
    assert int(case.flag.item()) == 0
