"""The paged cache without a GPU: the C ABI's refusals (each returns before any CUDA call) and page memory's checks."""
import ctypes

import pytest

from code_for_iclr27_b200 import abi
from code_for_iclr27_b200.paged import WORKSPACE_BYTES, Pages

LIB = abi.library()
ADDRESS = 1 << 20  # stands for device memory that no refused call touches


def pages(**changes):
    p = abi.Pages(keys=ADDRESS, values=ADDRESS, key_scales=ADDRESS, value_scales=ADDRESS, positions=ADDRESS, pages=4,
                  page_size=64, dimension=128, group=64, dtype=abi.BF16)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


def rows(data=ADDRESS, token=1024, head=128):
    return ctypes.byref(abi.Rows(data, token, head))


def append(p=None, width=4, stride=4, heads=2, tokens=3, sequences=1, k=None, v=None, q=None, query_heads=0, rotary=None,
           rotary_positions=0, rotary_dim=0, out=None, dtype=abi.BF16, flag=ADDRESS, lengths=ADDRESS):
    return LIB.lrk_paged_append(pages() if p is None else p, ADDRESS, stride, width, lengths, sequences, heads, ADDRESS,
                                tokens, rows() if k is None else k, rows() if v is None else v, ADDRESS, rotary,
                                rotary_positions, rotary_dim, 0, q, query_heads, out, dtype, flag, None)


def attend(p=None, width=4, stride=4, heads=2, tokens=3, sequences=1, q=None, query_heads=8, scale=0.1, out=ADDRESS,
           dtype=abi.BF16, workspace=ADDRESS, size=WORKSPACE_BYTES, flag=ADDRESS):
    return LIB.lrk_paged_attention(pages() if p is None else p, ADDRESS, stride, width, ADDRESS, sequences, heads, ADDRESS,
                                   tokens, rows() if q is None else q, query_heads, scale, 1, out, ADDRESS, dtype,
                                   workspace, size, flag, None)


def read(p=None, width=4, stride=4, slots=2, count=5, keys=ADDRESS, dtype=abi.BF16, flag=ADDRESS):
    return LIB.lrk_paged_read(pages() if p is None else p, ADDRESS, stride, width, ADDRESS, ADDRESS, slots, count, keys,
                              ADDRESS, ADDRESS, dtype, flag, None)


def test_workspace_size():
    assert LIB.lrk_paged_attention_workspace_bytes() == WORKSPACE_BYTES


@pytest.mark.parametrize("call", [append, attend, read])
def test_pages_are_checked(call):
    for changes in (dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(group=16), dict(group=96),
                    dict(dimension=64, group=128), dict(group=0, dtype=abi.F32), dict(keys=None), dict(values=None),
                    dict(positions=None), dict(key_scales=None), dict(value_scales=None), dict(pages=-1),
                    dict(pages=1 << 31), dict(keys=ADDRESS + 8), dict(value_scales=ADDRESS + 4)):
        assert call(pages(**changes)) == abi.ERR_INVALID, changes
        assert b"paged" in LIB.lrk_last_error()
    for dimension in (96, 256):
        assert call(pages(dimension=dimension, group=32)) == abi.ERR_UNSUPPORTED
    assert call(stride=3) == abi.ERR_INVALID
    assert call(width=-1) == abi.ERR_INVALID
    assert call(flag=None) == abi.ERR_INVALID


def test_append_is_checked():
    for changes in (dict(heads=0), dict(tokens=-1), dict(sequences=0), dict(dtype=abi.F32), dict(lengths=None),
                    dict(k=rows(None)), dict(k=rows(ADDRESS + 2)), dict(v=rows(token=12)), dict(k=rows(head=4)),
                    dict(rotary_dim=24), dict(rotary_dim=144), dict(rotary_dim=-16), dict(rotary_dim=32),
                    dict(rotary_dim=32, rotary=ADDRESS), dict(query_heads=-1), dict(query_heads=4),
                    dict(query_heads=4, q=rows()), dict(query_heads=4, q=rows(), out=ADDRESS + 8)):
        assert append(**changes) == abi.ERR_INVALID, changes
    assert append(pages(group=0, dtype=abi.F16)) == abi.ERR_INVALID  # bfloat16 rows into float16 pages
    assert append(tokens=0) == abi.OK


def test_attention_is_checked():
    for changes in (dict(heads=0), dict(tokens=-1), dict(sequences=0), dict(dtype=abi.F32), dict(query_heads=7),
                    dict(query_heads=1), dict(query_heads=0), dict(scale=float("inf")), dict(scale=float("nan")),
                    dict(q=rows(None)), dict(q=rows(ADDRESS + 8)), dict(q=rows(token=4)), dict(out=None),
                    dict(out=ADDRESS + 2)):
        assert attend(**changes) == abi.ERR_INVALID, changes
    assert attend(pages(group=0, dtype=abi.F16)) == abi.ERR_INVALID
    for changes in (dict(workspace=None), dict(size=WORKSPACE_BYTES - 1), dict(workspace=ADDRESS + 8)):
        assert attend(**changes) == abi.ERR_WORKSPACE, changes
    assert attend(tokens=0) == abi.OK


def test_read_is_checked():
    for changes in (dict(slots=0), dict(count=-1), dict(dtype=abi.F64), dict(keys=None), dict(keys=ADDRESS + 4)):
        assert read(**changes) == abi.ERR_INVALID, changes
    assert read(count=0) == abi.OK


def test_page_memory_is_checked():
    import torch

    for changes in (dict(bits=8), dict(page_size=20), dict(dim=96), dict(bits=4, group=16), dict(bits=4, dim=64, group=128)):
        with pytest.raises(ValueError):
            Pages.empty(**{**dict(pages=2, page_size=16, dim=128, device="cpu"), **changes})
    p = Pages.empty(3, 16, 128, "cpu", torch.float16)
    assert p.keys.shape == (3, 16, 128) and p.dim == 128 and p.key_scales is None
    p = Pages.empty(3, 32, 64, "cpu", bits=4, group=32)
    assert p.keys.shape == (3, 32, 32) and p.value_scales.shape == (3, 32, 2, 2) and p.dim == 64
