"""The paged cache's host side at edges that test_paged_host.py leaves out."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "code_for_iclr27_b200" / "csrc"


def test_every_bit_of_the_flag_has_a_cause_of_its_own():
    """The kernels' bits are distinct, and check_flags names the cause of each."""
    from code_for_iclr27_b200.paged import PagedCache

    bits = {name: int(value) for name, value in re.findall(r"constexpr uint32_t kFlag(\w+) = (\d+);", (CSRC / "paged.cuh").read_text())}
    assert sorted(bits.values()) == [1, 2, 4, 8]
    # A kernel whose shared memory is not aligned has met no wait that ran out.
    for source in ("paged_attention.cu", "paged_attention_tc.cu"):
        after = (CSRC / source).read_text().split("if (base & 1023)")[1][:200]
        assert "kFlagShared" in after and "kFlagTimeout" not in after
    cache = PagedCache(1, 1, 1, 64, 4, "cpu", page_size=16, max_rows=64)
    cache.check_flags()
    for bit, cause in ((1, "row outside its pages or token of no sequence"), (2, "rotary"), (4, "wait"), (8, "shared memory")):
        cache.flag.fill_(bit)
        with pytest.raises(RuntimeError, match=f"flagged: {bit} .*{bit}: [^,]*{cause}"):
            cache.check_flags()
        assert int(cache.flag.item()) == 0
