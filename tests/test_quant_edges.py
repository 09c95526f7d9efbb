"""CPU checks of the 8-bit row makers' newer arguments: what is refused before anything is launched."""
import pytest

from frisk_b200 import runtime as R
from frisk_b200 import workloads as W


def test_status_words_that_are_refused():
    desc = R.quant_desc(4, 8, W.BF16, W.I8, "silu_mul")
    for status, code in ((0x50002, -3), (0x20000, -1), (0x30000, -1)):   # off its alignment; q; the scales
        with pytest.raises(R.FriskError) as e:
            R.quant_run(desc, 0x10000, 0x20000, 0x30000, status=status)
        assert e.value.code == code
    R.quant_run(R.quant_desc(0, 8, W.BF16, W.I8, "silu_mul"), None, None, None, status=0x50000)   # no rows
