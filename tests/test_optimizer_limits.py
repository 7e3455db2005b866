"""CPU: how many elements a plan takes, as include/nerf_amd.h states it."""
import re
from pathlib import Path

import pytest

from test_optimizer import _create, _tensor

MOST = ((1 << 22) - 1) * 4096


def test_the_header_states_the_limit():
    header = (Path(__file__).parent.parent / "include" / "nerf_amd.h").read_text()
    text = re.search(r"#define NERF_ADAMW_MAX_ELEMENTS (\(.*?\)) /\*", header).group(1)
    assert eval(text.replace("(size_t)", "")) == MOST


@pytest.mark.parametrize("sizes,taken", [([MOST], True), ([MOST + 1], False), ([MOST - 4096, 4096], True), ([MOST - 4096, 1], True),
                                         ([MOST - 4096, 1, 1], False), ([MOST, 1], False), ([1 << 41], False), ([1 << 62], False),
                                         ([(1 << 64) - 1, 5], False)], ids=str)
def test_elements_of_a_list(sizes, taken):
    """a list that is taken fails with 2 where there is no GPU (with 1 where there is: the pointers are not its)"""
    from nerf_amd._lib import lib
    rc = _create([_tensor(n=n, w=0, m=0, v=0) for n in sizes], bits=0)
    assert rc == (1 if lib.nerf_device_count() or not taken else 2)
