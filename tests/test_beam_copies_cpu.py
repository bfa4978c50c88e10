"""What the copies of a beam search refuse, without a device."""
import pytest

from torchless_rs_b200.csrc.ops import KernelError, _pairs


def test_lists_of_copies():
    assert _pairs([], [], 4, "slot") == 0
    assert _pairs([0, 0, 2], [1, 3, 4], 5, "slot") == 3


@pytest.mark.parametrize("src,dst,why", [([0], [], "to write"), ([0], [5], "must lie"), ([5], [0], "must lie"), ([-1], [0], "must lie"),
                                         ([0], [-1], "must lie"), ([0, 1], [2, 2], "twice"), ([0, 2], [1, 0], "both read and written"),
                                         ([3], [3], "both read and written")])
def test_lists_of_copies_that_are_refused(src, dst, why):
    with pytest.raises(KernelError, match=why):
        _pairs(src, dst, 5, "slot")
