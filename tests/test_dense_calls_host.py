"""Calls of the dense operators that differ from the usual ones in one thing: an alignment, a buffer's place, a size at the end of
its range. What can be seen of them without a GPU."""
import ctypes as C

import pytest

from b2ctrain_amd import nn
from tests.test_dense_host import ADDRESS, M, Room


def column(n, ptr=ADDRESS):
    return nn.Matrix(ptr, n, 1, 1, nn.F32)


@pytest.mark.parametrize("rows,di,f,ld,pitch", [(64, 144, 256, 144, 256), (64, 256, 320, 272, 256), (200, 48, 1040, 48, 128)])
def test_i8_block_copies_both_input_weights_or_none(rows, di, f, ld, pitch):
    """The tiles read both with one distance between rows, so a weight beside one that is copied is copied too."""
    def room(gate, up):
        p = nn.I8FeedForward(M(rows, di), M(f, di, nn.I8, ld, ADDRESS + gate), column(f), M(f, di, nn.I8, ld, ADDRESS + up), column(f),
                             M(di, f, nn.I8), column(di), M(rows, di), room=Room())
        return p.args.workspace_bytes

    assert room(0, 8) == room(8, 0) == room(8, 8) == room(0, 0) + 2 * f * pitch
