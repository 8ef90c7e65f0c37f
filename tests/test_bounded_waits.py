"""Kernels whose waits run out end, report it, and leave the GPU usable; nothing here faults or hangs one.

The warps that share a row exchange values at a named barrier, which has no limit of its own: they have to give up
together.
"""

from __future__ import annotations

import itertools

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("warps", [1, 2, 4])
def test_warps_of_a_row_give_up_together(warps, steps):
    from lara_b200 import _native

    met = torch.empty(warps, dtype=torch.int32, device="cuda")
    for fail in itertools.product([-1, 0, 2, steps], repeat=warps):
        at = torch.tensor(fail, dtype=torch.int32, device="cuda")
        met.fill_(-9)
        _native.check(_native.lib.lara_selftest_group_exit(at.data_ptr(), met.data_ptr(), warps, steps,
                                                           torch.cuda.current_stream().cuda_stream), "selftest")
        assert met.tolist() == [min([steps] + [x for x in fail if x >= 0])] * warps, fail


def test_group_exit_refuses():
    from lara_b200._native import lib

    for args, code in [((0, 1 << 20, 2, 3, 0), 0x11), ((1 << 20, 0, 2, 3, 0), 0x11), ((1 << 20, 1 << 20, 0, 3, 0), 1),
                       ((1 << 20, 1 << 20, 33, 3, 0), 1), ((1 << 20, 1 << 20, 2, -1, 0), 1)]:
        assert lib.lara_selftest_group_exit(*args) == code
