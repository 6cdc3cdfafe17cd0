"""CPU: wait states that the compiler does not add inside inline assembly, looked up in the library's instructions."""
import os

import pytest

from dance_amd import _lib, build


def test_lds_copies_wait_for_m0():
    if not os.path.exists(build.OBJDUMP):
        pytest.skip("llvm-objdump not installed")
    copies, unwaited = build.lds_copies(_lib.SO_PATH)
    assert copies > 100                                    # the weight and operand stages' own
    assert unwaited == 0, "%d of %d copies to LDS directly behind a write of M0" % (unwaited, copies)
