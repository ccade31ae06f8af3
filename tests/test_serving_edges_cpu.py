"""What the serving entries refuse at the ends of their ranges, on a machine without a device."""

import pytest

pytest.importorskip("torch")

from intent_ir_b200 import _lib  # noqa: E402

from .test_serving_cpu import _norm  # noqa: E402


def test_rows_without_columns_need_room_for_their_scales():
    assert _norm(cols=0, group=0, scale=None) == _lib.ERR_INVALID
    assert _norm(cols=0, group=0, rows=1 << 41) == _lib.ERR_INVALID
    assert _norm(cols=0, group=32, scale=None) == _lib.OK and _norm(cols=0, group=0, out=_lib.BF16, scale=None) == _lib.OK  # no scales
