"""What the serving entries refuse at the ends of their ranges, on a machine without a device."""

import os
import shutil
import subprocess
import sys

import pytest

pytest.importorskip("torch")

from intent_ir_b200 import _lib  # noqa: E402

from .test_serving_cpu import P, _append, _attention, _norm, _w4  # noqa: E402


def test_rows_without_columns_need_room_for_their_scales():
    assert _norm(cols=0, group=0, scale=None) == _lib.ERR_INVALID
    assert _norm(cols=0, group=0, rows=1 << 41) == _lib.ERR_INVALID
    assert _norm(cols=0, group=32, scale=None) == _lib.OK and _norm(cols=0, group=0, out=_lib.BF16, scale=None) == _lib.OK  # no scales


@pytest.mark.parametrize("m,group,xt", [(17, 32, _lib.BF16), (64, 64, _lib.F16), (9, 128, _lib.BF16), (200, 128, _lib.E4M3)])
def test_a_k_whose_bytes_pass_32_bits_is_refused_where_x_is_copied_by_bytes(m, group, xt):
    """2^30 + 32 values of 16 bits: a copy's coordinate would wrap, and the rest of the sum be lost."""
    k = (1 << 30) + 32
    held = dict(xg=1) if xt == _lib.E4M3 else {}
    assert _w4(m=m, n=1, k=k, xs=k, group=group, xt=xt, **held) == _lib.ERR_UNSUPPORTED
    assert "2^30" in _lib.last_error()
    scratch = _lib.load().ib200_w4_scratch_bytes
    assert scratch(xt, m, 1, k, group) == 0
    assert scratch(xt, 16, 1, 1 << 30, 128) == 16 * (1 << 30) * 2  # the last that is taken


@pytest.mark.parametrize("m", [1, 12, 40])
@pytest.mark.parametrize("xt", [_lib.E4M3, _lib.I8])
def test_scales_of_x_are_needed_without_columns_too(m, xt):
    """K = 0: the result is still multiplied by the row's scale on its way out."""
    assert _w4(m=m, k=0, xt=xt, xg=1, xsc=None) == _lib.ERR_INVALID


GUARD = """
#include <cstdio>
#include <new>
#include <stdexcept>
#include "guard.h"
int main() {
  std::string message = "an older failure";
  if (ib200::guarded(message, -3, [] { return 7; }) != 7 || message != "an older failure") return 1;
  if (ib200::guarded(message, -3, []() -> int { throw std::runtime_error("no room"); }) != -3 || message != "exception: no room") return 2;
  if (ib200::guarded(message, -3, []() -> int { throw std::bad_alloc(); }) != -3 || message != "exception: std::bad_alloc") return 3;
  if (ib200::guarded(message, -3, []() -> int { throw 5; }) != -3 || message != "unknown exception") return 4;
  puts("guarded");
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="needs a C++ compiler")
def test_an_exception_at_a_c_entry_is_an_error_with_a_message_of_its_own(tmp_path):
    (tmp_path / "guard.cpp").write_text(GUARD)
    csrc = os.path.join(os.path.dirname(_lib.HERE), "intent_ir_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", csrc, str(tmp_path / "guard.cpp"), "-o", str(tmp_path / "guard")], check=True)
    assert subprocess.run([str(tmp_path / "guard")], capture_output=True, text=True, check=True).stdout == "guarded\n"


WITHOUT_CUDA = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda")]:
    delattr(torch._C, name)
from intent_ir_b200 import ops
from intent_ir_b200.errors import B200RuntimeError
try:
    ops.rmsnorm(torch.zeros(2, 64))
except B200RuntimeError:
    print("imported")
"""


def test_the_entries_import_where_torch_was_built_without_cuda():
    done = subprocess.run([sys.executable, "-c", WITHOUT_CUDA], cwd=os.path.dirname(_lib.HERE), capture_output=True, text=True, timeout=300)
    assert done.stdout == "imported\n", done.stderr[-2000:]


def test_tokens_of_no_sequence_are_refused():
    """Without offsets the tokens are dealt out evenly: to no sequences none can be, and the result would be left unwritten."""
    assert _append(batch=0) == _lib.ERR_INVALID and _attention(batch=0) == _lib.ERR_INVALID
    assert _append(batch=0, cu=P) == _lib.OK and _attention(batch=0, cu=P) == _lib.OK  # all tokens lie behind the last sequence
