"""The library with the PyTorch operators in C++ depends on the installed torch; the rest of the package does not depend
on it: imports with a library that does not fit, and the build's decision whether it does."""

import subprocess
import sys
from pathlib import Path

import pytest

from spio_b200 import _clib, build

ROOT = Path(__file__).resolve().parent.parent

# (the paths are changed before anything loads the library)
PROGRAM = """
import sys
from pathlib import Path
from spio_b200 import _clib
_clib.TORCH_LIB_PATH, _clib.TORCH_STAMP_PATH = Path(sys.argv[1]), Path(sys.argv[2])
import torch
from spio_b200.layers import Conv2dGw8, GroupNorm2d, LayerNorm2d
from spio_b200.functional import checkpoint8_pack, checkpoint8_unpack, conv2d_gw8, conv2d_gw8_checkpoint8, groupnorm_2d
from spio_b200.transform import transform
model = torch.nn.Sequential(torch.nn.Conv2d(16, 16, 3, groups=2), torch.nn.GroupNorm(4, 16))
assert isinstance(getattr(transform(model), "0"), Conv2dGw8)
assert _clib.load().spio_conv2d_gw8_num_variants() > 0
x, k = torch.zeros(1, 16, 4, 4), torch.zeros(16, 8, 3, 3)
for call in (lambda: groupnorm_2d(x, 4), lambda: GroupNorm2d(4, 16)(x), lambda: checkpoint8_pack(x),
             lambda: checkpoint8_unpack(x.char(), x[:, :2].byte()), lambda: conv2d_gw8_checkpoint8(x, k, groups=2)):
    try:
        call()
    except RuntimeError as e:
        assert sys.argv[3] in str(e) and "spio_b200.build" in str(e), e
    else:
        raise AssertionError("no error")
"""


def run(lib, stamp, message):
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(lib), str(stamp), message], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_imports_do_not_need_the_operators(tmp_path):
    run(tmp_path / "absent.so", tmp_path / "absent", "is missing")
    # a library with a symbol that nothing defines, as one that was built against another torch
    source, lib = tmp_path / "odd.c", tmp_path / "odd.so"
    source.write_text("extern int spio_no_such_symbol(void);\nint (*odd)(void) = spio_no_such_symbol;\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(lib)], check=True)
    run(lib, tmp_path / "absent", "does not load")
    stamp = tmp_path / "stamp"
    stamp.write_text("torch 1.0 cxx11_abi=0\n")
    run(_clib.TORCH_LIB_PATH, stamp, "was built for torch 1.0")


def test_library_of_another_torch_is_not_current(tmp_path, monkeypatch):
    lib, stamp = tmp_path / "lib.so", tmp_path / "stamp"
    lib.write_text("as new as can be")
    monkeypatch.setattr(build, "TORCH_LIB_PATH", lib)
    monkeypatch.setattr(build, "TORCH_STAMP_PATH", stamp)
    assert not build.torch_lib_is_current()
    stamp.write_text("torch 1.0 cxx11_abi=0\n")
    assert not build.torch_lib_is_current()
    stamp.write_text(_clib.torch_stamp() + "\n")
    assert build.torch_lib_is_current()


def test_build_without_cuda_in_torch(monkeypatch, capsys):
    import torch

    monkeypatch.setattr(torch.version, "cuda", None)
    monkeypatch.setattr(build, "_run", lambda *a: pytest.fail("nothing is to be compiled"))
    assert build.build_torch_lib(force=True) is None
    assert "not built" in capsys.readouterr().err
