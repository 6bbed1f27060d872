"""The CPython binding of the quantised layer's kernels: each interpreter has its own, and only the functions that go through it need it."""
import os
import subprocess
import sys
import sysconfig

import pytest

from basalt_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_file_carries_the_interpreters_tag():
    assert os.path.basename(build.PYTHON_BINDING) == "_klaunch" + sysconfig.get_config_var("EXT_SUFFIX")
    from basalt_b200 import _klaunch
    assert _klaunch.__file__ == build.PYTHON_BINDING


def test_the_other_kernels_do_without_it():
    code = """
import sys
sys.modules["basalt_b200._klaunch"] = None     # as if the file were not there
from basalt_b200 import kernels
assert kernels.vadd_i32 and kernels.matmul_f16 and kernels.sgemm_f32
for call in (lambda: kernels.rms_norm(16, 32, 0, 64, "f16"), lambda: kernels.quantize_e4m3(16, 32, 48, 0, 64, "f16"),
             lambda: kernels.matmul_e4m3(16, 32, 48, 64, 80, 0, 8, 64), lambda: kernels.matmul_w4(16, 32, 48, 64, 0, 8, 64, 32)):
    try:
        call()
    except ImportError as e:
        assert "python -m basalt_b200.build" in str(e), e
    else:
        raise SystemExit("no error")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_an_interpreter_without_headers_builds_the_rest(monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    build._build_python_binding(True, lambda command: pytest.fail(f"ran {command}"))
    assert "Python.h" in capsys.readouterr().err


@pytest.mark.parametrize("newer", ["python_binding.cpp", "basalt_b200_kernels.h"])
def test_it_is_built_again_when_a_source_changes(monkeypatch, newer):
    def age(path):
        return 2.0 if path.endswith(newer) else 1.0
    monkeypatch.setattr(build.os.path, "getmtime", age)
    ran = []
    build._build_python_binding(False, ran.append)
    assert len(ran) == 1
