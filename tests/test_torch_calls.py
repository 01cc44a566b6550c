"""The C++ module behind the paged operators and the batched sampler for torch tensors: what depends on
it, and when it is built again. No GPU."""
import os
import subprocess
import sys

import pytest

from kernel_optimization_webgpu_b200 import build

ROOT = build.ROOT


def _run(tmp_path, body):
    """Runs a program beside a torch package without C++ headers, no module having been built yet."""
    (tmp_path / "torch").mkdir()
    (tmp_path / "torch" / "__init__.py").write_text("__version__ = '0'\n")
    head = (f"import sys; sys.path[:0] = [{str(tmp_path)!r}, {ROOT!r}]\n"
            "from kernel_optimization_webgpu_b200 import build, _lib\n"
            f"build.CALLS = {str(tmp_path / '_torch_calls.so')!r}\n")
    return subprocess.run([sys.executable, "-c", head + body], capture_output=True, text=True, timeout=300)


def test_the_library_loads_where_the_torch_module_cannot_be_built(tmp_path):
    build.build()
    res = _run(tmp_path, "print(_lib.load().qd_paged_attn_decode_workspace_bytes(1, 1) > 0)")
    assert res.returncode == 0 and res.stdout.split() == ["True"], res.stderr


def test_only_the_calls_that_need_the_module_fail_and_say_so(tmp_path):
    build.build()
    res = _run(tmp_path, "from kernel_optimization_webgpu_b200 import runtime\n"
                         "try:\n    runtime.sample_rows(None, None)\n"
                         "except RuntimeError as err:\n    print('refused', '_torch_calls' in str(err))\n")
    assert res.returncode == 0 and res.stdout.split() == ["refused", "True"], res.stderr


def test_the_module_is_built_again_for_another_torch(monkeypatch, tmp_path):
    torch = pytest.importorskip("torch")
    calls = tmp_path / "_torch_calls.so"
    built = []

    def compiler(cmd, **kw):
        built.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "CALLS", str(calls))
    monkeypatch.setattr(build, "CALLS_KEY", str(tmp_path / "key"), raising=False)
    monkeypatch.setattr(build.subprocess, "run", compiler)
    for version, builds in (("1", 1), ("1", 1), ("2", 2), ("2", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        assert build.build_calls() == str(calls) and calls.exists()
        assert len(built) == builds
    os.remove(calls)
    build.build_calls()
    assert len(built) == 3
    # processes that build at once do not write one file
    assert all(str(os.getpid()) in cmd[cmd.index("-o") + 1] for cmd in built)
