"""What is built and imported without torch, without its headers and without the front ends' C++ side."""
from __future__ import annotations

import subprocess
import sys
import textwrap
from pathlib import Path
from types import SimpleNamespace

import pytest

from llm_accelerator_b200 import build

ROOT = Path(__file__).resolve().parent.parent


def _python(code):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout, r.stderr


def test_without_torch():
    """The library is built, and what needs no torch imports."""
    out, err = _python("""
        import sys
        sys.modules["torch"] = None
        from llm_accelerator_b200 import build
        build.up_to_date = lambda: True
        print(build.build() == build.LIB)
        from llm_accelerator_b200 import bundle, engine, ptq, quarot, runner, simulator
    """)
    assert out == "True\n" and "torch is not installed" in err


def test_the_library_comes_first(monkeypatch, tmp_path):
    """A front end that does not compile leaves a new library behind, and says so."""
    done = []
    lib = tmp_path / "lib.so"

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        done.append(out.name)
        if ".tmp" in out.name and out.name.startswith("_front"):
            return SimpleNamespace(returncode=1, stdout="", stderr="no such header")
        out.write_bytes(b"")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "LIB", lib)
    monkeypatch.setattr(build, "OBJDIR", tmp_path / "objects")
    monkeypatch.setattr(build, "subprocess", SimpleNamespace(run=run))
    monkeypatch.setattr(build, "front_up_to_date", lambda: False)
    monkeypatch.setattr(build, "front_missing", lambda: None)
    with pytest.raises(RuntimeError, match="no such header"):
        build.build()
    assert lib.exists() and done[-1].startswith("_front")


@pytest.mark.parametrize("what", ["cuda", "headers"])
def test_without_what_the_module_needs(what, monkeypatch, tmp_path, capsys):
    import torch
    if what == "cuda":
        monkeypatch.setattr(torch.version, "cuda", None)
    else:
        monkeypatch.setattr(build.sysconfig, "get_path", lambda name: str(tmp_path))
    monkeypatch.setattr(build, "up_to_date", lambda: True)
    monkeypatch.setattr(build, "front_up_to_date", lambda: False)
    monkeypatch.setattr(build, "build_front", lambda: pytest.fail("was built"))
    assert build.build() == build.LIB
    assert "left out" in capsys.readouterr().err


def test_the_file_goes_by_torch_and_python(monkeypatch):
    import torch
    here = build.front_path()
    assert here.parent == build.PKG and torch.__version__ in here.name
    monkeypatch.setattr(torch, "__version__", "1.0")
    assert build.front_path() != here and not build.front_up_to_date()
    monkeypatch.undo()
    monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert build.front_path() != here
    monkeypatch.undo()
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: ".cpython-30-x86_64-linux-gnu.so")
    assert build.front_path() != here


def test_modules_that_use_nothing_of_it_import_without_it():
    out, err = _python("""
        import warnings
        from pathlib import Path
        from llm_accelerator_b200 import build
        build.front_path = lambda: Path("/nonexistent/_front.so")
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            from llm_accelerator_b200 import gemm, kv4, w8a8
        with warnings.catch_warnings(record=True) as w:
            warnings.simplefilter("always")
            from llm_accelerator_b200 import logprobs, mxfp4, norm, ptq
            print([("llm_accelerator_b200.build" in str(x.message)) for x in w])
        import torch
        for call in (lambda: norm.rms_norm(torch.ones((2, 8)), torch.ones(8)), lambda: mxfp4.quantize(torch.ones((2, 8))),
                     lambda: logprobs.token_logprobs(torch.ones((2, 8)), torch.zeros(2, dtype=torch.int64))):
            try:
                call()
            except ValueError:
                print("refused by Python")
    """)
    assert out == "[True]\n" + 3 * "refused by Python\n"


@pytest.mark.gpu
def test_results_without_it():
    out, _ = _python("""
        import warnings
        import torch
        from pathlib import Path
        from llm_accelerator_b200 import _tensors, build
        x, w = torch.randn((3, 100), device="cuda"), torch.ones(100, device="cuda")
        t = torch.zeros(3, dtype=torch.int64, device="cuda")
        def calls():
            from llm_accelerator_b200 import logprobs, mxfp4, norm, ptq
            q, s = norm.rms_norm_i8(x, w)
            a = mxfp4.quantize(x)
            return [norm.rms_norm(x, w), ptq.dequantize_rows(q, s, 100), a.values(), mxfp4.linear(x, a), mxfp4.gemm(a, a),
                    *logprobs.token_logprobs(x, t, 4)]
        build.front_path = lambda: Path("/nonexistent/_front.so")
        warnings.simplefilter("ignore")
        without = calls()
        import sys
        for name in [n for n in sys.modules if n.startswith("llm_accelerator_b200")]:
            del sys.modules[name]
        from llm_accelerator_b200._tensors import front
        assert front.quantize(x) is not None
        print(all(torch.equal(a, b) for a, b in zip(without, calls())))
    """)
    assert out == "True\n"
