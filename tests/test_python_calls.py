"""What the Python package needs and takes: dtypes of torch tensors."""
import pytest
import torch


@pytest.fixture(scope="module")
def F(built_libs):
    from diopi_b200 import functions
    return functions


def test_float8_tensors_only_where_codes_are_meant(F):
    """The interface has no 8-bit float. An op without e4m3 codes does not take them for whole numbers."""
    x = torch.zeros(3, 2, 8).to(torch.float8_e4m3fn)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        F.destindex_copy_kv(x, torch.zeros(3, dtype=torch.int32), x.clone(), as_device=True)
    # the caches of the 8-bit operators are, also as handles made beforehand: what is refused here is the next argument
    from diopi_b200.runtime import DiopiError, Tensor
    cache, scale, ids = torch.zeros(4, 16, 2, 8).to(torch.float8_e4m3fn), torch.zeros(4, 2), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(DiopiError, match="softmax_scale"):
        F.quantized_paged_attention(torch.zeros(1, 2, 8).half(), cache, cache, scale, scale, ids, ids[0, :1], -1.0, as_device=True)
    handle = Tensor(cache, as_device=True)
    with pytest.raises(DiopiError, match="softmax_scale"):
        F.quantized_paged_attention(torch.zeros(1, 2, 8).half(), handle, handle, scale, scale, ids, ids[0, :1], -1.0, as_device=True)


# ---- the module that makes the calls of the 8-bit cache operators -----------------------------------
def test_the_other_ops_load_without_the_call_module(built_libs, tmp_path):
    """A tree without the CPython module (no Python headers where it was built) has every op but those that are called through it."""
    import shutil
    import subprocess
    import sys
    from diopi_b200 import _lib
    for name in ("libdiopi_rt.so", "libdiopi_impl.so"):
        shutil.copy(_lib.LIB_DIR / name, tmp_path / name)
    code = f"""
import pathlib, torch
from diopi_b200 import _lib
_lib.LIB_DIR = pathlib.Path({str(tmp_path)!r})
from diopi_b200 import functions as F
from diopi_b200.runtime import DiopiError
try:
    F.destindex_copy_kv(torch.zeros(1, 1, 1), torch.zeros(1), torch.zeros(1, 1, 1), as_device=True)
except DiopiError as e:
    print(e)
z = torch.zeros(1, dtype=torch.int32)
try:
    F.build_block_table(z[None], z, z, z, z, 4, slot_map=z, new_start=z, seq_lens=z, free_next=z, as_device=True)
except RuntimeError as e:
    print(e)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=_lib.LIB_DIR.parent.parent)
    assert r.returncode == 0, r.stderr
    lines = r.stdout.splitlines()
    assert "int32 or int64" in lines[0] and "_pycall" in lines[1] and "Python headers" in lines[1]


class FakeBuild:
    """diopi_b200.build in a folder of its own, with a compiler that only writes its output files."""

    def __init__(self, monkeypatch, tmp_path):
        from diopi_b200 import build as b
        self.b, self.linked, self.patch = b, [], monkeypatch
        monkeypatch.setattr(b, "LIB", tmp_path / "lib")
        monkeypatch.setattr(b, "OBJ", tmp_path / "obj")
        monkeypatch.setattr(b, "_compile", lambda src, *a: tmp_path / src.replace("/", "_"))
        monkeypatch.setattr(b, "_link", lambda objs, out, extra: (self.linked.append(out.name), out.write_text("")))

    def __call__(self):
        self.linked.clear()
        return self.b.build()

    def python(self, suffix, include):
        import sysconfig
        var = sysconfig.get_config_var
        self.patch.setattr(sysconfig, "get_config_var", lambda name: suffix if name == "EXT_SUFFIX" else var(name))
        self.patch.setattr(sysconfig, "get_paths", lambda: {"include": str(include)})


def test_build_goes_by_the_python_that_runs_it(monkeypatch, tmp_path):
    build = FakeBuild(monkeypatch, tmp_path)
    (tmp_path / "Python.h").write_text("")
    build.python(".cpython-312-x.so", tmp_path)
    assert build()["py"].name == "_pycall.cpython-312-x.so" and len(build.linked) == 3
    build()
    assert build.linked == []
    build.python(".cpython-313-x.so", tmp_path)   # another one does not take the first one's module
    assert build()["py"].name == "_pycall.cpython-313-x.so" and build.linked == ["_pycall.cpython-313-x.so"]
    build.python(".cpython-312-x.so", tmp_path / "nothing")   # and a module that is there needs no headers any more
    assert build()["py"].name == "_pycall.cpython-312-x.so" and build.linked == []


def test_build_without_python_headers(monkeypatch, tmp_path, capsys):
    build = FakeBuild(monkeypatch, tmp_path)
    build.python(".cpython-312-x.so", tmp_path / "nothing")
    assert set(build()) == {"impl", "rt"} and "Python.h" in capsys.readouterr().err
    build()
    assert build.linked == []


def test_handles_that_cannot_be_made_are_an_error(built_libs):
    """A C entry of the run time gives null back; an exception that leaves it would end the process (hence one of its own here)."""
    import subprocess
    import sys
    from diopi_b200 import _lib
    code = """
import ctypes
from diopi_b200 import _lib
rt = _lib.load().rt
rt.b200rt_batch_create.restype = ctypes.c_void_p
rt.b200rt_batch_create.argtypes = [ctypes.POINTER(ctypes.c_int64), ctypes.c_int, ctypes.c_void_p]
print(rt.b200rt_batch_create((ctypes.c_int64 * 4)(), -1, None))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=_lib.LIB_DIR.parent.parent)
    assert r.returncode == 0 and r.stdout.strip() == "None", (r.returncode, r.stderr[-300:])
