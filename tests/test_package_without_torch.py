"""The package, its C library and its build where torch or the extension on torch tensors is not there."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


def python(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


NO_TORCH = "import sys; sys.modules['torch'] = None\n"
NO_EXTENSION = "import sys; sys.modules['vesper_db_b200._attention'] = None\n"


def test_star_import_needs_no_torch():
    out = python(NO_TORCH + "from vesper_db_b200 import *\nprint(IvfPqIndex.__name__, flat_topk.__name__)")
    assert out.split() == ["IvfPqIndex", "flat_topk"]


@pytest.mark.parametrize("missing,says", [(NO_TORCH, "torch"), (NO_EXTENSION, "vesper_db_b200.build")],
                         ids=["torch", "extension"])
def test_operators_that_cannot_load_are_absent_attributes(missing, says):
    """hasattr and getattr with a default work; the message of the error says what is missing."""
    out = python(missing + "import vesper_db_b200 as V\nprint(hasattr(V, 'page_tables'), getattr(V, 'norm_rotate', 7))\n"
                 "try: V.prompt_attention\nexcept AttributeError as e: print(e)")
    assert out.split()[:2] == ["False", "7"] and says in out


def test_operators_are_listed_and_importable():
    python("import vesper_db_b200 as V\nfrom vesper_db_b200 import page_tables, PageTables\n"
           "assert {'page_tables', 'norm_rotate', 'prompt_attention', 'shared_prefix_attention', 'PageTables'} <= set(dir(V))\n"
           "assert hasattr(V, 'shared_prefix_attention') and not hasattr(V, 'no_such_thing')")


def test_library_builds_without_torch(tmp_path):
    """The C library alone needs no torch: the build says that it leaves the extension out."""
    out = python(NO_TORCH + "from vesper_db_b200 import build as b\n"
                 f"b.EXT = {str(tmp_path / '_attention.so')!r}\nassert b.build(verbose=True) == b.LIB\n"
                 "import os; assert not os.path.exists(b.EXT)")
    assert "torch" in out and "_attention.so" in out


def test_extension_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    """It is tied to the binary interface of the torch and the Python that it was compiled with."""
    from vesper_db_b200 import build as b
    built, real = [], b._run
    monkeypatch.setattr(b, "EXT", str(tmp_path / "_attention.so"))

    def run(cmd):
        if b.EXT not in cmd:  # the library's own parts are built as ever
            return real(cmd)
        built.append(cmd)
        open(b.EXT, "w").close()
    monkeypatch.setattr(b, "_run", run)
    import torch

    def builds():
        built.clear()
        b.build()
        return len(built)
    assert builds() == 1 and builds() == 0
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    assert builds() == 1 and builds() == 0
    os.utime(b.EXT, (1, 1))
    assert builds() == 1
