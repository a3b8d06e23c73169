"""The in-tree build of the extension."""
import importlib.util
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _setup():
    spec = importlib.util.spec_from_file_location(
        "mxa_setup", os.path.join(ROOT, "setup.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_a_changed_header_rebuilds(tmp_path):
    """Objects are stale when a header is newer, also one that is included
    through another; the others stay."""
    src, out = tmp_path / "src", tmp_path / "out"
    (src / "kernels").mkdir(parents=True)
    out.mkdir()
    (src / "kernels" / "a.h").write_text("#pragma once\n")
    (src / "kernels" / "b.h").write_text('#include "a.h"\n')
    (src / "bind.hip").write_text('#include "kernels/b.h"  // b\n')
    (src / "kernels" / "x.hip").write_text('#include "a.h"\n')
    (src / "kernels" / "y.hip").write_text("#include <vector>\n")
    objs = [out / n for n in ("bind_hip.o", "x_hip.o", "y.o")]
    for o in objs:
        o.write_text("")
    files = list(src.rglob("*.h*"))
    for i, f in enumerate(files):
        os.utime(f, (1000, 1000))
    for o in objs:
        os.utime(o, (2000, 2000))
    stale = _setup().stale_objects
    names = [str(o) for o in objs]
    assert stale(names, str(src)) == []
    os.utime(src / "kernels" / "b.h", (3000, 3000))
    assert stale(names, str(src)) == names[:1]
    os.utime(src / "kernels" / "a.h", (3000, 3000))
    assert stale(names, str(src)) == names[:2]
