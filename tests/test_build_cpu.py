"""Which sources a build compiles again (with a stand-in for hipcc that only writes its output)."""
import os

import pytest

from after_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    src, lib, log = tmp_path / "csrc", tmp_path / "lib", tmp_path / "log"
    src.mkdir()
    for n in ("a.hip", "b.hip", "c.h"):
        (src / n).write_text("")
    hipcc = tmp_path / "hipcc"
    hipcc.write_text("#!/bin/sh\n"
                     "if [ \"$1\" = --version ]; then echo \"HIP version: $(cat %s/version)\"; exit; fi\n"
                     "while [ $# -gt 0 ]; do [ \"$1\" = -c ] && echo \"$(basename $2)\" >> %s; [ \"$1\" = -o ] && : > \"$2\"; shift; done\n" % (tmp_path, log))
    hipcc.chmod(0o755)
    (tmp_path / "version").write_text("7.2.0")
    monkeypatch.setenv("HIPCC", str(hipcc))
    for name, value in (("CSRC", src), ("LIBDIR", lib), ("LIB", lib / "libafter_hip.so")):
        monkeypatch.setattr(build, name, str(value))

    def made():
        log.write_text("")
        build.build_library()
        return sorted(log.read_text().split())

    return tmp_path, made


def test_a_build_compiles_what_is_not_up_to_date(tree, monkeypatch):
    root, made = tree
    both = ["a.hip", "b.hip"]
    assert made() == both and made() == []
    later = os.path.getmtime(root / "lib" / "a.o") + 10
    os.utime(root / "csrc" / "b.hip", (later, later))
    assert made() == ["b.hip"]
    os.utime(root / "csrc" / "b.hip", (0, 0))
    assert made() == []
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DOTHER"])
    assert made() == both and made() == []
    (root / "version").write_text("7.2.1")
    assert made() == both and made() == []
    os.remove(root / "lib" / "hipcc_version.txt")  # (nobody knows what built these)
    assert made() == both and made() == []
