"""The library's build stands apart from the tests' folder: whatever
tests/sanitize lists or fails at, build() makes the library, and the sanitizer
library that its drivers link comes from the library's own recipe."""
import os
import subprocess
import sys

import pytest

import hachiue_amd  # noqa: F401 (the real one, whatever build() puts on the path)
from tests.test_build import ROOT, make

sys.path.insert(0, ROOT)
import __graft_entry__ as entry  # noqa: E402

CSRC = "all:\n\t@echo $@ >> made\n\nsanitize:\n\t@echo $@ >> made; mkdir -p $(SAN); echo new > $(SAN)/{}\n"
LIB = "libhachiue_sampler_asan.so"


def tree(tmp_path, sanitize, csrc=CSRC.format(LIB)):
    for where, text in (("hachiue_amd/csrc", csrc), ("oracle", "all:\n\t@echo ok > made\n"),
                        ("tests/sanitize", sanitize)):
        d = tmp_path / where
        d.mkdir(parents=True)
        (d / "Makefile").write_text(text)
    (tmp_path / "hachiue_amd/csrc/sampler_capi.hip").write_text("")
    out = tmp_path / "tests/sanitize/_build"
    out.mkdir()
    for driver in ("capi_check", "oracle_check"):
        (out / driver).write_text("stale")
    return out


def build(tmp_path, monkeypatch):
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    monkeypatch.setattr(sys, "path", list(sys.path))
    entry.build()
    assert (tmp_path / "hachiue_amd/csrc/made").read_text().split()[0] == "all"
    assert (tmp_path / "oracle/made").exists()


@pytest.mark.parametrize("sanitize", [
    "all:\n\t@false\n",                                     # a driver that does not compile
    "all: _build/no_such.o\n\t@true\n",                     # objects that nobody makes
    "this is no makefile\n"])
def test_a_failing_drivers_folder_stops_nothing(tmp_path, monkeypatch, capfd, sanitize):
    out = tree(tmp_path, sanitize)
    build(tmp_path, monkeypatch)
    assert "did not build" in capfd.readouterr().err
    assert not (out / "capi_check").exists() and not (out / "oracle_check").exists()   # none of an older build


def test_a_drivers_folder_with_another_list_of_objects(tmp_path, monkeypatch, capfd):
    """Its own recipe of the sanitizer library lists what does not exist: the
    library is there already, and the drivers are made from it."""
    out = tree(tmp_path, f"all: _build/capi_check _build/oracle_check\n"
                         f"_build/{LIB}: ../../hachiue_amd/csrc/_build/no_such.o\n\t@false\n"
                         f"_build/capi_check: _build/{LIB}\n\t@cp $< $@\n"
                         f"_build/oracle_check:\n\t@echo new > $@\n")
    build(tmp_path, monkeypatch)
    assert (out / "capi_check").read_text() == (out / "oracle_check").read_text() == "new\n"
    assert "did not build" not in capfd.readouterr().err


def test_no_drivers_folder(tmp_path, monkeypatch):
    tree(tmp_path, "all:\n\t@false\n")
    (tmp_path / "tests/sanitize/Makefile").unlink()
    build(tmp_path, monkeypatch)


def test_the_sanitizer_library_has_the_librarys_objects(tmp_path):
    """One object each, the C ABI's built anew under the sanitizers, the host's
    code alone."""
    out, cmds = tmp_path / "lib.so", {}
    for goal in ("all", "sanitize"):
        r = subprocess.run(["make", "-n", "-C", os.path.join(ROOT, "hachiue_amd/csrc"), f"OBJ={tmp_path}/obj",
                            f"OUT={out}", f"SAN={tmp_path}/san", goal], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        link = [line for line in r.stdout.splitlines() if "-shared" in line and "2>&1" in line]
        assert len(link) == 1
        cmds[goal] = (r.stdout, sorted({w for w in link[0].replace(")", " ").split() if w.endswith(".o")}))
    objs = cmds["all"][1]
    assert f"{tmp_path}/obj/sampler_capi.o" in objs and len(objs) >= 6
    want = [o.replace("sampler_capi.o", "sampler_capi_asan.o") for o in objs]
    assert cmds["sanitize"][1] == sorted(want)
    words = cmds["sanitize"][0].split()
    for i, w in enumerate(words):
        if w.startswith("-fsanitize"):
            assert words[i - 1] == "-Xarch_host"
    assert any(w.startswith("-fsanitize=address") for w in words)
    # a compiler that fails ends it
    r = make(tmp_path, "hachiue_amd/csrc", 3, f"OBJ={tmp_path}/obj2", f"SAN={tmp_path}/san2", "sanitize")
    assert r.returncode != 0 and not os.path.exists(tmp_path / "san2" / LIB)
