"""What od_wscl_amd/_build.py makes again, with a compiler that writes down its arguments."""
import os
import stat

import pytest

from od_wscl_amd import _build

FAKE = """#!/bin/sh
out=""
for a in "$@"; do
    if [ "$last" = "-o" ]; then out="$a"; fi
    last="$a"
done
echo "$@" > "$out"
basename "$out" >> "$LOG"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    here = tmp_path / "od_wscl_amd"
    csrc = here / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "a.h").write_text("")
    for n in ("one.hip", "two.hip", "odw.h", "bind.cpp"):
        (csrc / n).write_text("")
    old = os.stat(csrc / "one.hip").st_mtime - 100
    for p in list(csrc.iterdir()) + [tmp_path / "include" / "a.h"]:
        os.utime(p, (old, old))
    cc = tmp_path / "cc"
    cc.write_text(FAKE)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    log = tmp_path / "log"
    monkeypatch.setenv("LOG", str(log))
    for name, value in (("HERE", str(here)), ("CSRC", str(csrc)), ("LIB", str(here / "libodwscl.so")), ("BIND", str(here / "_bind.so")),
                        ("BIND_SRC", str(csrc / "bind.cpp")), ("RECORD", str(here / "build" / "commands.json")), ("HIPCC", str(cc)),
                        ("FLAGS", list(_build.FLAGS)), ("_bind_command", lambda: [str(cc), "-o", str(here / "_bind.so")])):
        monkeypatch.setattr(_build, name, value)

    def made(**more):
        if log.exists():
            log.unlink()
        _build.build(**more)
        return sorted(log.read_text().split()) if log.exists() else []
    return csrc, made


def test_only_what_is_stale_is_made_again(tree):
    csrc, made = tree
    every = ["_bind.so", "libodwscl.so", "one.o", "two.o"]
    assert made() == every and made() == [] and made(force=True) == every and made() == []
    later = os.stat(csrc / "one.o").st_mtime + 10
    os.utime(csrc / "one.hip", (later, later))
    assert made() == ["libodwscl.so", "one.o"]


def test_other_flags_reach_every_object(tree):
    csrc, made = tree
    made()
    _build.FLAGS.append("-DOTHER")
    assert made() == ["libodwscl.so", "one.o", "two.o"] and "-DOTHER" in (csrc / "two.o").read_text()
    assert made() == []
    os.remove(_build.RECORD)                    # a tree built before commands were written down
    assert made() == ["_bind.so", "libodwscl.so", "one.o", "two.o"] and made() == []
    os.remove(csrc / "two.hip")
    assert made() == ["libodwscl.so"]


def test_a_failed_build_is_not_taken_for_done(tree, monkeypatch):
    csrc, made = tree
    made()
    _build.FLAGS.append("-DOTHER")
    cc, bad = _build.HIPCC, csrc / "bad"
    bad.write_text("#!/bin/sh\nexit 1\n")
    bad.chmod(0o755)
    monkeypatch.setattr(_build, "HIPCC", str(bad))
    with pytest.raises(RuntimeError):
        made()
    monkeypatch.setattr(_build, "HIPCC", cc)
    assert made() == ["libodwscl.so", "one.o", "two.o"]
