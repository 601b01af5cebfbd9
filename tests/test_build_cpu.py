"""The library's build with a stand-in for the compiler."""

import os
import stat

import pytest

FAKE = """#!/bin/sh
# -c -o OBJ SOURCE, or a link; `loud` talks more than a pipe holds, `quiet` waits for it
out= ; src=
while [ $# -gt 0 ]; do
  case "$1" in
    -o) out="$2"; shift ;;
    *.cu) src="$1" ;;
  esac
  shift
done
case "$src" in
  *quiet.cu)
    i=0
    while [ ! -e "$MARK" ]; do
      i=$((i + 1)); [ $i -gt 50 ] && exit 1
      sleep 0.1
    done ;;
  *loud.cu)
    head -c 300000 /dev/zero | tr '\\0' 'w'
    echo "the end"
    : > "$MARK"
    [ -n "$FAIL" ] && exit 1 ;;
esac
: > "$out"
"""


@pytest.fixture
def fake_build(tmp_path, monkeypatch):
    from iquestrt_b200 import _build
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(FAKE)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    for name in ("quiet.cu", "loud.cu"):
        (tmp_path / name).write_text("")
    monkeypatch.setattr(_build, "_nvcc", lambda: str(nvcc))
    monkeypatch.setattr(_build, "SOURCES", {"quiet.cu": (), "loud.cu": ()})
    monkeypatch.setattr(_build, "CSRC", str(tmp_path))
    monkeypatch.setattr(_build, "OBJ", str(tmp_path / "build"))
    monkeypatch.setattr(_build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setenv("MARK", str(tmp_path / "mark"))
    return _build


def test_a_compiler_that_talks_does_not_wait_for_the_others(fake_build):
    """The first source's compiler ends only once the second's, whose messages fill any pipe, has."""
    assert os.path.exists(fake_build.build(force=True))


def test_messages_of_a_failed_build_are_shown_whole(fake_build, monkeypatch):
    monkeypatch.setenv("FAIL", "1")
    with pytest.raises(RuntimeError, match="w{300000}the end"):
        fake_build.build(force=True)
    assert not os.path.exists(fake_build.LIB)
