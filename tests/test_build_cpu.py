"""The build of the library: every source is compiled, each is reported when it is done, and a failure at once."""
import os
import re
import time

import pytest

from ccglib_amd import build as b


def test_every_source_is_compiled_once():
    units = {n for n in os.listdir(b.CSRC) if n.endswith(".hip")}
    included = set()
    for n in os.listdir(b.CSRC):
        with open(os.path.join(b.CSRC, n)) as f:
            included |= set(re.findall(r'^#include "([^"/]+\.hip)"', f.read(), re.M))
    assert sorted(b.SOURCES) == sorted(units - included)


@pytest.fixture
def pretended(monkeypatch, tmp_path):
    """Sources that take a while to compile; what was started, in order."""
    started = []

    def compile_one(src, force):
        started.append(src)
        time.sleep({"slow": 1.5, "bad": 0.2}.get(src.split("_")[0], 0.3))
        if src.startswith("bad"):
            raise RuntimeError("hipcc failed for bad")
        return src, ""
    monkeypatch.setattr(b, "_compile", compile_one)
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(b, "_stale", lambda target, deps: False)
    return started


def test_a_source_is_reported_when_it_is_done(pretended, monkeypatch, capsys):
    monkeypatch.setattr(b, "SOURCES", ["slow"] + ["quick_%d" % i for i in range(5)])
    b.build(verbose=True)
    lines = [l for l in capsys.readouterr().out.splitlines() if l]
    assert len(lines) == 6 and lines[-1].startswith("slow: ")


def test_a_failure_is_reported_before_the_others_are_done_and_starts_nothing_more(pretended, monkeypatch, capsys):
    monkeypatch.setattr(b, "SOURCES", ["slow_%d" % i for i in range(7)] + ["bad"] + ["later_%d" % i for i in range(40)])
    with pytest.raises(RuntimeError, match="hipcc failed for bad"):
        b.build()
    err = capsys.readouterr().err
    assert "bad: failed" in err and "compiler: " in err
    assert len(pretended) < 20


def failing(tmp_path, times, message):
    """A command that fails so many times before it succeeds, each time with that message."""
    count = tmp_path / "count"
    count.write_text("0")
    return ["sh", "-c", 'n=$(cat "$0"); echo $((n + 1)) > "$0"; test $n -ge %d || { echo "%s" >&2; exit 9; }' % (times, message),
            str(count)], lambda: int(count.read_text())


def test_a_compiler_that_was_killed_is_run_once_more(tmp_path):
    cmd, runs = failing(tmp_path, 1, "clang: error: unable to execute command: Killed")
    r = b._run(cmd)
    assert r.returncode == 0 and runs() == 2
    assert "unable to execute command" in r.stderr and "status 9" in r.stderr


def test_a_compiler_that_is_killed_again_has_failed(tmp_path):
    cmd, runs = failing(tmp_path, 5, "Killed")
    assert b._run(cmd).returncode == 9 and runs() == 2


@pytest.mark.parametrize("message", ["x.hip:3:14: error: expected expression", "x.hip:1:10: fatal error: file not found",
                                     "ld.lld: error: undefined symbol: f"])
def test_an_error_in_the_source_is_final(tmp_path, message):
    cmd, runs = failing(tmp_path, 5, message)
    assert b._run(cmd).returncode == 9 and runs() == 1


def test_no_more_compilers_than_processors(monkeypatch):
    for have, want in ((1, 1), (8, 8), (16, 16), (256, 16)):
        monkeypatch.setattr(os, "sched_getaffinity", lambda _: set(range(have)))
        assert b._jobs() == want
