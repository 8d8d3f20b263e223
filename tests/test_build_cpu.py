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
