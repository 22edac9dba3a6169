"""bench.py's options of the paged cache and of penalties."""
import importlib
import sys

import pytest


@pytest.fixture
def run(monkeypatch):
    bench = importlib.import_module("bench")
    ran = []
    monkeypatch.setattr(bench, "run_model", ran.append)

    def call(*options):
        monkeypatch.setattr(sys, "argv", ["bench.py", "--workload", "model", *options])
        bench.main()
        return bench.cache_options(ran[-1]), ran[-1]
    return call


def test_options_of_the_paged_cache(run):
    assert run("--kv-page", "64")[0] == {"kv_page": 64, "window": 0, "sinks": 0}
    assert run("--kv-page", "16", "--window", "100", "--sinks", "4")[0] == {"kv_page": 16, "window": 100, "sinks": 4}
    assert run()[0] == {} and run()[1].repetition is None
    assert run("--repetition", "1.2")[1].repetition == 1.2


@pytest.mark.parametrize("options", [["--kv-page", "64", "--kv-bits", "4"], ["--kv-page", "64", "--kv-budget", "100"], ["--repetition", "0"]])
def test_what_does_not_go_together(run, options):
    with pytest.raises(SystemExit) as stop:
        run(*options)
    assert stop.value.code == 2
