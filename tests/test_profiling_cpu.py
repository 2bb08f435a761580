"""CPU tier: a KernelTimer touches no native code of its own."""

import pytest

import ssm_scan
from ssm_scan import _abi, profiling


def test_a_timer_does_not_load_the_library(monkeypatch):
    def missing():
        raise RuntimeError("not built")

    monkeypatch.setattr(_abi, "_host", None)
    monkeypatch.setattr(_abi, "host", missing)
    monkeypatch.setattr(_abi, "lib", missing)
    with ssm_scan.KernelTimer() as t:
        assert profiling.active() is t
        with ssm_scan.KernelTimer():
            assert profiling.active() is not t
        assert profiling.active() is t
    assert profiling.active() is None


def test_a_library_loaded_within_a_timer_counts_it(monkeypatch):
    counts = []
    monkeypatch.setattr(_abi, "_host", None)
    with ssm_scan.KernelTimer():
        host = _abi.host()
        monkeypatch.setattr(_abi, "_host", type("Host", (), {"count_timers": staticmethod(counts.append)}))
        with pytest.raises(KeyError):
            with ssm_scan.KernelTimer():
                raise KeyError
    assert counts == [1, -1, -1]
    host.count_timers(-1)   # the one that was counted at its loading
