"""Checks against the reference's own CPU build, where it is not there."""
import pytest

import conftest


def _outcome(error):
    call = conftest.pytest_runtest_call(None)
    next(call)
    call.throw(error)


def test_absent_reference_skips(oracle, monkeypatch, tmp_path):
    monkeypatch.setattr(oracle, "REF_DIR", tmp_path)
    with pytest.raises(RuntimeError, match="not built") as absent:
        oracle.load_ref("lp")
    with pytest.raises(pytest.skip.Exception, match="not built"):
        _outcome(absent.value)


def test_other_errors_stay(oracle):
    with pytest.raises(RuntimeError, match="other"):
        _outcome(RuntimeError("other"))
