"""Tests that need the reference's compiled code skip where it was not built, and only those."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))

BODY = '''
import pytest
import __graft_entry__

@pytest.fixture
def lib():
    oracle = __graft_entry__.load_oracle()
    return oracle._load("/nowhere/libgqa_ref_layer.so")

def test_in_body():
    oracle = __graft_entry__.load_oracle()
    oracle._load("/nowhere/libgqa_ref_layer.so")

def test_in_fixture(lib):
    pass

def test_another_file():
    open("/nowhere/else")

def test_that_fails():
    assert False
'''


def test_only_a_missing_reference_is_skipped(tmp_path):
    with open(os.path.join(HERE, "conftest.py")) as f:
        conftest = f.read().replace("os.path.abspath(__file__)", repr(os.path.join(HERE, "x")))
    (tmp_path / "conftest.py").write_text(conftest)
    (tmp_path / "test_it.py").write_text(BODY)
    out = subprocess.run([sys.executable, "-m", "pytest", "-q", "-rsf", "-p", "no:cacheprovider",
                          str(tmp_path)], capture_output=True, text=True, cwd=tmp_path).stdout
    assert "2 failed, 2 skipped" in out, out
    assert "libgqa_ref_layer.so not built" in out
    for name in ("test_another_file", "test_that_fails"):
        assert f"FAILED test_it.py::{name}" in out, out


def test_the_restatement_is_not_the_reference(orc):
    """The oracle's own library missing is an error, not a reason to skip."""
    saved = orc.ORACLE_SO
    try:
        orc.ORACLE_SO = "/nowhere/liboracle.so"
        try:
            orc._load(orc.ORACLE_SO)
        except FileNotFoundError as e:
            assert not isinstance(e, orc.ReferenceMissing)
        else:
            raise AssertionError("loaded a file that is not there")
    finally:
        orc.ORACLE_SO = saved
