"""__graft_entry__.build() asks nothing of tests/: it makes the C++ programs that the Makefile there has, and no others.  The compilers of the
library and of the oracle are left out here; `make` runs over a folder of its own."""
import os

import pytest

import __graft_entry__ as entry
from mference_amd import _capi
from mference_amd import build as mf_build
from oracle import mf_oracle

RULE = "{0}:\n\ttouch {0}\n"


@pytest.fixture
def tree(tmp_path, monkeypatch):
    monkeypatch.setattr(mf_build, "build", lambda verbose=False: None)
    monkeypatch.setattr(mf_oracle, "build", lambda: None)
    monkeypatch.setattr(mf_oracle, "lib", lambda: None)
    monkeypatch.setattr(_capi, "lib", lambda: None)
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    return tmp_path


def _makefile(tree, *programs):
    cpp = tree / "tests" / "cpp"
    cpp.mkdir(parents=True)
    (cpp / "Makefile").write_text("".join(RULE.format(p) for p in programs))
    return cpp


def test_build_with_tests_that_lack_a_program(tree):
    cpp = _makefile(tree, "mirror_test")
    entry.build()
    assert os.path.exists(cpp / "mirror_test") and not os.path.exists(cpp / "adapters_test")


def test_build_with_all_programs(tree):
    cpp = _makefile(tree, "mirror_test", "adapters_test")
    entry.build()
    assert os.path.exists(cpp / "mirror_test") and os.path.exists(cpp / "adapters_test")


def test_build_with_a_program_whose_source_is_absent(tree):
    cpp = _makefile(tree, "mirror_test")
    with open(cpp / "Makefile", "a") as fh:
        fh.write("adapters_test: adapters_test.cpp\n\ttouch adapters_test\n")
    entry.build()
    assert os.path.exists(cpp / "mirror_test") and not os.path.exists(cpp / "adapters_test")


def test_build_with_a_program_that_only_makes_own_rules_know(tree):
    """a source without a rule in the Makefile: make would compile it by a rule of its own, which lacks the include paths"""
    cpp = _makefile(tree, "mirror_test")
    (cpp / "adapters_test.cpp").write_text('#include "mfmoe.hpp"\nint main() {}\n')
    entry.build()
    assert os.path.exists(cpp / "mirror_test") and not os.path.exists(cpp / "adapters_test")


def test_build_without_tests(tree):
    entry.build()


def test_build_reports_a_program_that_does_not_compile(tree):
    cpp = _makefile(tree)
    (cpp / "Makefile").write_text("mirror_test:\n\tfalse\n")
    with pytest.raises(Exception):
        entry.build()
