"""Options that only some compilers know do not decide whether the library is built."""
import os

import pytest

from ai_amd import build as B

pytestmark = pytest.mark.skipif(not os.path.exists(B.HIPCC), reason="no compiler")


def test_options_of_one_compiler_are_left_out_by_others(monkeypatch, capsys):
    (source, flags), = B.SOURCE_FLAGS.items()
    assert B._known(flags) == flags
    unknown = ["-mllvm", "-amdgpu-of-another-version=1"]
    assert B._known(unknown) == [] and "of-another-version" in capsys.readouterr().err

    seen = []
    monkeypatch.setattr(B, "SOURCE_FLAGS", {source: unknown})
    monkeypatch.setattr(B, "_run", lambda cmd, verbose: seen.append(cmd))
    monkeypatch.setattr(os, "replace", lambda a, b: None)
    B.build_rocm()
    compiled, = [c for c in seen if any(x.endswith(os.sep + source) for x in c)]
    assert len(seen) == len(B.ROCM_SOURCES) + 1 and unknown[1] not in compiled and "-O3" in compiled
