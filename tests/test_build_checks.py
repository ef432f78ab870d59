"""The build refuses kernels of certain sources that keep registers in memory."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _build():
    sys.path.insert(0, os.path.join(ROOT, "burn-gdn2_amd"))
    import build

    return build


def _remarks(name, size):
    return [f"x.hip:1:0: remark: Function Name: {name} [-Rpass-analysis=kernel-resource-usage]",
            f"x.hip:1:0: remark:     ScratchSize [bytes/lane]: {size} [-Rpass-analysis=kernel-resource-usage]"]


def test_remarks():
    build = _build()
    assert build.kernels_with_scratch(_remarks("a", 0) + _remarks("b", 16) + _remarks("c", 0)) == ["b"]
    for odd in ([], _remarks("a", 0)[:1], ["nothing"]):
        with pytest.raises(RuntimeError):
            build.kernels_with_scratch(odd)
    assert all(os.path.exists(os.path.join(ROOT, "burn-gdn2_amd", "csrc", n)) for n in build.NO_SCRATCH)


def test_a_source_with_scratch_is_refused(tmp_path):
    build = _build()
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    src = tmp_path / build.NO_SCRATCH[0]
    src.write_text('#include <hip/hip_runtime.h>\n'
                   '__global__ void k(int *p, int n) { int a[64]; for (int i = 0; i < 64; ++i) a[i] = p[i]; p[0] = a[n & 63] + a[p[n] & 63]; }\n')
    flags = [f for f in build.FLAGS if f != "-shared"]
    rc, msgs = build._compile(str(src), str(tmp_path / "k.o"), flags, False)
    assert rc != 0 and "keep registers in memory" in msgs[0]
    other = tmp_path / "other.hip"
    other.write_text(src.read_text())
    assert build._compile(str(other), str(tmp_path / "k.o"), flags, False)[0] == 0
