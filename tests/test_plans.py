"""How the launchers of batched serving plan their work, read from the sources."""
import glob
import os
import re

import pytest

from nanoserve_b200 import build

SOURCES = sorted(glob.glob(os.path.join(build.CSRC, "paged*.cu*")) + [os.path.join(build.CSRC, "sample.cu")])


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_sms_are_counted_by_the_device(path):
    """A slice of a device has fewer of them: no plan holds their number."""
    code = re.sub(r"//[^\n]*", "", open(path).read())
    assert not re.search(r"\b(?:148|132|160)\b", code)


def test_sampling_rows_are_cut_up_for_one_wave():
    """Of CTAs that fill an SM each there are no more than SMs, except where a row's slice would not fit in shared memory."""
    source = open(os.path.join(build.CSRC, "sample.cu")).read()
    rule = re.search(r"while \((C < 8 && .*)\) C \*= 2;", source).group(1)
    rule = rule.replace("&&", "and").replace("||", "or").replace("p.", "").replace("/", "//")
    slice_bytes = 150 * 1024
    assert "kSliceBytes = 150 * 1024;" in source
    for sm_count in (148, 37, 20):
        for rows in (1, 5, 18, 19, 20, 37, 64, 70, 74, 75, 100, 148, 1000):
            for V in (100, 4096, 12000, 40000, 152064, 262144):
                for size in (2, 4):
                    C = 1
                    while eval(rule, dict(C=C, rows=rows, V=V, row=V * size, sm_count=sm_count, kSliceBytes=slice_bytes)):
                        C *= 2
                    assert C <= 8 and (C == 1 or rows * C <= sm_count or V * size // (C // 2) > slice_bytes), (rows, V, size, C)
                    if C < 8 and V // C > 4096:
                        assert 2 * rows * C > sm_count
