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
