"""What happens where a bounded wait runs out, read from the kernels' sources: a run that shows it would be a broken kernel."""
import glob
import os
import re
import subprocess
import sys

import pytest

from nanoserve_b200 import build

SOURCES = {os.path.basename(f): open(f).read() for f in sorted(glob.glob(os.path.join(build.CSRC, "*.cu")))}
WAITING = sorted(n for n, s in SOURCES.items() if "mbar_wait" in s)


@pytest.mark.parametrize("name", [n for n in WAITING if n.startswith("paged_")])
def test_time_outs_of_the_paged_attention_are_recorded(name):
    """With no condition but the time-out itself: the word is part of the device image, so there is no call that runs without
    it (a first one, captured perhaps, before anything else of the library has run).  The status calls read and clear it."""
    s = SOURCES[name]
    assert re.search(r"^__device__ int g_timed_out;", s, re.M)
    assert len(re.findall(r"if \(tid == 0 && \*abort_flag\) g_timed_out = 1;", s)) == s.count("abort_flag = reinterpret_cast")
    assert "status" not in re.sub(r"//[^\n]*", "", s)
    reader = re.search(r"^int (\w+_timed_out)\(int dev, bool clear, int\* word\)", s, re.M).group(1)
    for call, clear in (("b2_device_status", "false"), ("b2_clear_status", "true")):
        body = SOURCES["capi.cu"].split(f"int {call}(void) {{")[1].split("\n}")[0]
        assert f"b2::{reader}(dev, {clear}, " in body


@pytest.mark.parametrize("name", [n for n in WAITING if n.startswith("paged_")])
def test_copies_of_the_paged_attention_land_behind_a_time_out(name):
    """Shared and tensor memory are not released under copies and products on their way: the loading warp issues none behind a
    wait that ran out (it could be thousands, into buffers whose barriers still count the last ones), and the CTA stays a while."""
    s = SOURCES[name]
    loader = s[s.index("// ------------------------------------------------------------ loads"):]
    end = "// -------------------------------------------------------------- products" if name == "paged_attention.cu" else \
        "// ------------------------------------------------------------ products"
    loader = loader[:loader.index(end)]
    waits = re.findall(r"^ *(\S.*mbar_wait\(.*)$", loader, re.M)
    assert len(waits) == (2 if name == "paged_attention.cu" else 1)
    for w in waits:
        assert re.match(r"if \(!__all_sync\(0xffffffffu, mbar_wait\(.*\)\)\) break;", w), w
    after = s[s.index("g_timed_out = 1;"):]
    assert re.match(r"g_timed_out = 1;\n  if \(\*abort_flag\)(?: \{)?\n    for \(int i = 0; i < 64; \+\+i\) __nanosleep\(2000\);", after)
    assert "tmem_dealloc" not in s[:s.index("g_timed_out = 1;")]


FIRST = """
import torch
from nanoserve_b200.ops import Kernels
k = Kernels()
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
cache, table, heads = (r(8, 2, 64, 64), r(8, 2, 64, 64)), ints(*range(8)).view(2, 4), (4, 2, 64)
q, n, cu, lens = r(100, 256), r(2, 256), ints(0, 60, 100), ints(200, 100)
run = lambda: (k.paged_attention(n, *cache, table, lens, *heads), k.paged_attention(q, *cache, table, lens, *heads, cu_tokens=cu))
assert k.device_status() == 0  # (nothing has run yet)
k.clear_status()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
free = torch.cuda.mem_get_info()[0]
assert k.device_status() == 0
k.clear_status()
assert k.device_status() == 0 and torch.cuda.mem_get_info()[0] == free  # (read and cleared without the library's state)
"""


@pytest.mark.gpu
def test_status_of_a_first_call_without_the_librarys_state(kernels):
    """Attention as the first call of a process, captured, without b2_init: the status calls answer, and make nothing."""
    done = subprocess.run([sys.executable, "-c", FIRST], cwd=build.ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
