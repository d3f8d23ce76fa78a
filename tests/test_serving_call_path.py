"""The native host side of the operators of batched serving: the same answers as through ctypes, and what it hands back."""
import shutil

import pytest
import torch

from nanoserve_b200 import ops


@pytest.fixture
def call(lib_path):
    """The extension, built with the library on demand; missing only where there is no g++ to build it."""
    if not ops._find_call():
        if shutil.which("g++"):
            pytest.fail("nanoserve_call.so was not built or does not load")
        pytest.skip("no g++ to build the extension")


def _serving_args(B=3, Hq=4, Hk=2, D=64, page=16):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    caches = (r(9, Hk, page, D), r(9, Hk, page, D))
    return r, ints, caches, torch.arange(9, device="cuda", dtype=torch.int32).view(3, 3), ints(5, 40, 33), (Hq, Hk, D)


@pytest.mark.gpu
def test_serving_calls_answer_as_through_ctypes(kernels, call):
    slow = ops.Kernels()
    slow._append = slow._attend = slow._prefix = slow._sample = None
    assert None not in (kernels._append, kernels._attend, kernels._prefix, kernels._sample)
    r, ints, caches, table, lens, heads = _serving_args()
    qkv, q, bias = r(3, 512), r(7, 256), r(512)
    inv = torch.rand(32, device="cuda")
    for cu, x in ((None, qkv), (ints(0, 2, 2, 3), qkv)):
        both = []
        for k in (kernels, slow):
            c = tuple(t.clone() for t in caches)
            out = torch.zeros(3, 264, dtype=torch.bfloat16, device="cuda")[:, :256]
            a = k.paged_kv_append(x, bias, inv, *c, table, lens, *heads, cu_tokens=cu)
            assert k.paged_kv_append(x, None, inv, *c, table, lens, *heads, cu_tokens=cu, q_out=out) is out
            both.append((a, out, *c))
        assert all(torch.equal(a, b) for a, b in zip(*both))
    for kw in (dict(cu_tokens=ints(0, 2, 5, 7)), dict(cu_tokens=ints(0, 2, 5, 7), max_tokens=3, window=9, sinks=2, scale=0.3)):
        a, b = (k.paged_attention(q, *caches, table, lens, *heads, **kw) for k in (kernels, slow))
        assert torch.equal(a, b) and a.dtype == torch.bfloat16 and a.shape == (7, 256)
    args = (q[:3], *caches, ints(1, 2), ints(20), table, lens, *heads)
    assert torch.equal(kernels.shared_prefix_attention(*args), slow.shared_prefix_attention(*args))
    logits, u = r(3, 777), torch.rand(3, device="cuda")
    for kw in (dict(), dict(temperature=0.5, top_k=20, top_p=0.8, min_p=0.01), dict(temperature=1, top_p=1),
               dict(top_k=ints(5, 0, 70), temperature=torch.rand(3, device="cuda"), top_p=torch.rand(3, device="cuda"))):
        a, b = (k.sample(logits, u, **kw) for k in (kernels, slow))
        assert torch.equal(a, b) and a.dtype == torch.int64


def test_serving_calls_hand_back_what_they_do_not_take(call):
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for name, n in (("paged_kv_append", 13), ("paged_attention", 16), ("shared_prefix_attention", 14), ("sample", 8)):
        fn = ops._serving[name]
        for args in [(), (1,), (1,) * n, (1, 1) + (x,) * (n - 2), (None,) * n]:
            assert fn(*args) is NotImplemented
