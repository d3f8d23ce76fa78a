"""What the operators of batched serving refuse, through the C ABI (no GPU: refused before anything is launched) and through
`Kernels`; and that no page number from a table is used before it is compared."""
import ctypes
import glob
import os
import re

import pytest
import torch

from nanoserve_b200 import build, ops

A = 1 << 20  # an aligned address that nothing reads
BAD_SHAPE, BAD_POINTER, TOO_LARGE, WORKSPACE = -1, -4, -6, -5


def cache(**kw):
    d = dict(k=A, v=A, page_stride=4 * 16 * 128, head_stride=16 * 128, token_stride=128, n_pages=10, page_size=16, n_kv_heads=4,
             head_dim=128, block_table=A, table_stride=8, table_width=8, n_seqs=2, seq_lens=A)
    d.update(kw)
    return ctypes.byref(ops.PagedCache(**d))


@pytest.fixture(scope="module")
def lib(lib_path):
    return ops.load_library(lib_path)


CACHES = [(dict(page_size=12), BAD_SHAPE), (dict(page_size=8), BAD_SHAPE), (dict(page_size=2048), BAD_SHAPE),
          (dict(n_pages=0), BAD_SHAPE), (dict(n_seqs=0), BAD_SHAPE), (dict(table_width=0), BAD_SHAPE),
          (dict(token_stride=132), BAD_SHAPE), (dict(token_stride=64), BAD_SHAPE), (dict(head_stride=120), BAD_SHAPE),
          (dict(page_stride=-8), BAD_SHAPE), (dict(table_stride=7), BAD_SHAPE), (dict(n_kv_heads=0), BAD_SHAPE),
          (dict(k=A + 8), BAD_POINTER), (dict(v=0), BAD_POINTER), (dict(seq_lens=0), BAD_POINTER),
          (dict(block_table=A + 2), BAD_POINTER), (dict(table_width=1 << 27, table_stride=1 << 27), TOO_LARGE)]


def append(lib, c, **kw):
    d = dict(qkv=A, stride=36 * 128, bias=None, inv=A, q=A, q_stride=28 * 128, cu=None, T=2, Hq=28)
    d.update(kw)
    return lib.b2_paged_kv_append(d["qkv"], d["stride"], d["bias"], d["inv"], d["q"], d["q_stride"], c, d["cu"], d["T"], d["Hq"],
                                  None)


def attend(lib, c, **kw):
    d = dict(q=A, q_stride=28 * 128, cu=None, T=2, most=1, Hq=28, window=0, sinks=0, out=A, out_stride=28 * 128, ws=A, n=1 << 40)
    d.update(kw)
    return lib.b2_paged_attention(d["q"], d["q_stride"], c, d["cu"], d["T"], d["most"], d["Hq"], d["window"], d["sinks"], 0.1,
                                  d["out"], d["out_stride"], d["ws"], d["n"], None)


def prefix(lib, c, **kw):
    d = dict(q=A, q_stride=28 * 128, table=A, width=3, n=A, Hq=28, out=A, out_stride=28 * 128, ws=A, bytes=1 << 40)
    d.update(kw)
    return lib.b2_shared_prefix_attention(d["q"], d["q_stride"], c, d["table"], d["width"], d["n"], d["Hq"], 0.1, d["out"],
                                          d["out_stride"], d["ws"], d["bytes"], None)


@pytest.mark.parametrize("change,code", CACHES)
def test_caches(lib, change, code):
    assert append(lib, cache(**change)) == code
    assert attend(lib, cache(**change)) == code
    assert prefix(lib, cache(**change)) == code


def test_no_cache(lib):
    assert append(lib, None) == attend(lib, None) == prefix(lib, None) == BAD_POINTER


@pytest.mark.parametrize("kw,code", [
    (dict(T=3), BAD_SHAPE), (dict(T=0), BAD_SHAPE), (dict(Hq=0), BAD_SHAPE), (dict(stride=36 * 128 - 8), BAD_SHAPE),
    (dict(stride=36 * 128 + 4), BAD_SHAPE), (dict(q_stride=27 * 128), BAD_SHAPE), (dict(qkv=0), BAD_POINTER),
    (dict(qkv=A + 2), BAD_POINTER), (dict(bias=A + 8), BAD_POINTER), (dict(inv=None), BAD_POINTER), (dict(q=A + 4), BAD_POINTER),
    (dict(cu=A + 1), BAD_POINTER)])
def test_append(lib, kw, code):
    assert append(lib, cache(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(T=3), BAD_SHAPE), (dict(T=0), BAD_SHAPE), (dict(Hq=27), BAD_SHAPE), (dict(most=2), BAD_SHAPE), (dict(most=0), BAD_SHAPE),
    (dict(window=-1), BAD_SHAPE), (dict(sinks=-1), BAD_SHAPE), (dict(q_stride=28 * 128 + 4), BAD_SHAPE),
    (dict(out_stride=27 * 128), BAD_SHAPE), (dict(q=A + 8), BAD_POINTER), (dict(out=0), BAD_POINTER), (dict(cu=A + 2), BAD_POINTER)])
def test_attention(lib, kw, code):
    assert attend(lib, cache(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(Hq=27), BAD_SHAPE), (dict(width=-1), BAD_SHAPE), (dict(q_stride=8), BAD_SHAPE), (dict(table=None), BAD_POINTER),
    (dict(n=None), BAD_POINTER), (dict(n=A + 2), BAD_POINTER), (dict(q=None), BAD_POINTER), (dict(out=A + 2), BAD_POINTER),
    (dict(width=1 << 27), TOO_LARGE)])
def test_prefix(lib, kw, code):
    assert prefix(lib, cache(), **kw) == code


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf"), 3e38])
def test_scales(lib, scale):
    c = cache()
    assert lib.b2_paged_attention(A, 28 * 128, c, None, 2, 1, 28, 0, 0, scale, A, 28 * 128, A, 1 << 40, None) == BAD_SHAPE
    assert lib.b2_shared_prefix_attention(A, 28 * 128, c, A, 3, A, 28, scale, A, 28 * 128, A, 1 << 40, None) == BAD_SHAPE


def test_sizes_beyond_31_bits(lib):
    assert attend(lib, cache(n_seqs=1 << 26, table_stride=8), T=1 << 26) == TOO_LARGE
    assert attend(lib, cache(n_seqs=1 << 20, table_width=1 << 14, table_stride=1 << 14), T=1 << 20) == TOO_LARGE


def test_head_dims(lib):
    for D, both in ((96, BAD_SHAPE), (256, BAD_SHAPE), (80, BAD_SHAPE)):
        c = dict(head_dim=D, token_stride=D, head_stride=16 * D, page_stride=64 * D)
        assert attend(lib, cache(**c), q_stride=28 * D, out_stride=28 * D) == both
        assert prefix(lib, cache(**c), q_stride=28 * D, out_stride=28 * D) == both
    assert append(lib, cache(head_dim=72)) == BAD_SHAPE


def sample(lib, **kw):
    d = dict(logits=A, stride=100, fp32=0, rows=2, V=100, u=A, t=None, k=None, p=None, m=None, tokens=A)
    d.update(kw)
    return lib.b2_sample(d["logits"], d["stride"], d["fp32"], d["rows"], d["V"], d["u"], d["t"], d["k"], d["p"], d["m"], 1.0, 0, 1.0,
                         0.0, d["tokens"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), BAD_SHAPE), (dict(V=0), BAD_SHAPE), (dict(stride=-1), BAD_SHAPE), (dict(V=262145), TOO_LARGE),
    (dict(rows=(1 << 20) + 1), TOO_LARGE), (dict(logits=None), BAD_POINTER), (dict(logits=A + 2, fp32=1), BAD_POINTER),
    (dict(logits=A + 1), BAD_POINTER), (dict(u=None), BAD_POINTER), (dict(tokens=A + 4), BAD_POINTER), (dict(t=A + 2), BAD_POINTER),
    (dict(k=A + 1), BAD_POINTER), (dict(p=A + 2), BAD_POINTER), (dict(m=A + 3), BAD_POINTER)])
def test_sample(lib, kw, code):
    assert sample(lib, **kw) == code


def test_tensors_on_the_host_are_refused(lib_path):
    k = ops.Kernels(lib_path)
    c = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        k.paged_attention(torch.zeros(1, 64, dtype=torch.bfloat16), c, c, t, n, 1, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        k.paged_kv_append(torch.zeros(1, 192, dtype=torch.bfloat16), None, torch.zeros(32), c, c, t, n, 1, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        k.sample(torch.zeros(1, 8), torch.zeros(1))


@pytest.mark.gpu
def test_kernels_refuses(kernels):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")
    c, t, n, q = z(2, 1, 16, 64), z(1, 1, dtype=torch.int32), z(1, dtype=torch.int32), z(1, 64)
    kernels.paged_attention(q, c, c, t, n, 1, 1, 64)
    for bad in (dict(q=z(1, 64, dtype=torch.float16)), dict(q=z(2, 64)), dict(q=z(1, 128)), dict(k=z(2, 1, 16, 128)),
                dict(k=z(2, 1, 16, 64, dtype=torch.float32)), dict(t=z(1, 1, dtype=torch.int64)), dict(t=z(2, 1, dtype=torch.int32)),
                dict(n=z(1, dtype=torch.int64)), dict(n=z(1, 1, dtype=torch.int32)), dict(v=z(2, 16, 1, 64).transpose(1, 2)[:1]),
                dict(q=z(1, 128)[:, ::2])):
        d = dict(q=q, k=c, v=c, t=t, n=n)
        d.update(bad)
        with pytest.raises(ValueError):
            kernels.paged_attention(d["q"], d["k"], d["v"], d["t"], d["n"], 1, 1, 64)
    with pytest.raises(ValueError):
        kernels.paged_attention(q, c, c, t, n, 1, 1, 64, cu_tokens=z(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="b2_paged_attention failed with code -1"):
        kernels.paged_attention(q, c, c, t, n, 1, 1, 64, max_tokens=3)
    with pytest.raises(ValueError):
        kernels.paged_kv_append(z(1, 192), z(64), z(32, dtype=torch.float32), c, c, t, n, 1, 1, 64)
    with pytest.raises(ValueError):
        kernels.shared_prefix_attention(q, c, c, t, n, t, n, 1, 1, 64)
    with pytest.raises(ValueError):
        kernels.sample(z(2, 8), z(3, dtype=torch.float32))
    with pytest.raises(ValueError):
        kernels.sample(z(2, 8, dtype=torch.float16), z(2, dtype=torch.float32))
    with pytest.raises(ValueError):
        kernels.sample(z(2, 8), z(2, dtype=torch.float32), top_k=z(2, dtype=torch.int64))
    assert kernels.sample(z(0, 8), z(0, dtype=torch.float32)).numel() == 0


def test_no_page_number_is_used_unseen():
    """An entry of a table is data: every kernel that reads one compares it with the pages that there are."""
    files = [f for f in glob.glob(os.path.join(build.CSRC, "paged*.cu*"))]
    found = 0
    for f in files:
        text = open(f).read()
        for m in re.finditer(r"__ldcg\((?:c\.)?(?:\w+\.)?table", text):
            found += 1
            after = text[m.start():m.start() + 400]
            assert re.search(r"page < c\.n_pages|page >= c\.n_pages|< \(unsigned\)\w*\.?\w*n_pages|valid_page\(", after), (f, after[:120])
    assert found >= 1
