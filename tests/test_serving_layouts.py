"""Layouts that the operators of batched serving take: the stride of a dimension of one says nothing."""
import ctypes

import pytest
import torch

from nanoserve_b200 import ops

A = 1 << 20  # an aligned address that nothing reads
BAD_SHAPE, BAD_POINTER = -1, -4


@pytest.mark.parametrize("stride", [0, 1, 7, 517, -8])
def test_one_row_and_one_head_of_any_stride(lib_path, stride):
    """Refused for the pointer, which is looked at behind the shapes; several rows or heads are refused for the stride."""
    lib = ops.load_library(lib_path)

    def calls(rows, n_pages, heads, **kw):
        d = dict(k=A, v=A, page_stride=512 * 64, head_stride=16 * 64, token_stride=64, n_pages=n_pages, page_size=16,
                 n_kv_heads=heads, head_dim=64, block_table=A, table_stride=8, table_width=8, n_seqs=rows, seq_lens=A)
        d.update({n: v for n, v in kw.items() if n in d})
        c, W = ctypes.byref(ops.PagedCache(**d)), 64 * heads
        s = lambda name, n: kw.get(name, n)
        return {lib.b2_paged_kv_append(A + 2, s("qkv", 3 * W), None, A, A, s("q", W), c, None, rows, heads, None),
                lib.b2_paged_attention(A + 2, s("q", W), c, None, rows, 1, heads, 0, 0, 0.1, A, s("out", W), A, 1 << 40, None),
                lib.b2_shared_prefix_attention(A + 2, s("q", W), c, A, 3, A, heads, 0.1, A, s("out", W), A, 1 << 40, None)}

    assert calls(1, 4, 2, qkv=stride, q=stride, out=stride) == {BAD_POINTER}
    assert calls(2, 4, 2, qkv=stride, q=stride, out=stride) == {BAD_SHAPE}
    assert calls(1, 1, 1, page_stride=stride, head_stride=stride) == {BAD_POINTER}
    assert calls(1, 4, 1, page_stride=stride) == calls(1, 1, 4, head_stride=stride) == {BAD_SHAPE}


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_contiguous_rows_with_a_stride_of_one(kernels, native):
    """A column turned into a row is contiguous to torch, and its row stride is 1; a cache of one head with any stride there."""
    k = kernels
    if not native:
        k = ops.Kernels()
        k._append = k._attend = k._prefix = k._sample = None
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    turned = lambda t: torch.empty(t.shape[1], 1, dtype=t.dtype, device="cuda").copy_(t.t()).t()  # [1, W] with strides (1, 1)
    Hq, Hk, D, page = 4, 1, 64, 16
    caches, odd = [r(9, Hk, page, D) for _ in range(2)], []
    for c in caches:
        odd.append(torch.empty(c.numel(), dtype=c.dtype, device="cuda").as_strided(c.shape, (page * D, 3, D, 1)))
        odd[-1].copy_(c)
    table, lens, heads = ints(*range(9))[None], ints(140), (Hq, Hk, D)
    qkv, inv = r(1, (Hq + 2 * Hk) * D), torch.rand(D // 2, device="cuda", generator=g)
    assert turned(qkv).stride() == (1, 1) and turned(qkv).is_contiguous()

    def run(qkv, caches, shape):
        q = k.paged_kv_append(qkv, None, inv, *caches, table, lens, *heads, q_out=shape(torch.zeros(1, Hq * D, dtype=qkv.dtype,
                                                                                                    device="cuda")))
        out = [k.paged_attention(shape(q), *caches, table, lens, *heads, out=shape(torch.zeros_like(q))),
               k.paged_attention(shape(q), *caches, table, lens, *heads, cu_tokens=ints(0, 1), max_tokens=200, window=30, sinks=2),
               k.shared_prefix_attention(shape(q), *caches, ints(3, 4), ints(20), table, lens, *heads, out=shape(torch.zeros_like(q)))]
        return [q, *out, *caches]

    want = run(qkv, caches, lambda t: t)
    got = run(turned(qkv), odd, turned)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_settings_beyond_an_int_of_c(kernels, native):
    """A window, first tokens, a bound of rows or a top-k of 2^32 and more leave all that there is."""
    k = kernels
    if not native:
        k = ops.Kernels()
        k._append = k._attend = k._prefix = k._sample = None
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    caches, table, lens, heads = (r(9, 2, 16, 64), r(9, 2, 16, 64)), ints(*range(9))[None], ints(140), (4, 2, 64)
    args, far = (r(5, 256), *caches, table, lens, *heads), 2 ** 32 + 1
    attend = lambda **kw: k.paged_attention(*args, cu_tokens=ints(0, 5), out=torch.zeros_like(args[0]), **kw)
    want = attend(max_tokens=5)
    assert torch.equal(attend(max_tokens=5, window=far), want)
    assert torch.equal(attend(max_tokens=5, window=3, sinks=far), attend(max_tokens=5, window=3, sinks=140))
    assert torch.equal(attend(max_tokens=far), attend(max_tokens=2 ** 31 - 1)) and (attend(max_tokens=far) != 0).any(1).all()
    logits, u = r(1, 999), torch.full((1,), 0.9, device="cuda")
    pick = lambda n: int(k.sample(logits, u, temperature=30.0, top_k=n))
    assert pick(0) != pick(1) and pick(far) == pick(0) == pick(-far) == pick(-2 ** 40)
    for bad in (dict(window=-far), dict(max_tokens=-far), dict(window=3, sinks=-far)):
        with pytest.raises(RuntimeError, match="b2_paged_attention failed with code -1"):
            attend(**bad)


def test_a_prefix_whose_blocks_31_bits_do_not_count(lib_path):
    """One tile of rows reads 2^24 blocks of 64 keys for each of 256 heads: 2^32, which would count as none."""
    lib = ops.load_library(lib_path)

    def call(heads, width):
        c = ops.PagedCache(k=A, v=A, page_stride=heads * 1024 * 64, head_stride=1024 * 64, token_stride=64, n_pages=4, page_size=1024,
                           n_kv_heads=heads, head_dim=64, block_table=A, table_stride=8, table_width=8, n_seqs=2, seq_lens=A)
        return lib.b2_shared_prefix_attention(A, heads * 64, ctypes.byref(c), A, width, A + 2, heads, 0.1, A, heads * 64, A, 1 << 40,
                                              None)

    assert call(256, 1 << 20) == call(128, 1 << 20) == -6
    assert call(256, 1 << 18) == call(64, 1 << 20) == BAD_POINTER  # (the length's address, which is looked at next)
