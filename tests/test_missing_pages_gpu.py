"""GPU tests of page numbers that are none: an entry of a table is data, and whatever it holds no kernel follows it."""
import pytest
import torch

from tests.paged_cases import Batch, check, paged_reference
from tests.test_paged_gpu import append_reference, attend, prefix_reference

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


def _spoil(table, n_pages, keep):
    """Entries that are no pages, of every kind, in turn: one of three columns, rows and columns counted together."""
    bad = [-1, n_pages, n_pages + 1, MOST, -MOST - 1, -n_pages, 1 << 24, -(1 << 30)]
    flat = table.view(-1)
    for x, i in enumerate(range(keep, flat.numel(), 3)):
        flat[i] = bad[x % len(bad)]


# one token each; several rows for the few-rows kernel; single and double tiles of many rows, their keys split and not
@pytest.mark.parametrize("new,past,Hq,Hk,D,page", [
    ([1] * 5, [700, 16, 17, 0, 3000], 28, 4, 128, 16),
    ([2, 1, 0, 2], [700, 160, 17, 3000], 8, 1, 64, 32),
    ([40, 1, 100], [900, 160, 3000], 2, 2, 64, 16),
    ([300, 1, 130], [900, 160, 3000], 28, 4, 128, 64),
])
@pytest.mark.parametrize("keep", [0, 1, 2])
def test_attention_and_append(kernels, new, past, Hq, Hk, D, page, keep):
    b = Batch(new, [n + p for n, p in zip(new, past)], Hq, Hk, D, page, seed=90 + keep)
    _spoil(b.table, b.cache_k.shape[0], keep)
    for window, sinks in ((0, 0), (100, 20)):
        ref, tol = paged_reference(b, window, sinks)
        check(attend(kernels, b, cu_tokens=b.cu, max_tokens=max(new), window=window, sinks=sinks), ref, tol)
    qkv = torch.randn(b.T, (Hq + 2 * Hk) * D, device="cuda").to(torch.bfloat16)
    inv = torch.rand(D // 2, device="cuda")
    was = [c.clone() for c in (b.cache_k, b.cache_v)]
    q = kernels.paged_kv_append(qkv, None, inv, b.cache_k, b.cache_v, b.table, b.seq_lens, *b.heads, cu_tokens=b.cu)
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).cuda()
    ref, tol = append_reference(qkv, None, inv, pos, Hq, Hk, D)
    check(q.view(-1, Hq, D), ref[:, :Hq], tol[:, :Hq])
    at = b.table[seq, pos // page].long()
    there = (at >= 0) & (at < b.cache_k.shape[0])
    at, slot = at[there], pos[there] % page
    for cache, old, h in ((b.cache_k, was[0], Hq), (b.cache_v, was[1], Hq + Hk)):
        check(cache[at, :, slot], ref[there, h:h + Hk], tol[there, h:h + Hk])
        old[at, :, slot] = cache[at, :, slot]
        assert torch.equal(torch.nan_to_num(cache, 99.0), torch.nan_to_num(old, 99.0))  # nothing else was written


# the prefix as one tile of rows, as several, and through the kernel for many
@pytest.mark.parametrize("B,prefix,own,Hq,Hk,D,page", [
    (2, 900, [70, 200], 28, 4, 128, 16),
    (6, 300, [70, 20, 1, 300, 0, 33], 28, 4, 128, 16),
    (20, 4000, [70, 20, 1, 300] * 5, 28, 4, 128, 64),
    (3, 700, [70, 20, 300], 40, 2, 64, 32),
])
@pytest.mark.parametrize("keep", [0, 1, 2])
def test_shared_prefix(kernels, B, prefix, own, Hq, Hk, D, page, keep):
    b = Batch([0] + [1] * B, [prefix] + own, Hq, Hk, D, page, seed=95 + keep)
    n_pages = b.cache_k.shape[0]
    table, b.table, b.seq_lens, b.lens = b.table[0, :-(-prefix // page)].contiguous(), b.table[1:].contiguous(), b.seq_lens[1:], own
    _spoil(table, n_pages, keep)
    _spoil(b.table, n_pages, keep)
    plen = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    ref, tol = prefix_reference(b, table, prefix)
    check(kernels.shared_prefix_attention(b.q, b.cache_k, b.cache_v, table, plen, b.table, b.seq_lens, *b.heads), ref, tol)
