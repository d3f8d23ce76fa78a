"""GPU tests of the paged cache's append and of attention over it, against plain forms in 64 bits."""
import pytest
import torch

from tests.paged_cases import BF16_STEP, Batch, attention_64, check, paged_reference, tolerance

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- append
def append_reference(qkv, bias, inv_freq, positions, Hq, Hk, D):
    """[T, heads, D] in 64 bits, and its tolerance: the angle's reduction is rounded to 32 bits (2^-24 of pi, in sin and cos,
    which are themselves good to 2^-22), four products and sums in 32 bits, one rounding to bf16."""
    x = qkv.double() + (0 if bias is None else bias.double())
    x = x.view(-1, Hq + 2 * Hk, D)
    size = (qkv.double().abs() + (0 if bias is None else bias.double().abs())).view(-1, Hq + 2 * Hk, D)
    a = torch.outer(positions.double(), inv_freq.double())[:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    rot = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)
    ref = torch.cat([rot[:, :Hq + Hk], x[:, Hq + Hk:]], 1)
    both = (size[..., :D // 2] + size[..., D // 2:]).repeat(1, 1, 2)
    return ref, BF16_STEP * ref.abs() + 2.0 ** -20 * both + 1e-30


@pytest.mark.parametrize("new,past,Hq,Hk,D,page,order,with_bias", [
    ([1], [0], 4, 1, 128, 16, "hsd", True),
    ([1, 1, 1], [0, 31, 700], 28, 4, 128, 16, "hsd", True),
    ([5, 1, 0, 40], [0, 15, 9, 60], 8, 8, 64, 32, "shd", False),
    ([130, 7], [3, 1 << 20], 6, 2, 80, 1024, "hsd", True),
    ([3, 300], [0, 0], 3, 1, 256, 256, "shd", True),
])
def test_append(kernels, new, past, Hq, Hk, D, page, order, with_bias):
    b = Batch(new, [n + p for n, p in zip(new, past)], Hq, Hk, D, page, seed=len(new), order=order, extra_rows=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    W = (Hq + 2 * Hk) * D
    wide = torch.randn(b.T, W + 8, device="cuda", generator=g).to(torch.bfloat16)
    qkv = wide[:, :W]
    bias = torch.randn(W, device="cuda", generator=g).to(torch.bfloat16) if with_bias else None
    inv_freq = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").float() / D))
    q_out = torch.full((b.T, Hq * D + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    before = wide.clone()
    want_k, want_v = b.cache_k.clone(), b.cache_v.clone()
    got = kernels.paged_kv_append(qkv, bias, inv_freq, b.cache_k, b.cache_v, b.table, b.seq_lens, Hq, Hk, D, cu_tokens=b.cu,
                                  q_out=q_out[:, :Hq * D])
    assert got.data_ptr() == q_out.data_ptr() and torch.equal(before, wide)
    n = sum(new)
    pos = torch.cat([torch.arange(p, p + m, device="cuda") for m, p in zip(new, past)])
    ref, tol = append_reference(qkv[:n], bias, inv_freq, pos, Hq, Hk, D)
    check(q_out[:n, :Hq * D].reshape(n, Hq, D), ref[:, :Hq], tol[:, :Hq])
    assert (q_out[n:] == 7.0).all() and (q_out[:, Hq * D:] == 7.0).all()  # rows behind the last sequence, columns beside
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    pages = b.table[seq, pos // page].long()
    check(b.cache_k[pages, :, pos % page], ref[:, Hq:Hq + Hk], tol[:, Hq:Hq + Hk])
    check(b.cache_v[pages, :, pos % page], ref[:, Hq + Hk:], tol[:, Hq + Hk:])
    for cache, want in ((b.cache_k, want_k), (b.cache_v, want_v)):  # nothing else of the cache is touched
        cache[pages, :, pos % page] = 0
        want[pages, :, pos % page] = 0
        assert torch.equal(torch.nan_to_num(cache, 99.0), torch.nan_to_num(want, 99.0))


def test_append_leaves_out_what_has_no_place(kernels):
    """Rows at negative positions, pages that are not there (-1, too large, beyond the table's width)."""
    Hq, Hk, D, page = 4, 2, 64, 16
    b = Batch([4, 2, 2, 2], [2, 20, 20, 200], Hq, Hk, D, page, spare_width=0)
    b.table[1, 1] = -1
    b.table[2, 1] = 1 << 30
    b.table = b.table[:, :2].contiguous()  # the last sequence's positions lie beyond it
    W = (Hq + 2 * Hk) * D
    qkv = torch.randn(b.T, W, device="cuda").to(torch.bfloat16)
    inv_freq = torch.rand(D // 2, device="cuda")
    q_out = torch.full((b.T, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    k0, v0 = b.cache_k.clone(), b.cache_v.clone()
    kernels.paged_kv_append(qkv, None, inv_freq, b.cache_k, b.cache_v, b.table, b.seq_lens, Hq, Hk, D, cu_tokens=b.cu, q_out=q_out)
    pos = torch.tensor([-2, -1, 0, 1, 18, 19, 18, 19, 198, 199], device="cuda")
    ref, tol = append_reference(qkv, None, inv_freq, pos, Hq, Hk, D)
    assert (q_out[:2] == 7.0).all()
    check(q_out[2:].view(-1, Hq, D), ref[2:, :Hq], tol[2:, :Hq])
    page0 = int(b.table[0, 0])
    check(b.cache_k[page0, :, :2].transpose(0, 1), ref[2:4, Hq:Hq + Hk], tol[2:4, Hq:Hq + Hk])
    k0[page0, :, :2], v0[page0, :, :2] = b.cache_k[page0, :, :2], b.cache_v[page0, :, :2]
    assert torch.equal(torch.nan_to_num(b.cache_k, 99.0), torch.nan_to_num(k0, 99.0))
    assert torch.equal(torch.nan_to_num(b.cache_v, 99.0), torch.nan_to_num(v0, 99.0))


# ---------------------------------------------------------------- attention
def attend(kernels, b, **kw):
    out = torch.full((b.T, b.Hq * b.D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = kernels.paged_attention(b.q, b.cache_k, b.cache_v, b.table, b.seq_lens, *b.heads, out=out, **kw)
    assert got.data_ptr() == out.data_ptr()
    return out


@pytest.mark.parametrize("lens,Hq,Hk,D,page,window,sinks,order", [
    ([1], 28, 4, 128, 16, 0, 0, "hsd"),
    ([0, 1, 2], 4, 4, 64, 16, 0, 0, "hsd"),
    ([700], 28, 4, 128, 16, 512, 4, "hsd"),
    ([5, 0, 333, 64, 65, 1024], 28, 4, 128, 64, 0, 0, "shd"),
    ([15, 16, 17, 127, 128, 129, 4000], 64, 8, 128, 32, 100, 4, "hsd"),
    ([300, 41, 2000], 16, 1, 64, 128, 1, 0, "hsd"),
    ([300, 41, 2000], 16, 2, 64, 1024, 64, 70, "shd"),
    ([257] * 40, 8, 2, 128, 16, 0, 0, "hsd"),
    ([3, 900], 32, 1, 128, 16, 64, 1, "hsd"),  # more query heads per key head than a tile of sixteen rows
    ([20000, 30, 5000], 28, 4, 128, 256, 0, 0, "hsd"),
    ([20000, 30, 5000], 7, 1, 128, 256, 4096, 300, "hsd"),
])
def test_attention_one_token_each(kernels, lens, Hq, Hk, D, page, window, sinks, order):
    b = Batch([1] * len(lens), lens, Hq, Hk, D, page, seed=len(lens), order=order)
    ref, tol = paged_reference(b, window, sinks)
    out = attend(kernels, b, window=window, sinks=sinks)
    check(out, ref, tol)
    assert torch.equal(out, attend(kernels, b, window=window, sinks=sinks))
    assert torch.equal(out, attend(kernels, b, window=window, sinks=sinks, cu_tokens=b.cu, max_tokens=1))


@pytest.mark.parametrize("new,past,Hq,Hk,D,page,window,sinks,order", [
    ([2], [0], 4, 4, 64, 16, 0, 0, "hsd"),
    ([3, 1, 0, 2], [0, 40, 7, 500], 4, 1, 128, 16, 0, 0, "hsd"),
    ([9, 1, 5], [100, 2000, 0], 28, 4, 128, 32, 64, 4, "shd"),
    ([128], [0], 7, 1, 128, 128, 0, 0, "hsd"),
    ([513, 1, 77], [0, 900, 333], 28, 4, 128, 64, 0, 0, "hsd"),
    ([513, 1, 77], [5, 900, 333], 16, 2, 64, 64, 100, 4, "shd"),
    ([300], [700], 8, 8, 64, 16, 1, 0, "hsd"),
    ([300], [700], 8, 8, 128, 16, 130, 129, "hsd"),
    ([1200, 40, 3], [0, 0, 3000], 28, 4, 128, 256, 256, 1, "hsd"),
    ([150, 700], [2000, 1], 64, 8, 128, 1024, 0, 0, "hsd"),
    ([700], [5000], 3, 3, 64, 32, 1000, 64, "hsd"),
    ([1, 0, 200], [6000, 0, 100], 32, 1, 64, 16, 0, 0, "hsd"),
])
def test_attention_several_tokens(kernels, new, past, Hq, Hk, D, page, window, sinks, order):
    b = Batch(new, [n + p for n, p in zip(new, past)], Hq, Hk, D, page, seed=len(new), order=order, extra_rows=3)
    ref, tol = paged_reference(b, window, sinks)
    n = sum(new)
    for bound in (None, max(new)):
        out = attend(kernels, b, window=window, sinks=sinks, cu_tokens=b.cu, max_tokens=bound)
        check(out[:n], ref[:n], tol[:n])
        assert (out[n:] == 7.0).all()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [4, 4, 40, 300]])
def test_attention_rows_and_pages_that_see_nothing(kernels, new):
    """Sequences shorter than their rows (negative positions), of no token, with pages that are not there; a page that is not
    there in the middle; every visible page gone."""
    lens = [0, max(1, new[1] - 2), 200, 400]
    b = Batch(new, lens, 14, 2, 128, 16, seed=3)
    b.table[2, 0] = -1
    b.table[2, 5] = 1 << 30
    b.table[3] = -1
    ref, tol = paged_reference(b)
    out = attend(kernels, b, cu_tokens=b.cu)
    check(out, ref, tol)
    assert (out[:new[0]] == 0).all() and (out[-new[3]:] == 0).all()
    # the table ends before the sequence does
    b = Batch(new, [50, 60, 700, 900], 14, 2, 128, 16, seed=4)
    b.table = b.table[:, :6].contiguous()
    ref, tol = paged_reference(b)
    check(attend(kernels, b, cu_tokens=b.cu), ref, tol)


def test_attention_large_scores_and_scale(kernels):
    """Scores of some hundreds: the running maximum carries them; one key takes all."""
    for new in ([1, 1], [70, 200]):
        b = Batch(new, [300, 900], 4, 2, 64, 32, seed=5)
        b.q *= 30
        for scale in (1.0, 0.01):
            ref, tol = paged_reference(b, 128, 2, scale=scale)
            check(attend(kernels, b, cu_tokens=b.cu, window=128, sinks=2, scale=scale), ref, tol)


@pytest.mark.parametrize("new", [[1, 1], [64, 200]])
def test_one_key_far_above_the_others(kernels, new):
    """One key, at every place of a block in turn, whose scores are hundreds of powers of two above all others: it takes all."""
    b = Batch(new, [400, 600], 2, 1, 64, 128, seed=14)
    q = torch.zeros_like(b.q.view(b.T, 2, 64))
    q[..., 0] = 30.0  # rows score the keys' first column alone
    b.q = q.view(b.T, -1)
    plain_k = b.cache_k.clone()
    for j in list(range(130, 258)):
        b.cache_k = plain_k.clone()
        for i in range(2):
            b.cache_k[int(b.table[i, j // 128]), :, j % 128, 0] = 20.0
        out = attend(kernels, b, cu_tokens=b.cu, scale=1.0).view(b.T, 2, 64)
        for i in range(2):
            v = b.cache_v[int(b.table[i, j // 128]), 0, j % 128]
            rows = slice(b.starts[i], b.starts[i] + new[i])
            assert ((out[rows].float() - v.float()).abs() <= BF16_STEP * v.float().abs()).all(), (j, i)


def test_attention_strided_rows(kernels):
    """q as a view of the projection's rows, out as a view of a wider buffer."""
    for new in ([1, 1, 1], [30, 1, 100]):
        b = Batch(new, [200, 300, 111], 8, 2, 128, 16, seed=6)
        wide = torch.full((b.T, 12 * 128), 3.0, dtype=torch.bfloat16, device="cuda")
        wide[:, :1024] = b.q
        out = torch.full((b.T, 1032), 7.0, dtype=torch.bfloat16, device="cuda")
        kernels.paged_attention(wide[:, :1024], b.cache_k, b.cache_v, b.table, b.seq_lens, *b.heads, cu_tokens=b.cu,
                                out=out[:, :1024])
        ref, tol = paged_reference(b)
        check(out[:, :1024], ref, tol)
        assert (out[:, 1024:] == 7.0).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 40, 200]])
def test_attention_of_rows_that_are_not_numbers(kernels, new):
    """A row of q that holds a nan, or an infinity against finite keys, is not a number; no other row notices."""
    b = Batch(new, [100, 300, 500], 14, 2, 128, 32, seed=8)
    want = attend(kernels, b, cu_tokens=b.cu)
    row = new[0] + new[1] - 1  # the second sequence's last
    b.q[row, 5 * 128 + 3] = float("nan")
    b.q[row, 9 * 128 + 7] = float("inf")
    got = attend(kernels, b, cu_tokens=b.cu).view(b.T, 14, 128)
    hit = torch.zeros(b.T, 14, dtype=torch.bool, device="cuda")
    hit[row, 5] = hit[row, 9] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want.view(b.T, 14, 128)[~hit])


@pytest.mark.parametrize("new,most", [([2, 1, 2], 1), ([5, 300, 20], 16), ([300, 20, 700], 130)])
def test_rows_in_front_of_the_first_and_beyond_max_tokens(kernels, new, most):
    b = Batch(new, [400, 700, 900], 7, 1, 64, 64, seed=10, extra_rows=1)
    ref, tol = paged_reference(b)
    start = 4  # rows in front of the first sequence
    b.q = torch.cat([b.q.new_full((start, 7 * 64), 5.0), b.q])
    b.cu, b.T = b.cu + start, b.T + start
    out = attend(kernels, b, cu_tokens=b.cu, max_tokens=most)
    kept = torch.zeros(b.T, dtype=torch.bool, device="cuda")
    for n, s in zip(new, b.starts):
        kept[start + s:start + s + min(n, most)] = True
    check(out[kept], ref[kept[start:]], tol[kept[start:]])
    assert (out[~kept] == 7.0).all()
    q_out = torch.full((b.T, 7 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kernels.paged_kv_append(torch.ones(b.T, 9 * 64, dtype=torch.bfloat16, device="cuda"), None, torch.zeros(32, device="cuda"),
                            b.cache_k, b.cache_v, b.table, b.seq_lens, 7, 1, 64, cu_tokens=b.cu, q_out=q_out)
    assert (q_out[:start] == 7.0).all() and (q_out[start:-1] == 1.0).all() and (q_out[-1:] == 7.0).all()


def test_long_sequences_split_over_many_ctas(kernels):
    """One sequence whose keys all SMs share, for few rows and for many; a short chunk behind a long context."""
    for new, window in ((1, 0), (2, 0), (64, 0), (64, 30000)):
        b = Batch([new], [70001], 4, 1, 64, 256, seed=12)
        ref, tol = paged_reference(b, window, 5)
        check(attend(kernels, b, cu_tokens=b.cu, window=window, sinks=5), ref, tol)


def test_many_sequences(kernels):
    """More sequences than a warp has lanes, than lengths are kept, empty ones among them."""
    for B in (33, 129, 300):
        g = torch.Generator().manual_seed(B)
        lens = torch.randint(0, 200, (B,), generator=g).tolist()
        b = Batch([1] * B, lens, 4, 2, 64, 16, seed=B)
        ref, tol = paged_reference(b)
        check(attend(kernels, b), ref, tol)
        new = torch.randint(0, 12, (B,), generator=g).tolist()
        b = Batch(new, [n + x for n, x in zip(new, lens)], 4, 2, 64, 16, seed=B)
        ref, tol = paged_reference(b)
        check(attend(kernels, b, cu_tokens=b.cu), ref, tol)
        check(attend(kernels, b, cu_tokens=b.cu, max_tokens=12), ref, tol)


def test_output_in_place_of_q(kernels):
    for new in ([1, 1], [70, 300]):
        b = Batch(new, [500, 600], 8, 2, 128, 64, seed=13)
        want = attend(kernels, b, cu_tokens=b.cu)
        got = kernels.paged_attention(b.q, b.cache_k, b.cache_v, b.table, b.seq_lens, *b.heads, cu_tokens=b.cu, out=b.q)
        assert torch.equal(got, want)


# ---------------------------------------------------------------- shared prefix
def prefix_reference(b, prefix_table, prefix_len, scale=None):
    scale = b.D ** -0.5 if scale is None else scale
    q = b.q.double().view(b.T, b.Hq, b.D)
    ref, tol = torch.zeros_like(q), torch.zeros_like(q)
    pk, pv, p_there = b.sequence(prefix_table, max(prefix_len, 1))
    for i, length in enumerate(b.lens):
        k, v, there = b.sequence(b.table[i], max(length, 1))
        k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        p_seen = p_there & (torch.arange(p_there.numel(), device=q.device) < prefix_len)
        seen = torch.cat([p_seen, there & (torch.arange(there.numel(), device=q.device) < length)])[None]
        ref[i:i + 1], size, most = attention_64(q[i:i + 1], k, v, seen, scale)
        tol[i:i + 1] = tolerance(ref[i:i + 1], size, most, b.D)
    return ref.view(b.T, -1), tol.view(b.T, -1)


@pytest.mark.parametrize("B,prefix,own,Hq,Hk,D,page", [
    (1, 1, [1], 4, 4, 64, 16),
    (3, 0, [5, 1, 40], 28, 4, 128, 16),
    (3, 777, [5, 0, 200], 28, 4, 128, 16),
    (16, 2000, list(range(1, 17)), 28, 4, 128, 64),
    (17, 2049, [3] * 17, 8, 1, 64, 32),
    (64, 5003, [1, 70, 300, 17] * 16, 28, 4, 128, 128),
    (5, 129, [600, 1, 2, 3, 4], 32, 1, 128, 1024),
    (40, 4096, [33] * 40, 64, 8, 128, 256),
    (300, 700, [9, 0, 1] * 100, 2, 2, 64, 16),
    (2, 30000, [1, 2], 28, 4, 128, 256),
])
def test_shared_prefix(kernels, B, prefix, own, Hq, Hk, D, page):
    # the prefix is sequence 0 of the cache; its table is cut off, so it may end inside a page
    b = Batch([0] + [1] * B, [prefix] + own, Hq, Hk, D, page, seed=B, order="shd" if B % 2 else "hsd")
    table, b.table, b.seq_lens, b.lens = b.table[0, :max(1, -(-prefix // page))].contiguous(), b.table[1:], b.seq_lens[1:], own
    plen = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    ref, tol = prefix_reference(b, table, prefix)
    args = (b.cache_k, b.cache_v, table, plen, b.table, b.seq_lens, *b.heads)
    out = kernels.shared_prefix_attention(b.q, *args)
    check(out, ref, tol)
    assert torch.equal(out, kernels.shared_prefix_attention(b.q, *args))
    # pages of the prefix that are not there, a length beyond its table
    if prefix > 500:
        table[1] = -1
        table[2] = 1 << 29
        plen += 100
        # (behind the prefix's end its last page holds nothing: fill it)
        last = int(table[-1])
        for c in (b.cache_k, b.cache_v):
            c[last] = torch.nan_to_num(c[last], 0.5)
        ref, tol = prefix_reference(b, table, min(prefix + 100, table.numel() * page))
        check(kernels.shared_prefix_attention(b.q, *args), ref, tol)


def test_shared_prefix_equals_attention_over_aliased_tables(kernels):
    """The same pages in front of every sequence's own: one paged_attention call gives the same values."""
    B, prefix, page, Hq, Hk, D = 6, 640, 64, 28, 4, 128
    b = Batch([0] + [1] * B, [prefix] + [10 * i + 1 for i in range(B)], Hq, Hk, D, page, seed=9)
    plen = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    both = torch.cat([b.table[:1, :prefix // page].expand(B, -1), b.table[1:]], 1).contiguous()
    one = kernels.paged_attention(b.q, b.cache_k, b.cache_v, both, b.seq_lens[1:] + prefix, Hq, Hk, D)
    two = kernels.shared_prefix_attention(b.q, b.cache_k, b.cache_v, b.table[0, :prefix // page].contiguous(), plen, b.table[1:],
                                          b.seq_lens[1:].contiguous(), Hq, Hk, D)
    table, b.table, b.lens = b.table[0, :prefix // page], b.table[1:], b.lens[1:]
    ref, tol = prefix_reference(b, table, prefix)
    check(one, ref, tol)
    check(two, ref, tol)


# ---------------------------------------------------------------- how they are called
def test_captured_and_replayed(kernels):
    """One graph holds append and attention; the lengths grow on the device between replays.  Two graphs in turn."""
    Hq, Hk, D, page, B = 28, 4, 128, 16, 3
    b = Batch([1] * B, [40, 100, 7], Hq, Hk, D, page, seed=11, spare_width=4)
    for r in range(B):  # room for the tokens to come
        b.table[r] = torch.arange(r * b.table.shape[1], (r + 1) * b.table.shape[1])
    n_pages = int(b.table.max()) + 1
    b.cache_k = torch.randn(n_pages, Hk, page, D, device="cuda").to(torch.bfloat16)
    b.cache_v = torch.randn(n_pages, Hk, page, D, device="cuda").to(torch.bfloat16)
    W = (Hq + 2 * Hk) * D
    qkv = torch.randn(B, W, device="cuda").to(torch.bfloat16)
    inv_freq = 1.0 / (1e4 ** (torch.arange(0, D, 2, device="cuda").float() / D))

    def step():
        q = kernels.paged_kv_append(qkv, None, inv_freq, b.cache_k, b.cache_v, b.table, b.seq_lens, Hq, Hk, D)
        return q, kernels.paged_attention(q, b.cache_k, b.cache_v, b.table, b.seq_lens, Hq, Hk, D, window=64, sinks=2)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        step()
        torch.cuda.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                graphs.append((g, step()))
            torch.cuda.synchronize()
        for i in range(6):
            b.seq_lens += 1
            b.lens = b.seq_lens.tolist()
            qkv.copy_(torch.randn(B, W, device="cuda"))
            g, (q, out) = graphs[i % 2]
            g.replay()
            torch.cuda.synchronize()
            b.q = q
            ref, tol = paged_reference(b, 64, 2)
            check(out, ref, tol)


def test_two_streams_at_once(kernels):
    """Calls on different streams that overlap have scratch of their own."""
    bs = [Batch([1] * 3, [5000, 3000 + i, 100], 28, 4, 128, 64, seed=20 + i) for i in range(2)]
    want = [attend(kernels, b) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, b) in enumerate(zip(streams, bs)):
            with torch.cuda.stream(s):
                got[i].append(attend(kernels, b))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_offsets_beyond_32_bits(kernels):
    """A cache whose last pages start beyond 2^32 elements: pages 5 GB apart, three of them."""
    Hq, Hk, D, page = 8, 2, 128, 64
    far = 2_400_000_000  # elements from page to page
    store = torch.empty(2 * far + 2 * Hk * page * D, dtype=torch.bfloat16, device="cuda")
    shape, stride = (3, Hk, page, D), (far, page * D, D, 1)
    cache_k = store.as_strided(shape, stride)
    cache_v = store[Hk * page * D:].as_strided(shape, stride)
    for new in ([1, 1], [60, 100]):
        b = Batch(new, [60, 120], Hq, Hk, D, page, seed=7, spare_width=0)
        for c, big in ((b.cache_k, cache_k), (b.cache_v, cache_v)):
            for col, p in ((0, 2), (1, 1)):
                big[p].copy_(c[int(b.table[1, col])])
            big[0].copy_(c[int(b.table[0, 0])])
        ref, tol = paged_reference(b)
        table = torch.tensor([[0, -1], [2, 1]], dtype=torch.int32, device="cuda")
        out = kernels.paged_attention(b.q, cache_k, cache_v, table, b.seq_lens, Hq, Hk, D, cu_tokens=b.cu)
        check(out, ref, tol)
        n = b.T
        qkv = torch.randn(n, (Hq + 2 * Hk) * D, device="cuda").to(torch.bfloat16)
        kernels.paged_kv_append(qkv, None, torch.zeros(D // 2, device="cuda"), cache_k, cache_v, table, b.seq_lens, Hq, Hk, D,
                                cu_tokens=b.cu)
        assert torch.equal(cache_v[1, :, 119 - 64], qkv[-1].view(-1, D)[Hq + Hk:])
        assert torch.equal(cache_k[0, :, 59], qkv[new[0] - 1].view(-1, D)[Hq:Hq + Hk])


@pytest.mark.parametrize("new", [[1, 1], [64, 200]])
def test_large_values_under_a_jump_of_the_scores(kernels, new):
    """Values of 2^85 and a key, behind the first blocks, whose weight is some 2^50 times theirs: the sums stay finite."""
    b = Batch(new, [400, 600], 4, 2, 64, 64, seed=15)
    q = torch.zeros(b.T, 4, 64, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 4.0  # rows score the keys' first column alone: up to some 4 * 4, and 12 * 4 at that key
    b.q = q.view(b.T, -1)
    for i in range(2):
        b.cache_k[int(b.table[i, 200 // 64]), :, 200 % 64, 0] = 12.0
    b.cache_v *= 2.0 ** 85
    ref, tol = paged_reference(b, scale=1.0)
    out = attend(kernels, b, cu_tokens=b.cu, scale=1.0)
    check(out, ref, tol)


def test_no_sequence(kernels):
    """A call without sequences answers with nothing."""
    b = Batch([1, 1], [20, 30], 4, 2, 64, 16, seed=16)
    none = lambda t: t[:0]
    plen = torch.tensor([16], dtype=torch.int32, device="cuda")
    args = (b.cache_k, b.cache_v, b.table[0], plen, none(b.table), none(b.seq_lens), *b.heads)
    assert kernels.shared_prefix_attention(none(b.q), *args).shape == (0, 4 * 64)
    args = (b.cache_k, b.cache_v, none(b.table), none(b.seq_lens), *b.heads)
    assert kernels.paged_attention(none(b.q), *args).shape == (0, 4 * 64)
    qkv = torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device="cuda")
    assert kernels.paged_kv_append(qkv, None, torch.zeros(32, device="cuda"), *args).shape == (0, 4 * 64)


def test_many_rows_and_prefixes_on_streams_and_in_graphs(kernels):
    """Prompts, split prompts and shared prefixes: two streams that overlap, and two graphs of each, replayed in turn on two
    streams with other lengths than at their capture, give the bits of single calls."""
    prompts = [Batch([300, 1, 64], [300, 900 + i, 5000], 28, 4, 128, 64, seed=30 + i) for i in range(2)]
    tails = [Batch([0] + [1] * 20, [4000 + 64 * i] + [30 + i] * 20, 28, 4, 128, 64, seed=40 + i) for i in range(2)]
    few = [Batch([0] + [1] * 2, [3000 + 64 * i] + [300, 20 + i], 14, 2, 64, 64, seed=50 + i) for i in range(2)]

    def prompt(b):
        return attend(kernels, b, cu_tokens=b.cu)

    def prefix(b):
        return kernels.shared_prefix_attention(b.q, b.cache_k, b.cache_v, b.table[0], b.seq_lens[:1], b.table[1:], b.seq_lens[1:],
                                               *b.heads)

    runs = [lambda i, f=f, bs=bs: f(bs[i]) for f, bs in ((prompt, prompts), (prefix, tails), (prefix, few))]
    want = [[run(i) for i in range(2)] for run in runs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for r, run in enumerate(runs):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got.append((r, i, run(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[r][i]) for r, i, o in got)
    # captured with shorter lengths
    batches, lens = [prompts, tails, few], [[b.seq_lens.clone() for b in bs] for bs in (prompts, tails, few)]
    for bs in batches:
        for b in bs:
            b.seq_lens.copy_((b.seq_lens - 7).clamp(min=1))
    graphs = []
    torch.cuda.synchronize()
    for r, run in enumerate(runs):
        for i, s in enumerate(streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = run(i)
            graphs.append((r, i, g, out))
    for bs, ls in zip(batches, lens):
        for b, n in zip(bs, ls):
            b.seq_lens.copy_(n)
    torch.cuda.synchronize()
    for _ in range(4):
        for r, i, g, _ in graphs:
            with torch.cuda.stream(streams[i]):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[r][i]) for r, i, _, out in graphs)


@pytest.mark.parametrize("B,prefix,own,Hq,Hk,D,page,spare", [
    (3, 200, [1, 64, 65], 9, 1, 128, 16, 0),       # a sequence to a tile
    (5, 300, [0, 2, 70, 5, 1], 16, 1, 64, 32, 0),
    (18, 190, [3] * 18, 28, 4, 128, 16, 0),        # 126 rows; 19 sequences: 133
    (19, 190, [3] * 19, 28, 4, 128, 16, 0),
    (33, 100, [7, 0, 130] * 11, 2, 2, 64, 16, 0),  # sixteen sequences to a tile
    (4, 500, [700, 1, 90, 5], 64, 8, 128, 64, 0),  # both kernels beside one another
    (3, 777, [20, 30, 1], 28, 4, 128, 16, 400),    # wide tables, short sequences
    (3, 0, [20, 30, 0], 28, 4, 128, 16, 0),
])
def test_shared_prefix_in_several_tiles(kernels, B, prefix, own, Hq, Hk, D, page, spare):
    """Short prefixes, which tiles of sixteen rows read one by one."""
    b = Batch([0] + [1] * B, [prefix] + own, Hq, Hk, D, page, seed=60 + B, spare_width=spare)
    table, b.table, b.seq_lens, b.lens = b.table[0, :max(1, -(-prefix // page))].contiguous(), b.table[1:], b.seq_lens[1:], own
    plen = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    ref, tol = prefix_reference(b, table, prefix)
    wide = torch.full((b.T, Hq * D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (b.cache_k, b.cache_v, table, plen, b.table, b.seq_lens, *b.heads)
    out = kernels.shared_prefix_attention(b.q, *args, out=wide[:, :Hq * D])
    check(out, ref, tol)
    assert (wide[:, Hq * D:] == 7.0).all() and torch.equal(out, kernels.shared_prefix_attention(b.q, *args))


@pytest.mark.parametrize("B", [2, 9, 70])
def test_shared_prefix_without_a_page(kernels, B):
    """A prefix table of no page, whatever the length says: the own keys alone."""
    b = Batch([1] * B, [30 + i for i in range(B)], 28, 4, 128, 16, seed=80 + B)
    table = torch.empty(0, dtype=torch.int32, device="cuda")
    ref, tol = paged_reference(b)
    for length in (0, 50, -3):
        plen = torch.tensor([length], dtype=torch.int32, device="cuda")
        check(kernels.shared_prefix_attention(b.q, b.cache_k, b.cache_v, table, plen, b.table, b.seq_lens, *b.heads), ref, tol)
