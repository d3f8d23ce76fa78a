"""GPU tests of several sequences at once: append, attention over the paged cache and behind a shared prefix, and sampling as they
are used together.  Each call inside a run is compared with its definition in 64 bits on the inputs that it had there: whole runs
on random weights with unit norm gains amplify a row's rounding to several percent of the logits (of either path, the
single-sequence runner's too), so two paths' logits say little about a kernel."""
import pytest
import torch

from nanoserve_b200.batch import Batch
from nanoserve_b200.qwen import Qwen2Config, Qwen2Runner
from tests.paged_cases import BF16_STEP, attention_64, check, tolerance
from tests.test_sample_gpu import reference as sampled

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def runner(kernels):
    cfg = Qwen2Config(hidden=512, n_layers=2, n_heads=14, n_kv_heads=2, head_dim=64, intermediate=1024, vocab=1024)
    return Qwen2Runner(cfg, kernels, torch.device("cuda"), max_len=600, norm_gain=1.0)


def ids(n, seed):
    return torch.randint(0, 1024, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


class Checked:
    """The kernels, each call of an operator of batched serving compared with its definition."""

    def __init__(self, k):
        self.k, self.calls = k, {}

    def __getattr__(self, name):
        return getattr(self.k, name)

    def _count(self, name):
        self.calls[name] = self.calls.get(name, 0) + 1

    def paged_kv_append(self, qkv, bias, inv_freq, ck, cv, table, lens, Hq, Hk, D, cu_tokens=None):
        q = self.k.paged_kv_append(qkv, bias, inv_freq, ck, cv, table, lens, Hq, Hk, D, cu_tokens=cu_tokens)
        self._count("append")
        x = (qkv.double() + bias.double()).view(-1, Hq + 2 * Hk, D)
        size = (qkv.double().abs() + bias.double().abs()).view(-1, Hq + 2 * Hk, D)
        row = 0
        for b, (n, length) in enumerate(zip(self._new(lens, cu_tokens), lens.tolist())):
            pos = torch.arange(length - n, length, device="cuda")
            a = torch.outer(pos.double(), inv_freq.double())[:, None]
            z, s = x[row:row + n], size[row:row + n]
            lo, hi = z[..., :D // 2], z[..., D // 2:]
            rot = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)
            ref = torch.cat([rot[:, :Hq + Hk], z[:, Hq + Hk:]], 1)
            tol = BF16_STEP * ref.abs() + 2.0 ** -20 * (s[..., :D // 2] + s[..., D // 2:]).repeat(1, 1, 2) + 1e-30
            page, slot = table[b].long()[pos // ck.shape[2]], pos % ck.shape[2]
            got = torch.cat([q[row:row + n].view(n, Hq, D), ck[page, :, slot], cv[page, :, slot]], 1)
            check(got, ref, tol)
            row += n
        return q

    @staticmethod
    def _new(lens, cu):
        return [1] * lens.numel() if cu is None else (cu[1:] - cu[:-1]).tolist()

    def _sequence(self, cache, table, n):
        j = torch.arange(n, device="cuda")
        return cache[table.long()[j // cache.shape[2]], :, j % cache.shape[2]].transpose(0, 1).double()

    def _compare(self, q, out, keys, values, first, D):
        n, L = q.shape[0], keys.shape[1]
        seen = torch.arange(L, device="cuda")[None] <= first + torch.arange(n, device="cuda")[:, None]
        ref, size, most = attention_64(q.double().view(n, -1, D), keys, values, seen, D ** -0.5)
        check(out, ref.view(n, -1), tolerance(ref, size, most, D).view(n, -1))

    def paged_attention(self, q, ck, cv, table, lens, Hq, Hk, D, cu_tokens=None, max_tokens=None):
        out = self.k.paged_attention(q, ck, cv, table, lens, Hq, Hk, D, cu_tokens=cu_tokens, max_tokens=max_tokens)
        self._count("attention")
        row = 0
        for b, (n, length) in enumerate(zip(self._new(lens, cu_tokens), lens.tolist())):
            self._compare(q[row:row + n], out[row:row + n], self._sequence(ck, table[b], length),
                          self._sequence(cv, table[b], length), length - n, D)
            row += n
        return out

    def shared_prefix_attention(self, q, ck, cv, prefix_table, prefix_len, table, lens, Hq, Hk, D):
        out = self.k.shared_prefix_attention(q, ck, cv, prefix_table, prefix_len, table, lens, Hq, Hk, D)
        self._count("prefix")
        P = int(prefix_len)
        for b, length in enumerate(lens.tolist()):
            both = [torch.cat([self._sequence(c, prefix_table, P), self._sequence(c, table[b], length)], 1) for c in (ck, cv)]
            self._compare(q[b:b + 1], out[b:b + 1], *both, P + length - 1, D)
        return out

    def sample(self, logits, u, out=None, **kw):
        self.k.sample(logits, u, out=out, **kw)
        self._count("sample")
        x, v = logits.double().cpu().numpy(), u.double().tolist()
        f32 = lambda t: float(torch.tensor(t, dtype=torch.float32))
        assert out.tolist() == [sampled(x[b], v[b], f32(kw["temperature"]), kw["top_k"], f32(kw["top_p"]), f32(kw["min_p"]))
                                for b in range(len(x))]
        return out


@pytest.mark.parametrize("prefix,prompts,page", [(200, [5, 0, 33, 1], 16), (64, [3, 20], 64), (0, [7, 30, 2], 32), (129, [0], 64),
                                                 (300, [1] * 12, 32)])
@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(temperature=0.9, top_k=100, top_p=0.9)])
def test_a_run_of_all_four(runner, prefix, prompts, page, settings):
    n_new = 5
    b = Batch(runner, len(prompts), 300, 80, page=page)
    pre, own = ids(prefix, 1), [ids(n, 2 + i) for i, n in enumerate(prompts)]
    got = b.generate(pre, own, n_new, **settings)
    assert b.generate(pre, own, n_new, **settings) == got  # (the same graph, after another prefill)
    checked = b.k = Checked(b.k)
    assert b.generate(pre, own, n_new, use_graph=False, **settings) == got
    layers, shared = runner.cfg.n_layers, b.shared > 0
    assert checked.calls["append"] == layers * (n_new + shared) and checked.calls["sample"] == n_new
    assert checked.calls.get("prefix", 0) == layers * (n_new - 1) * shared
    assert checked.calls["attention"] == layers * (1 + shared + (n_new - 1) * (not shared))


def test_one_sequence_follows_the_single_sequence_runner(kernels):
    """With the runner's own small norm gains, where a row's rounding stays one: the same greedy tokens."""
    cfg = Qwen2Config(hidden=512, n_layers=2, n_heads=14, n_kv_heads=2, head_dim=64, intermediate=1024, vocab=1024)
    r = Qwen2Runner(cfg, kernels, torch.device("cuda"), max_len=600)
    prompt = ids(150, 9)
    want = r.generate(prompt, 12)
    got = Batch(r, 3, 128, 64).generate(prompt, [ids(0, 1)] * 3, 12, temperature=0.0)
    assert got == [want] * 3


def test_equal_prompts_and_numbers_draw_equal_tokens(runner):
    """What a sequence draws depends on its own numbers alone."""
    B, n_new = 6, 12
    b = Batch(runner, B, 128, 64)
    pre = ids(100, 5)
    u = torch.rand(n_new, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).expand(-1, B)
    got = b.generate(pre, [ids(4, 7)] * B, n_new, temperature=1.0, top_k=200, top_p=0.95, u=u)
    assert all(g == got[0] for g in got) and len(set(got[0])) > 1
    other = b.generate(pre, [ids(4, 7)] * B, n_new, temperature=1.0, top_k=200, top_p=0.95, seed=3)
    assert len({tuple(g) for g in other}) > 1


def test_refusals(runner):
    b = Batch(runner, 2, 64, 32)
    with pytest.raises(ValueError):
        b.generate(ids(10, 1), [ids(1, 2)], 3)
    with pytest.raises(ValueError):
        b.generate(ids(10, 1), [ids(1, 2)] * 2, 33)
    with pytest.raises(ValueError):
        b.generate(ids(10, 1), [ids(120, 2)] * 2, 20)
    with pytest.raises(ValueError):
        b.generate(ids(0, 1), [ids(1, 2), ids(0, 3)], 2)


def test_rows_without_a_token_go_on(runner):
    """-1 (a row whose logits were not numbers) is no row of the embedding: such a sequence goes on from token 0."""
    b = Batch(runner, 3, 64, 8, page=16)
    b.u.fill_(0.5)
    b.prefill(ids(40, 1), [ids(3, 2 + i) for i in range(3)])
    lens, step_no = b.lens.clone(), b.step_no.clone()
    b.last[1] = 0
    b.step()
    want = b.tokens[1].tolist()
    b.lens.copy_(lens)
    b.step_no.copy_(step_no)
    b.last.copy_(b.tokens[0])
    b.last[1] = -1
    b.step()
    assert b.tokens[1].tolist() == want
    torch.cuda.synchronize()


def test_steps_end_with_the_room(runner):
    b = Batch(runner, 2, 64, 4, page=16)
    with pytest.raises(ValueError):
        b.step()
    b.prefill(ids(40, 1), [ids(3, 2), ids(1, 3)])
    for _ in range(3):
        b.step()
    with pytest.raises(ValueError):  # (four tokens are drawn)
        b.step()
    b.prefill(ids(33, 1), [ids(18, 2), ids(1, 3)])  # 19 of a sequence's 32 slots are taken, one token is drawn
    assert b.left == 3
    b.generate(ids(40, 1), [ids(3, 2), ids(1, 3)], 4)
    assert b.left == 0
    b.prefill(ids(33, 1), [ids(31, 2), ids(1, 3)])  # (32 of 32)
    with pytest.raises(ValueError):
        b.step()
