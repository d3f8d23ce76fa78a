"""The room that a batch of several sequences has."""
from types import SimpleNamespace

import pytest
import torch

from nanoserve_b200.batch import Batch
from nanoserve_b200.qwen import Qwen2Config, Qwen2Runner


class Counting:
    """Kernels of a pick on the host: the tokens drawn are the calls so far."""

    def __init__(self):
        self.calls = 0

    def lm_head(self, h, weight, logits):
        logits.zero_()

    def sample(self, logits, u, out, **sampling):
        assert u.shape == (logits.shape[0],)
        self.calls += 1
        out.fill_(self.calls)


def on_host(**cfg):
    d = dict(n_layers=1, n_heads=2, n_kv_heads=1, head_dim=64, vocab=32)
    d.update(cfg)
    return SimpleNamespace(cfg=SimpleNamespace(**d), world=1, dev=torch.device("cpu"), k=Counting(), lm_head=None)


def test_picks_beyond_the_room_write_the_last_row():
    """A captured step may be replayed once too often, when nothing on the host says so: an index beyond the rows would end in a
    device assertion."""
    b = Batch(on_host(), 2, max_prefix=0, max_own=3, page=16)
    for _ in range(5):
        b._pick(torch.zeros(2, 8))
    assert b.tokens.tolist() == [[1, 1], [2, 2], [5, 5]] and b.last.tolist() == [5, 5]


@pytest.mark.gpu
def test_a_captured_step_replayed_beyond_the_room(kernels):
    cfg = Qwen2Config(hidden=512, n_layers=2, n_heads=14, n_kv_heads=2, head_dim=64, intermediate=1024, vocab=1024)
    runner = Qwen2Runner(cfg, kernels, torch.device("cuda"), max_len=600, norm_gain=1.0)
    ids = lambda n, seed: torch.randint(0, 1024, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    prefix, prompts = ids(40, 1), [ids(3, 2), ids(9, 3)]
    b = Batch(runner, 2, max_prefix=64, max_own=12, page=16)
    b.sampling = dict(temperature=0.0)
    u = torch.zeros(12, 2, device="cuda")
    want = b.generate(prefix, prompts, 12, temperature=0.0, u=u, use_graph=False)
    with torch.cuda.stream(runner.stream):
        b.prefill(prefix, prompts)
        lens, step_no, last = b.lens.clone(), b.step_no.clone(), b.last.clone()
        b.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=runner.stream):
            b.step()
        b.lens.copy_(lens)
        b.step_no.copy_(step_no)
        b.last.copy_(last)
        for _ in range(11):
            graph.replay()
        torch.cuda.synchronize()
        assert b.tokens.T.tolist() == want
        for _ in range(40):  # (beyond its pages, too)
            graph.replay()
        torch.cuda.synchronize()
    assert b.tokens[:-1].T.tolist() == [w[:-1] for w in want]
    assert ((b.tokens >= 0) & (b.tokens < 1024)).all()
    runner.check_status()


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_seqs=-1), dict(max_own=0), dict(max_prefix=-1), dict(page=8), dict(page=48),
                                dict(page=2048), dict(head_dim=96)])
def test_sizes_that_a_batch_does_not_take(kw):
    """Refused when it is made: without a row of random numbers the first pick would end in a device assertion."""
    d = dict(n_seqs=2, max_prefix=64, max_own=3, page=16)
    runner = on_host(**{n: v for n, v in kw.items() if n == "head_dim"})
    d.update({n: v for n, v in kw.items() if n != "head_dim"})
    with pytest.raises(ValueError):
        Batch(runner, **d)
    Batch(on_host(), 1, 0, 1, page=1024)
