"""GPU tests of the operators of batched serving called by several host threads at once."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _at_once(*runs):
    """Every run in a thread of its own, started together; raises what a thread raised."""
    go, errors = threading.Barrier(len(runs)), []

    def body(run):
        go.wait()
        try:
            run()
        except Exception as e:  # noqa: BLE001 (told by the caller's thread)
            errors.append(e)

    threads = [threading.Thread(target=body, args=(r,)) for r in runs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]


@pytest.mark.parametrize("dtype,sizes", [(torch.bfloat16, (152064, 40000)), (torch.float32, (131072, 36000))])
def test_vocabularies_of_different_sizes_at_once(kernels, dtype, sizes):
    """Two threads sample rows that take the same kernel with different amounts of shared memory."""
    runs = []
    for i, V in enumerate(sizes):
        logits = torch.randn(1, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(dtype)
        u = torch.zeros(1, device="cuda")
        want = int(logits[0].double().argmax())
        logits[0, want] += 8  # (the only one of its value)

        def run(logits=logits, u=u, want=want):
            out = [kernels.sample(logits, u, temperature=0.0) for _ in range(2000)]
            assert torch.equal(torch.cat(out).cpu(), torch.full((2000,), want))
        runs.append(run)
    torch.cuda.synchronize()
    _at_once(*runs)
