"""The kernel between logits and the choice of a token at the ends of its arguments' ranges."""
import pytest
import torch

import _paged_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("r", [2.0 ** -126, 3e-38, 2.0 ** 126, 5e37])
def test_repetitions_at_the_ends_of_their_range(r):
    from ghost_flow_b200 import ops

    x = torch.randn(2, 300) * torch.tensor([[1e-3], [1e30]])
    t = torch.randint(0, 300, (2, 90), dtype=torch.int32)
    want, off = oracle.logits(x, t, r=r)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * float("inf"), want)
    number = ops.process_logits(x.cuda(), t.cuda(), repetition=r)
    oracle.close(number, want, off)
    assert torch.equal(ops.process_logits(x.cuda(), t.cuda(), repetition=torch.tensor([r, r], device="cuda")), number)


@pytest.mark.parametrize("r", [1e-39, 2.0 ** 127])
def test_repetitions_beyond_it(r):
    from ghost_flow_b200 import ops

    with pytest.raises(ValueError, match="repetition"):
        ops.process_logits(torch.zeros(2, 8, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), repetition=r)


def test_vocabularies_of_other_threads(kernel_status):
    """Slices of other lengths want other amounts of shared memory, asked for at the same time."""
    import threading

    from ghost_flow_b200 import ops

    work = []
    for V in (4500, 9000, 17000, 17408, 23000, 34000, 50257, 128256):
        x = torch.randn(300, V, device="cuda").bfloat16()
        t = torch.randint(0, V, (300, 50), device="cuda", dtype=torch.int32)
        work.append((x, t))
    torch.cuda.synchronize()
    got, gate, failed = {}, threading.Barrier(len(work)), []

    def call(i):
        x, t = work[i]
        gate.wait()
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = ops.process_logits(x, t, repetition=1.5, presence=0.25)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=call, args=(i,)) for i in range(len(work))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    for i, (x, t) in enumerate(work):
        assert torch.equal(got[i], ops.process_logits(x, t, repetition=1.5, presence=0.25))
