"""sample_tokens on the device against the definition: sizes, layouts, rows whose order has many equal entries, captured calls, other streams."""
import pytest
import torch

import _sample_oracle as oracle

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _rows(kind, B, V, dtype, lead=0, pad=0):
    r = torch.randn(B, V, device="cuda")
    r = {"random": 3 * r, "flat": 0.01 * r, "equal": torch.zeros_like(r), "two": (r > 1).float(), "far": 1e4 * r, "narrow": 100 + 0.1 * r,
         "masked": torch.where(torch.rand_like(r) < 0.9, -INF, 2 * r), "lowest": torch.where(torch.rand_like(r) < 0.9, torch.finfo(dtype).min, 2 * r)}[kind]
    x = torch.full((B, lead + V + pad), NAN, device="cuda").to(dtype)                # nothing beside a row is looked at
    x[:, lead:lead + V] = r.to(dtype)
    x[:, lead + V // 2] = 0.0
    return x[:, lead:lead + V]


def _check(x, u, **c):
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    n = _lib.launch_count()
    got = ops.sample_tokens(x, u, **c)
    assert _lib.launch_count() == n + 1 and got.shape == (x.shape[0], 1) and got.dtype is torch.int64
    assert got.flatten().tolist() == oracle.tokens(x, u, **c)


CHOICES = [{}, dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=2000, top_p=0.5), dict(top_k=20, top_p=0.75, min_p=0.125, temperature=0.5),
           dict(top_p=0.999, temperature=4.0)]


@pytest.mark.parametrize("kind", ["random", "flat", "equal", "two", "far", "narrow", "masked", "lowest"])
@pytest.mark.parametrize("choice", CHOICES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_kinds_of_rows(kind, choice, dtype, kernel_status):
    _check(_rows(kind, 3, 5003, dtype, 3, 5), torch.rand(3, device="cuda"), **choice)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 511, 512, 513, 2048, 4095, 4097, 50257])
@pytest.mark.parametrize("lead", [0, 1, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(V, lead, dtype):
    x, u = _rows("random", 2, V, dtype, lead, 3), torch.rand(2, device="cuda")
    for c in ({}, dict(top_k=3), dict(top_k=max(2, V - 1)), dict(top_p=0.6)):
        _check(x, u, **c)


def test_the_largest_vocabulary_and_a_larger_one():
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import sampling

    for V in (1 << 20, (1 << 20) + 1):
        x, u = torch.randn(2, V, device="cuda"), torch.rand(2, device="cuda")
        assert torch.equal(ops.sample_tokens(x, u, top_p=0.8), sampling._sample_ref(x, u, 1.0, 0, 0.8, 0.0))


def test_choices_of_each_row_and_rows_without_probabilities():
    x = _rows("random", 9, 700, torch.bfloat16)
    x[1, [5, 60]], x[2, [8, 9]], x[3] = NAN, INF, -INF
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t = lambda v: torch.tensor(v, device="cuda")  # noqa: E731
    _check(x, t([0.0, 0.5, 0.5, 0.5, 0.25, 1 - 2.0 ** -24, 0.5, 0.75, 0.125]),
           temperature=t([1.0, 1.0, 1.0, 1.0, 0.0, 0.5, 2.0, 1e-3, 0.75]), top_k=ints([0, 0, 9, 3, 2, 600, 1, 800, 30]),
           top_p=t([1.0, 0.5, 1.0, 0.5, 0.5, 0.75, 0.5, 1.0, 0.25]), min_p=t([0.0, 0.0, 0.5, 0.0, 0.0, 2.0 ** -10, 0.5, 1.0, 0.0]))


def test_rows_behind_32_bit_offsets():
    free = torch.cuda.mem_get_info()[0]
    if free < 12 << 30:
        pytest.skip("not enough memory")
    x = torch.empty(3, (1 << 30) + 64, dtype=torch.bfloat16, device="cuda")[:, :1000]
    x.copy_(torch.randn(3, 1000, device="cuda"))
    _check(x, torch.rand(3, device="cuda"), top_p=0.9)


def test_captured_on_another_stream_and_twice_at_once():
    from ghost_flow_b200 import ops

    x, u, k = _rows("random", 4, 3001, torch.float32), torch.rand(4, device="cuda"), torch.full((4,), 40, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, b = ops.sample_tokens(x, u, top_k=k), ops.sample_tokens(x, u, top_p=0.5)
    other = ops.sample_tokens(x, u, 0.5)
    torch.cuda.synchronize()
    assert a.flatten().tolist() == oracle.tokens(x, u, top_k=k) and b.flatten().tolist() == oracle.tokens(x, u, top_p=0.5)
    assert other.flatten().tolist() == oracle.tokens(x, u, 0.5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = ops.sample_tokens(x, u, top_k=k), ops.next_tokens(x, 0.7, top_p=0.9)
    x.copy_(_rows("random", 4, 3001, torch.float32))
    u.uniform_()
    k.fill_(7)
    g.replay()
    assert a.flatten().tolist() == oracle.tokens(x, u, top_k=k) and ((b >= 0) & (b < 3001)).all()


def test_what_a_gradient_or_a_trace_follows_takes_other_operations():
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    x, u = torch.randn(2, 90, device="cuda", requires_grad=True), torch.rand(2, device="cuda")
    n = _lib.launch_count()
    assert ops.sample_tokens(x, u, 0.5, 10).flatten().tolist() == oracle.tokens(x, u, 0.5, 10)
    assert ops.sample_tokens(x.detach().t().contiguous().t(), u, 0.5).flatten().tolist() == oracle.tokens(x, u, 0.5)
    assert _lib.launch_count() == n


@pytest.mark.parametrize("V", [23999, 24000, 32003, 50257, 128256])
@pytest.mark.parametrize("cuts", [{}, dict(top_k=50), dict(top_k=900), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.999), dict(top_k=64, top_p=0.5), dict(min_p=0.05),
                                  dict(top_p=0.8, min_p=0.02)], ids=lambda k: "-".join(k) or "none")
def test_a_row_has_one_token_however_many_rows_there_are(V, cuts):
    """Rows of a few are read by several blocks each, rows of many by one: the same token of either, of rows without probabilities and of equal entries too."""
    from ghost_flow_b200 import ops

    x = _rows("random", 200, V, torch.bfloat16, 0, 5).clone()
    x[3], x[5, 7], x[8, V - 1], x[11], x[14, V // 3:], x[17, : V // 2] = -INF, NAN, INF, 1.5, -INF, 20.0
    x[20] *= 1e-3
    x[23] *= 50
    u = torch.rand(200, device="cuda")
    u[:4] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.5, 0.25])
    all_ = ops.sample_tokens(x, u, 0.9, **cuts)
    for n in (1, 5, 13, 30, 60, 120):
        for at in (0, 2, 80):
            assert torch.equal(ops.sample_tokens(x[at:at + n], u[at:at + n], 0.9, **cuts), all_[at:at + n]), (n, at)
    for row in (0, 1, 3, 5, 8, 11, 14, 17, 20, 23, 30):
        assert torch.equal(ops.sample_tokens(x[row:row + 1], u[row:row + 1], 0.9, **cuts), all_[row:row + 1]), row


@pytest.mark.parametrize("kw", [{}, dict(top_k=5), dict(top_p=0.5), dict(min_p=0.9), dict(top_p=0.7, min_p=0.3)], ids=lambda k: "-".join(k) or "none")
def test_temperatures_without_end_and_the_least(kw):
    """At an infinite temperature what has a probability has the same; what has none still has none. At the least one the likeliest share it."""
    from ghost_flow_b200 import ops

    x = torch.tensor([[-INF, 2.0, -INF, 1.0, -3.0, -INF, 0.5, 7.0]], device="cuda").repeat(64, 1)
    u = (torch.arange(64, device="cuda") + 0.5) / 64
    order = [7, 1, 3, 6, 4]
    kept = order[:3] if kw.get("top_p") == 0.5 else order[:4] if kw.get("top_p") == 0.7 else order
    want = [sorted(kept)[int(v * len(kept))] for v in u.tolist()]
    for t in (INF, torch.full((64,), INF, device="cuda"), 3e38, 1e38):
        assert ops.sample_tokens(x, u, t, **kw).flatten().tolist() == want, t
    for t in (1e-45, 1e-60, torch.full((64,), 1e-45, device="cuda")):
        assert ops.sample_tokens(x, u, t, **kw).flatten().tolist() == [7] * 64


def test_numbers_have_64_bits():
    """A temperature or a share that is no number of 32 bits is taken as it is: the border of the second of two tokens lies between its neighbours."""
    from ghost_flow_b200 import ops

    x = torch.tensor([[0.0, 0.0, -INF]], device="cuda")
    for p, want in ((0.5, 0), (0.5 + 2.0 ** -40, 1)):           # of 32 bits both are a half
        assert ops.sample_tokens(x, torch.tensor([0.75], device="cuda"), 1.0, 0, p).item() == want
