"""Kernels over a paged cache against the definitions in 64 bits: lengths, heads, pages, layouts, empty sequences, what lies around."""
import pytest
import torch

import _paged_oracle as oracle

pytestmark = pytest.mark.gpu

BATCHES = {"one": ([1], [1]), "two keys": ([2], [1]), "one each": ([1, 63, 64, 65, 128, 129, 300], [1] * 7),
           "empty slots": ([0, 17, 0, 130], [1, 1, 0, 1]), "prompt": ([130], [130]), "prompts": ([5, 128, 257, 31], [5, 128, 257, 31]),
           "chunk": ([385], [100]), "chunk behind a page": ([272], [16]), "mixed": ([300, 1, 77, 400, 0, 200], [1, 1, 30, 129, 0, 1]),
           "fewer keys than tokens": ([3, 20, 0], [9, 4, 2]),
           "server": ([300, 700, 1, 64, 0, 129, 500, 17, 90, 0, 33, 250], [120, 1, 1, 1, 1, 1, 300, 1, 2, 0, 1, 1]),
           "nobody has one token": ([30, 40, 50, 60, 70, 80, 90, 200], [2, 3, 0, 60, 5, 2, 90, 7]), "more than 32 sequences": ([*range(1, 40)], [1 + b % 3 for b in range(39)])}
HEADS = [(1, 1, 64), (4, 2, 64), (6, 2, 128), (5, 1, 128), (8, 1, 64), (16, 1, 128), (12, 12, 64), (3, 1, 128)]


def _attend(s, cu=True, **kw):
    from ghost_flow_b200 import ops

    return ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"] if cu else None, **kw)


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("H,Hk,D", HEADS)
def test_attention(name, H, Hk, D, kernel_status):
    lens, new = BATCHES[name]
    lens = [max(n, 0) for n in lens]
    s = oracle.batch(lens, new, H, Hk, D, 16 if D == 64 else 32, device="cuda", behind=3)
    want, off = oracle.attention(s)
    out = torch.full_like(s["q"], 7.0)
    _attend(s, out=out)
    n = sum(new)
    oracle.close(out[:n], want[:n], off[:n], name)
    assert (out[n:] == 7).all()                          # behind the last sequence
    assert torch.equal(_attend(s)[:n], out[:n])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["dense", "heads first", "together"])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 2, 128)])
def test_attention_pages_and_layouts(page, layout, H, Hk, D, kernel_status):
    lens, new = [page - 1, page, page + 1, 3 * page + 5, 300], [1, 2, page + 1, 40, 1]
    s = oracle.batch(lens, new, H, Hk, D, page, device="cuda", layout=layout)
    want, off = oracle.attention(s)
    oracle.close(_attend(s), want, off)


@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 1, 128), (16, 1, 64), (20, 2, 128), (11, 1, 64), (40, 1, 128)])
@pytest.mark.parametrize("scale", [None, 0.02, -0.3])
def test_attention_of_one_token_each(H, Hk, D, scale, kernel_status):
    lens = [1, 16, 17, 0, 64, 1000, 515]
    s = oracle.batch(lens, [1] * len(lens), H, Hk, D, 16, device="cuda")
    want, off = oracle.attention(s, scale)
    oracle.close(_attend(s, cu=False, scale=scale), want, off)


@pytest.mark.parametrize("parts", [1, 3, 16, -1, -5, -300])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (8, 1, 128), (24, 2, 64), (16, 1, 128)])
def test_attention_of_some_with_one_token(parts, H, Hk, D, monkeypatch, kernel_status):
    """Sequences of one token beside others, however their keys are cut; also where there is none of them, or nothing but them."""
    from ghost_flow_b200.ops import paged

    monkeypatch.setattr(paged, "_parts_beside", lambda *a: parts)
    lens = [900, 40, 64, 0, 1, 200, 333, 70, 5, 1200]
    for new in ([1, 40, 1, 1, 1, 2, 1, 33, 0, 1], [2, 40, 3, 2, 0, 2, 7, 33, 5, 0], [1] * 10, [0, 0, 0, 0, 0, 0, 0, 0, 1, 0]):
        s = oracle.batch(lens, new, H, Hk, D, 16, device="cuda", behind=1)
        want, off = oracle.attention(s)
        out = torch.full_like(s["q"], 7.0)
        for _ in range(2):
            _attend(s, out=out)
        n = sum(new)
        oracle.close(out[:n], want[:n], off[:n])
        assert (out[n:] == 7).all()


@pytest.mark.parametrize("lens,new", [([9000], [1]), ([5000, 3], [1, 1]), ([4000, 700], [40, 300]), ([20000], [3])])
@pytest.mark.parametrize("H,Hk,D", [(4, 1, 128), (4, 4, 64)])
def test_attention_over_long_sequences(lens, new, H, Hk, D, kernel_status):
    s = oracle.batch(lens, new, H, Hk, D, 64, device="cuda")
    want, off = oracle.attention(s)
    oracle.close(_attend(s), want, off)


def test_attention_with_scores_far_apart(kernel_status):
    """Maxima that move by a lot, upwards and downwards along the keys, and scores of the type's size."""
    for sizes in ((0.01, 40), (40, 0.01)):
        s = oracle.batch([700, 300], [130, 1], 4, 2, 64, 32, device="cuda")
        rows = torch.arange(700, device="cuda")
        at = s["table"][0, rows // 32].long(), rows % 32
        s["kp"][at] = (s["kp"][at].float() * torch.linspace(*sizes, 700, device="cuda")[:, None, None]).bfloat16()
        want, off = oracle.attention(s)
        oracle.close(_attend(s), want, off)


def test_attention_of_views(kernel_status):
    """q as a part of a packed projection, out with rows further apart."""
    s = oracle.batch([40, 300], [7, 33], 6, 2, 64, 16, device="cuda")
    packed = torch.randn(40, 10, 64, device="cuda").bfloat16()
    packed[:, :6] = s["q"]
    wide = torch.full((40, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    want, off = oracle.attention(s)
    from ghost_flow_b200 import ops
    got = ops.paged_attention(packed[:, :6], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], out=wide[:, 1:7])
    oracle.close(got, want, off)
    assert (wide[:, 0] == 7).all() and (wide[:, 7] == 7).all()
    odd = s["q"].transpose(1, 2).contiguous().transpose(1, 2)        # a layout that is copied first
    oracle.close(ops.paged_attention(odd, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]), want, off)


def test_attention_without_kernels_for_it(kernel_status):
    """Types, head sizes and pages that PyTorch's operations take."""
    for D, page, dtype in [(32, 16, torch.bfloat16), (64, 24, torch.bfloat16), (64, 16, torch.float32), (64, 16, torch.float16)]:
        s = oracle.batch([40, 300, 0], [7, 33, 1], 6, 2, D, page, dtype, device="cuda")
        want, off = oracle.attention(s)
        oracle.close(_attend(s), want, off + 2 ** -20)


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("H,Hk,D,layout", [(1, 1, 16, "dense"), (4, 2, 64, "together"), (25, 25, 64, "dense"), (32, 8, 128, "heads first"),
                                           (5, 1, 80, "dense"), (40, 40, 128, "dense"), (2, 1, 256, "dense")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(name, H, Hk, D, layout, interleaved, kernel_status):
    from ghost_flow_b200 import ops

    lens, new = BATCHES[name]
    s = oracle.batch(lens, new, H, Hk, D, 16 if D == 64 else 32, device="cuda", layout=layout, behind=2)
    cos, sin = ops.rope_tables(1024, D, 1e4, "cuda")
    q, qo, k, ko, v = oracle.append(s, H, Hk, cos, sin, interleaved)
    with torch.no_grad():
        got = ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"], interleaved)
    n = sum(new)
    oracle.close(got[:n], q[:n], qo[:n])
    oracle.close(s["kp"], k, ko)
    oracle.close(s["vp"], v, 0.0)


def test_append_then_attend_is_attention_of_the_whole(kernel_status):
    """A prompt in chunks and token by token, against the whole prompt through the dense operators."""
    from ghost_flow_b200 import ops

    H, Hk, D, page, S = 8, 2, 64, 16, 200
    cos, sin = ops.rope_tables(256, D, 1e4, "cuda")
    x = torch.randn(2, S, H + 2 * Hk, D, device="cuda").bfloat16()
    with torch.no_grad():
        q, k, v = ops.rope_qkv(x, H, Hk, cos, sin)
        whole = ops.flash_attention(q, k, v)
        kp, vp = (torch.full((40, page, Hk, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        table = torch.randperm(40, device="cuda").int()[:26].view(2, 13)
        at, got = [0, 0], [[], []]
        for step in [(100, 1), (1, 60), (0, 17), (50, 50), (1, 1), (47, 71), (1, 0)]:
            lens = [a + n for a, n in zip(at, step)]
            cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device="cuda")
            new = torch.cat([x[b, at[b]:lens[b]] for b in range(2)])
            n = torch.tensor(lens, dtype=torch.int32, device="cuda")
            o = ops.paged_attention(ops.rope_qkv_to_pages(new, H, Hk, cos, sin, kp, vp, table, n, cu), kp, vp, table, n, cu)
            for b in range(2):
                got[b].append(o[int(cu[b]):int(cu[b + 1])])
            at = lens
    assert at == [S, S]
    got = torch.stack([torch.cat(g) for g in got])
    # both round probabilities and results to bf16: half a step each, of sums of |v| (below 4) at most twice
    assert (got.float() - whole.float()).abs().max() < 4 * 4 * 2 ** -8
    assert (got.float() - whole.float()).norm() / whole.float().norm() < 2 * 2 ** -8


def test_pages_and_positions_that_are_not_there():
    """Left out, and reported: nothing around them changes."""
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
    for change, raises in [(lambda s: s["table"].__setitem__((1, 1), 10 ** 6), True), (lambda s: s["table"].__setitem__((1, 1), -5), True),
                           (lambda s: s["lens"].__setitem__(1, 10 ** 6), True), (lambda s: None, False)]:
        for new in ([1, 1], [1, 20]):
            s = oracle.batch([7, 20], new, 4, 2, 64, 16, device="cuda")
            before = s["kp"].clone(), s["vp"].clone()
            change(s)
            _lib.check_status()
            a = _attend(s)
            assert torch.isfinite(a[:1]).all()
            if raises:
                with pytest.raises(_lib.KernelStatusError):
                    _lib.check_status()
            ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"])
            if raises:
                with pytest.raises(_lib.KernelStatusError):
                    _lib.check_status()
                page = s["table"][1, 0]                      # other rows keep what they held
                rest = torch.ones(s["kp"].shape[0], dtype=torch.bool, device="cuda")
                rest[page], rest[s["table"][0, 0]] = False, False
                for x, y in zip((s["kp"], s["vp"]), before):
                    assert torch.equal(x[rest].nan_to_num(3), y[rest].nan_to_num(3))
            _lib.check_status()


def test_replayed_calls_go_by_what_the_lengths_hold(kernel_status):
    from ghost_flow_b200 import ops

    H, Hk, D = 8, 2, 64
    s = oracle.batch([200, 330, 5], [1, 1, 1], H, Hk, D, 16, device="cuda")
    cos, sin = ops.rope_tables(512, D, 1e4, "cuda")
    pools = s["kp"].clone(), s["vp"].clone()

    def step(kp, vp):
        q = ops.rope_qkv_to_pages(s["qkv"], H, Hk, cos, sin, kp, vp, s["table"], s["lens"])
        return ops.paged_attention(q, kp, vp, s["table"], s["lens"])

    with torch.no_grad():
        step(s["kp"], s["vp"])
        graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
        for g in graphs:                                    # two of them, that could share a workspace
            with torch.cuda.graph(g):
                outs.append(step(s["kp"], s["vp"]))
        for lens in ([200, 330, 5], [17, 0, 1], [199, 64, 3]):
            s["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
            for x, y in zip((s["kp"], s["vp"]), pools):
                x.copy_(y)
            want = step(s["kp"], s["vp"])
            for x, y in zip((s["kp"], s["vp"]), pools):
                x.copy_(y)
            for g, o in zip(graphs, outs):
                g.replay()
            for o in outs:
                assert torch.equal(o, want)


def test_two_streams_at_once(kernel_status):
    batches = [oracle.batch([3000 + 7 * i, 40], [1, 33], 8, 2, 128, 32, device="cuda", seed=i) for i in range(4)]
    want = [_attend(s) for s in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [None] * len(batches)
    for _ in range(3):
        for i, (s, st) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(st):
                got[i] = _attend(s)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_writes_are_visible_to_autograd_and_to_dispatch_modes():
    from torch.utils._python_dispatch import TorchDispatchMode

    from ghost_flow_b200 import ops

    s = oracle.batch([7, 20], [1, 2], 4, 2, 64, 16, device="cuda")
    kp, vp = s["kp"].nan_to_num(0, 0, 0), s["vp"].nan_to_num(0, 0, 0)
    cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
    args = s["table"], s["lens"], s["cu"]
    w = torch.ones_like(kp, requires_grad=True)
    for saved in (kp, vp):
        y = (saved * w).sum()
        with torch.no_grad():
            ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, kp, vp, *args)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            seen.append(func._schema.name)
            return func(*a, **(kw or {}))

    want = ops.paged_attention(s["q"], kp, vp, *args)
    with torch.no_grad(), Mode():
        got = ops.paged_attention(s["q"], kp, vp, *args)
    assert "aten::_softmax" in seen and (got.float() - want.float()).abs().max() < 2 ** -4


@pytest.mark.parametrize("which", ["append", "one each", "chunk", "prompts", "server", "logits"])
def test_count_is_the_kernels_of_a_call(which, kernel_status):
    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib
    from test_gpu_launch_count import _kernels

    lens, new = {"one each": ([3000, 5], [1, 1]), "chunk": ([2000], [33]), "prompts": ([4100] * 2, [4100] * 2),
                 "server": BATCHES["server"]}.get(which, ([20, 30], [3, 1]))
    H, Hk = (32, 8) if which == "prompts" else (8, 2)
    s = oracle.batch(lens, new, H, Hk, 128, 64, device="cuda")
    cos, sin = ops.rope_tables(64, 128, 1e4, "cuda")
    x = torch.randn(4, 100, device="cuda")
    f = {"append": lambda: ops.rope_qkv_to_pages(s["qkv"], 8, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]),
         "logits": lambda: ops.process_logits(x, repetition=1.5)}.get(which, lambda: _attend(s, cu=which != "one each"))
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.no_grad():
        f()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            n = _lib.launch_count()
            f()
            n = _lib.launch_count() - n
    assert n == _kernels(graph) > 0


def test_tensors_on_another_stream_and_calls_from_two_threads(kernel_status):
    import threading

    batches = [oracle.batch([700, 40, 300], [1, 33, 129], 8, 2, 64, 16, device="cuda", seed=i) for i in range(4)]
    want = [_attend(s) for s in batches]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(_attend(batches[i]), want[i]):
                    wrong.append(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_results_do_not_depend_on_what_scratch_memory_held(kernel_status):
    """NaN in the allocator's free blocks, which workspaces and results are made of."""
    for lens, new in (([3000], [40]), ([5000, 70], [1, 1]), BATCHES["server"], BATCHES["empty slots"]):
        s = oracle.batch(lens, new, 8, 2, 128, 32, device="cuda")
        one = set(new) == {1}
        want = _attend(s, cu=not one)
        for _ in range(2):
            torch.full((64 << 20,), float("nan"), device="cuda")
            assert torch.equal(_attend(s, cu=not one), want)


def test_batches_of_nothing_and_tensors_that_autograd_does_not_follow(kernel_status):
    from ghost_flow_b200 import ops

    cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
    s = oracle.batch([], [], 4, 2, 64, 16, device="cuda", behind=3)
    assert _attend(s).shape == (3, 4, 64)
    assert ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]).shape == (3, 4, 64)
    s = oracle.batch([7, 20], [1, 2], 4, 2, 64, 16, device="cuda")
    args = s["table"], s["lens"], s["cu"]
    want = _attend(s)
    with torch.inference_mode():
        pools = s["kp"].clone(), s["vp"].clone()
        assert torch.equal(ops.paged_attention(s["q"].clone(), *pools, *args), want)
        ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, *pools, *args)
    leaf = torch.zeros_like(s["q"], requires_grad=True)
    with pytest.raises(RuntimeError):                       # as a write to a leaf is
        _attend(s, out=leaf)
    with torch.no_grad():
        _attend(s, out=leaf)
    assert torch.equal(leaf.detach(), want)


def test_gradients_of_shared_heads_on_the_device():
    """A call with a gradient to record takes PyTorch's operations, in the type of its tensors."""
    s = oracle.batch([40, 9], [7, 9], 4, 2, 64, 16, device="cuda")
    s = {k: v.nan_to_num(0, 0, 0) if k in ("kp", "vp") else v for k, v in s.items()}
    t = [s[n].float().requires_grad_() for n in ("q", "kp", "vp")]
    d = [s[n].double().requires_grad_() for n in ("q", "kp", "vp")]
    b = [s[n].clone().requires_grad_() for n in ("q", "kp", "vp")]
    from ghost_flow_b200 import ops

    w = torch.randn(16, 4, 64, device="cuda")
    grads = [torch.autograd.grad((ops.paged_attention(*x, s["table"], s["lens"], s["cu"]) * w.to(x[0].dtype)).sum(), x) for x in (d, t, b)]
    for exact, single, half in zip(*grads):
        # 32 bits: sums of at most 40 products of numbers of this size; bf16: the products' inputs and results are rounded, and grads once more
        assert (single.double() - exact).norm() <= 64 * 2 ** -24 * 16 * exact.norm()
        assert (half.double() - exact).norm() <= 8 * 2 ** -8 * exact.norm()


@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (16, 1, 128), (20, 1, 128)])
@pytest.mark.parametrize("lens,new", [([40, 90], [1, 1]), ([3000, 70], [1, 1]), ([300] * 40, [1] * 40), ([130, 70], [130, 70]), ([5000, 300], [3, 100]),
                                      ([2000, 30, 50, 60, 64, 5, 80, 90, 700], [200, 1, 1, 1, 1, 1, 1, 1, 2])], ids=str)
def test_what_is_not_a_number_stays_so_and_where_it_is(lens, new, H, Hk, D, kernel_status):
    """A query that is not a number gives a row that is not, one of the keys every row that sees it; all other rows are as they were."""
    s = oracle.batch(lens, new, H, Hk, D, 16, device="cuda")
    one = set(new) == {1}
    want = _attend(s, cu=not one)
    t = sum(new[:2]) - 1                                 # the last token of the second sequence
    q = s["q"].clone()
    s["q"][t, H - 1, 5] = float("nan")
    got = _attend(s, cu=not one)
    assert got[t, H - 1].isnan().all()
    got[t, H - 1] = want[t, H - 1]
    assert torch.equal(got, want)
    s["q"] = q
    at = lens[0] // 2                                    # a key of the first sequence
    s["kp"][int(s["table"][0, at // 16]), at % 16, 0, 7] = float("nan")
    got = _attend(s, cu=not one)
    sees = torch.zeros(len(want), H, dtype=torch.bool, device="cuda")
    sees[max(0, at - (lens[0] - new[0])):new[0], :H // Hk] = True
    assert got[sees].isnan().all()
    got[sees] = want[sees]
    assert torch.equal(got, want)


def test_projections_in_the_pages_are_refused(kernel_status):
    from ghost_flow_b200 import ops

    s = oracle.batch([7, 20], [1, 2], 4, 2, 64, 16, device="cuda")
    cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
    for pool in (s["kp"], s["vp"]):
        before = pool.nan_to_num(1, 2, 3)
        with pytest.raises(ValueError, match="shares memory"):
            ops.rope_qkv_to_pages(pool.view(-1)[:3 * 8 * 64].view(3, 8, 64), 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"])
        assert torch.equal(pool.nan_to_num(1, 2, 3), before)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("inside,kernels", [("nothing", True), ("a device", True), ("a function mode", False), ("a dispatch mode", False),
                                            ("forward mode", False), ("a gradient", False), ("no gradients", True), ("tracing", False)])
def test_kernels_run_where_nothing_follows(inside, kernels, kernel_status):
    import contextlib

    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    from ghost_flow_b200 import ops
    from ghost_flow_b200.ops import _lib

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, a=(), kw=None):
            return func(*a, **(kw or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            return func(*a, **(kw or {}))

    s = oracle.batch([7, 20], [1, 2], 4, 2, 64, 16, device="cuda")
    s["kp"], s["vp"] = s["kp"].nan_to_num(0, 0, 0), s["vp"].nan_to_num(0, 0, 0)
    cos, sin = ops.rope_tables(64, 64, 1e4, "cuda")
    x = torch.randn(2, 90, device="cuda")
    around = {"a device": torch.device("cuda"), "a function mode": Function(), "a dispatch mode": Dispatch(),
              "forward mode": torch.autograd.forward_ad.dual_level(), "no gradients": torch.no_grad()}.get(inside, contextlib.nullcontext())
    if "gradient" in inside:
        s["q"].requires_grad_(), s["qkv"].requires_grad_(), x.requires_grad_()
    calls = [lambda: _attend(s), lambda: ops.process_logits(x, bias=torch.ones(90, device="cuda"))]
    if inside != "a gradient":                               # to pools that are no leaves
        calls.append(lambda: ops.rope_qkv_to_pages(s["qkv"], 4, 2, cos, sin, s["kp"], s["vp"], s["table"], s["lens"], s["cu"]))
    for f in calls:
        n = _lib.launch_count()
        with around:
            torch.jit.trace(lambda _: f(), (torch.ones(1),), check_trace=False) if inside == "tracing" else f()
        assert (_lib.launch_count() > n) == kernels
