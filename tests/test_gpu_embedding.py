"""GPU tests of the embedding and its gradient against float64 evaluations of their formulas.

Tolerances, with u = 2^-24 (half a step of float32): scale * e is one rounding, u relative. exp(scale * e): the argument's
rounding, |scale e| u, and expf's two units in the last place, 4 u, so (|scale e| + 5) u. A sum of n terms in any order is off by
at most n u times the sum of their magnitudes; with the factor (the above and one product) (n + |scale e| + 8) u."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _case(N, V, D, seed, dtype=None, skew=False):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    ids = torch.randint(0, V, (N,), device="cuda", generator=g, dtype=dtype or torch.int64)
    if skew:                                         # half of the tokens are one id
        ids[torch.rand(N, device="cuda", generator=g) < 0.5] = V // 2
    table = torch.rand(V, D, device="cuda", generator=g) * 2 - 0.5
    up = torch.randn(N, D, device="cuda", generator=g)
    return ids, table, up


def _check(ids, table, up, y, grad, scale, spikes, padding=None, no_spike=1e5):
    """y and grad against the formulas; ids outside the table allowed."""
    import torch
    V, D = table.shape
    flat = ids.reshape(-1).long()
    there = (flat >= 0) & (flat < V)
    if padding is not None:
        there &= flat != padding
    at = flat.clamp(0, V - 1)
    arg = table.double() * float(np.float32(scale))
    value = arg.exp() if spikes else arg
    want = torch.where(there[:, None], value[at], torch.full((), no_spike, dtype=torch.float64, device=y.device))
    tol = want.abs() * U * ((arg[at].abs() + 5) if spikes else 1) * 1.0001
    assert ((y.reshape(-1, D).double() - want).abs() <= torch.where(there[:, None], tol, torch.zeros_like(tol))).all()
    if grad is None:
        return
    f = float(np.float32(scale)) * (value if spikes else torch.ones_like(value))
    total = torch.zeros(V, D, dtype=torch.float64, device=y.device).index_put_((at[there],), up.reshape(-1, D)[there].double(), accumulate=True)
    size = torch.zeros(V, D, dtype=torch.float64, device=y.device).index_put_((at[there],), up.reshape(-1, D)[there].double().abs(), accumulate=True)
    n = torch.bincount(at[there], minlength=V)[:, None].double()
    bound = (n + (arg.abs() if spikes else 0) + 8) * U * size * f.abs()
    err = (grad.double() - total * f).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())
    assert (grad[n[:, 0] == 0] == 0).all()


SIZES = [(1, 1, 1), (1, 10007, 784), (2, 2, 3), (31, 7, 4), (32, 1, 33), (33, 300, 128), (257, 255, 129), (257, 256, 64), (300, 257, 100),
         (1000, 65536, 12), (4097, 1000, 100), (5000, 3, 257), (7007, 50021, 129), (20000, 65535, 36), (40000, 131072, 8), (70001, 90, 16),
         (3, 100, 5000), (65536, 1 << 20, 4), (40, 3, 2_100_001), (8192, 40, 7), (8193, 40, 8), (8200, 600, 31), (303_105, 513, 3), (150_000, 262_144, 2), (8193, 1000, 512), (8192, 777, 20), (8193, 777, 20), (8193, 500, 701), (8500, 300_000, 515),
         (40_000, 9, 128)]


@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("spikes", [False, True])
def test_values_and_gradient(N, V, D, spikes):
    import torch
    from snntc_2023_b200 import ops
    ids, table, up = _case(N, V, D, N + V + D, skew=N % 2 == 1)
    w = table.clone().requires_grad_(True)
    y = ops.snn_embedding(ids, w, scale=1.5, spikes=spikes)
    assert y.shape == (N, D)
    y.backward(up)
    _check(ids, table, up, y.detach(), w.grad, 1.5, spikes)
    first = w.grad.clone()                           # the same bits again
    w.grad = None
    ops.snn_embedding(ids, w, scale=1.5, spikes=spikes).backward(up)
    assert torch.equal(first, w.grad)
    with torch.no_grad():
        assert torch.equal(ops.snn_embedding(ids, w, scale=1.5, spikes=spikes), y)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("N,V,D", [(129, 50, 24), (9000, 700, 33)])
def test_padding_and_ids_outside_the_table_never_spike(bits, N, V, D):
    import torch
    from snntc_2023_b200 import ops
    dtype = torch.int32 if bits == 32 else torch.int64
    ids, table, up = _case(N, V, D, 5, dtype)
    ids[::7] = -1
    ids[1::11] = V
    ids[2::13] = torch.iinfo(dtype).max if bits == 32 else 2 ** 40 + 3      # (the low 32 bits are an id of the table)
    ids[5::17] = torch.iinfo(dtype).min
    ids[3::5] = 4
    up[::7] = float("nan")                           # what comes back for a token that does not spike is not read
    w = table.clone().requires_grad_(True)
    y = ops.snn_embedding(ids, w, scale=0.5, padding_idx=4, spikes=True, no_spike=2e5)
    y.backward(up)
    _check(ids, table, up, y.detach(), w.grad, 0.5, True, padding=4, no_spike=2e5)
    assert (w.grad[4] == 0).all() and (y[::7] == 2e5).all()


def test_no_token_at_all_and_no_ids():
    import torch
    from snntc_2023_b200 import ops
    w = torch.rand(9, 4, device="cuda").requires_grad_(True)
    y = ops.snn_embedding(torch.full((6,), -1, device="cuda"), w)
    y.backward(torch.ones_like(y))
    assert (y == 1e5).all() and (w.grad == 0).all()
    w.grad = None
    y = ops.snn_embedding(torch.empty(2, 0, dtype=torch.long, device="cuda"), w)
    assert y.shape == (2, 0, 4)
    y.sum().backward()
    assert (w.grad == 0).all()


def test_one_id_everywhere():
    """A run over all tiles: every partial sum is of the same row."""
    import torch
    from snntc_2023_b200 import ops
    for N, D in ((100000, 20), (5001, 512)):
        ids, table, up = _case(N, 40, D, 8)
        ids.fill_(39)
        w = table.clone().requires_grad_(True)
        y = ops.snn_embedding(ids, w, scale=2.0)
        y.backward(up)
        _check(ids, table, up, y.detach(), w.grad, 2.0, False)


def test_strides_shapes_and_offsets():
    import torch
    from snntc_2023_b200 import ops
    g = torch.Generator("cuda").manual_seed(2)
    big = torch.rand(50, 14, device="cuda", generator=g)
    ids = torch.randint(0, 50, (6, 8, 2), device="cuda", generator=g)
    w = big[:, 1:14].requires_grad_(True)                                     # strided rows, off 16 bytes
    y = ops.snn_embedding(ids.transpose(0, 1), w, spikes=True)
    assert y.shape == (8, 6, 2, 13)
    up = torch.randn(13, 8, 6, 2, device="cuda", generator=g).permute(1, 2, 3, 0)   # an upstream gradient with other strides
    (grad,) = torch.autograd.grad(y, w, up)
    _check(ids.transpose(0, 1).contiguous(), big[:, 1:14].contiguous(), up.contiguous(), y.detach(), grad, 1.0, True)
    flat = torch.rand(1 + 30 * 8, device="cuda", generator=g)                 # a contiguous table that starts off 16 bytes
    w = flat[1:].view(30, 8).detach().requires_grad_(True)
    ids = torch.randint(0, 30, (777,), device="cuda", generator=g)
    y = ops.snn_embedding(ids, w)
    (grad,) = torch.autograd.grad(y.sum(), w)                                 # (the upstream gradient is one number, expanded)
    _check(ids, w.detach(), torch.ones(777, 8, device="cuda"), y.detach(), grad, 1.0, False)


def test_a_table_beyond_32_bit_offsets():
    import torch
    from snntc_2023_b200 import ops
    V, D = 2_200_003, 1001                                                    # 2.2e9 elements
    table = torch.empty(V, D, device="cuda")
    ids = torch.tensor([0, V - 1, 2_150_000, V - 1, 7], device="cuda")
    table[ids] = torch.rand(5, D, device="cuda")
    w = table.requires_grad_(True)
    y = ops.snn_embedding(ids, w, scale=3.0)
    assert torch.equal(y.detach(), table.detach()[ids] * 3.0)
    up = torch.randn(5, D, device="cuda")
    (grad,) = torch.autograd.grad(y, w, up)
    assert torch.equal(grad[V - 1], 3.0 * (up[1] + up[3])) and torch.equal(grad[2_150_000], 3.0 * up[2])
    assert torch.equal(grad[0], 3.0 * up[0]) and torch.equal(grad[7], 3.0 * up[4])
    grad[ids] = 0
    assert not grad.any()


def test_more_than_32_bits_of_values():
    """2.2e9 values of 2.2 million tokens. Upstream ones: a row's gradient is the number of its tokens, exactly."""
    import torch
    from snntc_2023_b200 import ops
    N, V, D = 2_200_003, 300, 1000
    ids = torch.randint(0, V, (N,), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    w = torch.rand(V, D, device="cuda").requires_grad_(True)
    y = ops.snn_embedding(ids, w)
    for t in (0, 1, N // 2, N - 2, N - 1):
        assert torch.equal(y[t].detach(), w.detach()[ids[t]])
    (grad,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(grad, torch.bincount(ids, minlength=V).float()[:, None].expand(V, D))


def test_one_id_without_a_shape_and_arrays_by_dlpack():
    import torch
    from snntc_2023_b200 import ops

    class Array:
        def __init__(self, t):
            self.t = t

        def __dlpack__(self, **kw):
            return self.t.__dlpack__(**kw)

        def __dlpack_device__(self):
            return self.t.__dlpack_device__()

    w = torch.rand(5, 7, device="cuda")
    assert torch.equal(ops.snn_embedding(torch.tensor(3, device="cuda"), w, scale=2.0), 2.0 * w[3])
    assert torch.equal(ops.snn_embedding(Array(torch.tensor([4, 1], device="cuda")), Array(w)), w[[4, 1]])


def test_two_threads_at_once():
    """Lookup, sort and gradient from two host threads on streams of their own."""
    import threading

    import torch
    from snntc_2023_b200 import ops
    cases = [_case(12_000, 3000, 400, 1), _case(500, 90, 33, 2)]

    def call(ids, table, up):
        w = table.clone().requires_grad_(True)
        y = ops.snn_embedding(ids, w, spikes=True)
        return y.detach(), torch.autograd.grad(y, w, up)[0]

    plain = [call(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call(*cases[k])
                torch.cuda.current_stream().synchronize()
                bad.extend(1 for a, b in zip(got, plain[k]) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals():
    import torch
    from snntc_2023_b200 import ops
    w = torch.rand(5, 4, device="cuda").requires_grad_(True)
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    for bad in (ids.float(), ids.bool(), ids.short(), ids.cpu()):
        with pytest.raises(ValueError):
            ops.snn_embedding(bad, w)
    for bad in (w.double(), w.half(), w[0], w[:0]):
        with pytest.raises(ValueError):
            ops.snn_embedding(ids, bad)
    with pytest.raises(ValueError):
        ops.snn_embedding(ids, w, scale=float("nan"))
    for sink in (torch.zeros(4, 5, device="cuda"), torch.zeros(5, 8, device="cuda")[:, ::2], torch.zeros(5, 4)):
        with pytest.raises(ValueError):
            ops.snn_embedding(ids, w, grad_sink=sink)
    y = ops.snn_embedding(ids, w)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), w, create_graph=True)


def test_the_sort_beside_the_lookup_is_the_backward_s_own():
    """A lookup that is long enough sorts its tokens for the backward, on another stream where the library may: the same bits as
    without that stream, and as from the C entry point that sorts in the backward. The ids are the caller's again after the lookup."""
    import torch
    from snntc_2023_b200 import _lib, ops
    lib = _lib.load()
    N, V, D = 30_011, 5000, 256
    ids, table, up = _case(N, V, D, 3, skew=True)
    ids[::50] = -1
    w = table.clone().requires_grad_(True)
    grads = []
    for overlap in (1, 0):
        lib.snntc_set_overlap(overlap)
        try:
            mine = ids.clone()
            y = ops.snn_embedding(mine, w, scale=0.5, spikes=True)
            mine.fill_(3)
            grads.append(torch.autograd.grad(y, w, up)[0])
        finally:
            lib.snntc_set_overlap(1)
    _check(ids, table, up, y.detach(), grads[0], 0.5, True)
    out = torch.empty_like(table)
    size = lib.snntc_embedding_backward_workspace_bytes(N, V, D)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    rc = lib.snntc_embedding_backward(ids.data_ptr(), 8, 0, up.data_ptr(), table.data_ptr(), out.data_ptr(), N, V, D, 0.5, 1, -1, ws.data_ptr(),
                                      size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(grads[0], grads[1]) and torch.equal(grads[0], out)


@pytest.mark.parametrize("N,V,D", [(3001, 500, 36), (12_001, 700, 512)])
def test_captured_replayed_and_on_another_stream(N, V, D):
    """Lookup and gradient captured once, replayed on other ids; and two streams at once: the results of plain calls."""
    import torch
    from snntc_2023_b200 import ops
    ids, table, up = _case(N, V, D, 1)
    w = table.clone().requires_grad_(True)

    def step(i, g):
        y = ops.snn_embedding(i, w, spikes=True)
        return y.detach(), torch.autograd.grad(y, w, g)[0]

    other = (torch.randint(-1, V, (N,), device="cuda"), torch.randn(N, D, device="cuda"))
    plain = [step(ids, up), step(*other)]
    sid, sup = ids.clone(), up.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sid, sup)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sid, sup)
    for k, (i, g) in enumerate(((ids, up), other, (ids, up))):
        sid.copy_(i)
        sup.copy_(g)
        graph.replay()
        assert torch.equal(out[0], plain[k % 2][0]) and torch.equal(out[1], plain[k % 2][1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(step(*((ids, up), other)[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, plain[k][0]) and torch.equal(b, plain[k][1]) for k in range(2) for a, b in got[k])


def test_a_capture_beside_a_live_eager_graph_is_refused():
    """Autograd would run the leaf's accumulation on the eager graph's stream, inside the capture. The call says so instead."""
    import torch
    from snntc_2023_b200 import ops
    ids, table, up = _case(64, 20, 8, 1)
    w = table.clone().requires_grad_(True)
    alive = ops.snn_embedding(ids, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            ops.snn_embedding(ids, w).backward(up)
    torch.cuda.synchronize()
    alive.backward(up)                               # the eager graph is as it was
    _check(ids, table, up, alive.detach(), w.grad, 1.0, False)


def test_a_capture_beside_a_live_graph_of_a_side_stream():
    """The usual warm-up: on a side stream, its last graph still alive when the capture begins."""
    import torch
    from snntc_2023_b200 import ops
    ids, table, up = _case(300, 20, 8, 3)
    w = table.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = ops.snn_embedding(ids, w)
        alive.backward(up)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.snn_embedding(ids, w)
        y.backward(up)
    ids.copy_(ids.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    _check(ids, table, up, y.detach(), w.grad, 1.0, False)


def test_a_long_lookup_beside_another_thread_s_capture():
    """While one thread captures long lookups with their gradients -- sorts on the library's streams are then part of its capture --
    another runs eagerly, and one captures for itself: each has its own results, and the captures are whole."""
    import contextlib
    import threading
    from concurrent.futures import ThreadPoolExecutor

    import torch
    from snntc_2023_b200 import ops
    N, V, D = 12_001, 700, 512
    cases = [_case(N, V, D, 40 + k) for k in range(3)]

    def step(k, times=1):
        ids, table, up = cases[k]
        for _ in range(times):
            w = table.detach().requires_grad_(True)
            y = ops.snn_embedding(ids, w, spikes=True)
            out = y.detach(), torch.autograd.grad(y, w, up)[0]
        return out

    plain = [step(k) for k in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for k, s in enumerate(streams):                   # what the eager calls below allocate is there already
        with torch.cuda.stream(s):
            kept = [step(k) for _ in range(6)]
            del kept
    torch.cuda.synchronize()
    inside, finished = threading.Barrier(3, timeout=60), threading.Barrier(3, timeout=60)

    def captured(k):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[k]):
            try:
                graph.capture_begin(capture_error_mode="thread_local")
                out = step(k)
                inside.wait()                         # both captures have drawn a stream of the library's
                out = step(k, times=4)
                finished.wait()
                graph.capture_end()
            except BaseException:
                inside.abort()
                finished.abort()
                with contextlib.suppress(RuntimeError):
                    graph.capture_end()
                raise
        return graph, out

    def eager(k):
        try:
            inside.wait()
            with torch.cuda.stream(streams[k]):
                out = [step(k) for _ in range(6)]
                streams[k].synchronize()
            finished.wait()
        except BaseException:
            inside.abort()
            finished.abort()
            raise
        return out

    with ThreadPoolExecutor(3) as pool:
        work = [pool.submit(captured, 0), pool.submit(captured, 1), pool.submit(eager, 2)]
        results = [f.result() for f in work]
    same = lambda got, k: torch.equal(got[0], plain[k][0]) and torch.equal(got[1], plain[k][1])  # noqa: E731
    assert all(same(out, 2) for out in results[2])
    for k in range(2):
        graph, out = results[k]
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, k)
    assert same(step(2), 2)                           # and the library's streams serve eager calls again


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("spikes", [False, True])
def test_a_sink_behind_the_sort_beside_the_lookup(bits, spikes):
    """A long lookup in training, whose tokens are sorted beside it, with the gradient into a sink: the bits that autograd would hand
    out, nothing of what the sink held, nothing for autograd."""
    import torch
    from snntc_2023_b200 import ops
    ids, table, up = _case(12_001, 700, 512, 17, torch.int32 if bits == 32 else torch.int64, skew=True)
    ids[::9] = -1
    w = table.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(ops.snn_embedding(ids, w, scale=0.5, spikes=spikes), w, up)
    sink = torch.full_like(table, float("nan"))
    for _ in range(2):
        y = ops.snn_embedding(ids, w, scale=0.5, spikes=spikes, grad_sink=sink)
        y.backward(up)
        assert torch.equal(sink, want) and w.grad is None
    _check(ids, table, up, y.detach(), sink, 0.5, spikes)


def test_two_threads_and_their_errors():
    """As test_two_threads_at_once, with an error in a thread as an error of the test, and every round counted."""
    from concurrent.futures import ThreadPoolExecutor

    import torch
    from snntc_2023_b200 import ops
    cases = [_case(12_000, 3000, 400, 1), _case(500, 90, 33, 2)]

    def call(ids, table, up):
        w = table.clone().requires_grad_(True)
        y = ops.snn_embedding(ids, w, spikes=True)
        return y.detach(), torch.autograd.grad(y, w, up)[0]

    plain = [call(*c) for c in cases]
    torch.cuda.synchronize()

    def work(k):
        equal = 0
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call(*cases[k])
                torch.cuda.current_stream().synchronize()
                equal += all(torch.equal(a, b) for a, b in zip(got, plain[k]))
        return equal

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(work, range(2))) == [20, 20]
