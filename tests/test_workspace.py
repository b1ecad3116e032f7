"""The scratch that the operators share: of which stream and which graph it is."""
import pytest
import torch

fp8gq = pytest.importorskip("fp8gq")
from fp8gq import ops  # noqa: E402


@pytest.fixture
def fresh(monkeypatch):
    for name in ("_workspaces", "_captured"):
        monkeypatch.setattr(ops, name, {})
    monkeypatch.setattr(ops, "_outgrown", [])


CPU = torch.device("cpu")


def test_kept_per_stream_and_grown(fresh):
    a = ops._workspace_entry(CPU, 100, 0)
    assert a[0].numel() >= 100 and not a[0].any() and a[1] == a[0].data_ptr() and a[2] == a[0].numel()
    assert ops._workspace_entry(CPU, 1 << 20, 0) is a and ops._workspace_entry(CPU, 100, 7) is not a
    b = ops._workspace_entry(CPU, (1 << 20) + 1, 0)
    assert b is not a and b[2] > 1 << 20 and ops._outgrown[0] is a[0]
    assert ops._workspace_entry(CPU, 100, 0) is b


def test_scratch_of_a_capture_is_that_graphs_alone(fresh, monkeypatch):
    """Zeros made within a capture are there when that graph runs, not before: no
    call outside it and no other graph may take them for cleared."""
    now = [5]
    monkeypatch.setattr(ops, "_capture_id", lambda stream: now[0])
    a = ops._workspace_entry(CPU, 100, 3)
    assert ops._workspace_entry(CPU, 200, 3) is a          # the same graph: cleared once
    big = ops._workspace_entry(CPU, 2 << 20, 3)
    assert big is not a and ops._workspace_entry(CPU, 100, 3) is big
    now[0] = 6
    b = ops._workspace_entry(CPU, 100, 3)
    assert b is not a and b is not big
    now[0] = 0
    c = ops._workspace_entry(CPU, 100, 3)
    assert c is not b and ops._workspace_entry(CPU, 100, 3) is c
    now[0] = 7                                             # there before the capture, and enough
    assert ops._workspace_entry(CPU, 100, 3) is c
    d = ops._workspace_entry(CPU, 4 << 20, 3)              # there, but not enough
    now[0] = 0
    assert ops._workspace_entry(CPU, 100, 3) is c and ops._workspace_entry(CPU, 4 << 20, 3) is not d


def test_threads_get_the_same_scratch(fresh, monkeypatch):
    """Two threads' first calls on a stream: neither's scratch may be dropped while
    its call is about to use it."""
    import threading
    zeros, inside = torch.zeros, threading.Barrier(2)

    def slow(*a, **kw):
        try:
            inside.wait(0.5)             # both in here at once, if they can be
        except threading.BrokenBarrierError:
            pass
        return zeros(*a, **kw)
    monkeypatch.setattr(torch, "zeros", slow)
    got = []
    threads = [threading.Thread(target=lambda: got.append(ops._workspace_entry(CPU, 100, 3))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0] is got[1] is ops._workspaces[(None, 3)]


def test_no_capture_without_a_gpu():
    assert ops._capture_id(0) == 0


@pytest.mark.gpu
def test_second_graph_replayed_first(cuda_device):
    """Two graphs captured on a stream that was never used; the second runs first, and
    calls outside the graphs run in between."""
    from tests.test_serve_ops import decode_case, prompt_case, randn
    from tests.test_zz_no_alloc import _operands
    fp8gq.device_error(clear=True)
    kc, vc, table, ln = decode_case(24, [3000, 50], 2, 128, 16, torch.bfloat16)
    qd = randn(8, 2, 8, 128).bfloat16()
    q, k, v, cu_q, cu_k = prompt_case(22, [40, 3], [3100, 2500], 8, 2, 128, spare=0)
    q2, k2, v2, cu2, _ = prompt_case(23, [900, 77], [900, 77], 8, 2, 128, spare=0)
    x, wq, ws = _operands(4, 4096, 6144, 1, "cuda")

    def work():
        return [fp8gq.paged_decode_attention(qd, kc, vc, table, ln), fp8gq.prompt_attention(q, k, v, cu_q, cu_k),
                fp8gq.prompt_attention(q2, k2, v2, cu2), fp8gq.fused_gemv_quant(x, wq, ws),
                fp8gq.paged_decode_attention(qd, kc, vc, table, ln)]

    prev = fp8gq.set_tm_options(fp8gq.TM_WORKSPACE_SPLITK)
    side = torch.cuda.Stream()
    kept = ops._workspaces.pop((0, side.cuda_stream), None)
    try:
        want = work()
        side.wait_stream(torch.cuda.current_stream())
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                graphs.append((g, work()))
        assert (0, side.cuda_stream) not in ops._workspaces
        for i in (1, 0, 1, 1, 0):
            for o in graphs[i][1]:
                o.zero_()
            torch.cuda.synchronize()
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want))
            with torch.cuda.stream(side):
                assert all(torch.equal(a, b) for a, b in zip(work(), want))
        assert fp8gq.device_error() == 0
    finally:
        fp8gq.set_tm_options(prev)
        if kept is not None:
            ops._outgrown.append(kept[0])
