"""Buffers that go while a graph is being recorded: a garbage collector runs when it likes, and the recording has to go on."""
import numpy as np
import pytest

from cases import bind

pytestmark = pytest.mark.gpu


def _norm(ctx, n):
    x, w, y = ctx.buffer_from_iter(np.full(n * 256, 0x3C00, np.uint16)), ctx.buffer_from_iter(np.ones(256, np.float32)), ctx.new_buffer(n * 256, np.uint16)
    return bind(x, w, y), y


def test_releases_while_recording():
    import super_gemma_b200 as sg

    ctx, other = sg.GpuContext(0), sg.GpuContext(0)
    kernel = ctx.load_kernel("rmsnorm_256")
    calls = [_norm(ctx, 40) for _ in range(3)]
    gone = [ctx.new_buffer(1 << 20, np.uint8), other.new_buffer(1 << 20, np.uint8), other.new_buffer(64, np.uint8), ctx.new_buffer(64, np.uint8)]
    lost = _norm(ctx, 40)
    ctx.dispatch(kernel, lost[0], None, [40, 1, 1])  # work that is still to use what is released

    third = [sg.GpuContext(0)]

    def record(at):
        nonlocal lost
        third.pop()
        at.dispatch(kernel, calls[0][0], None, [40, 1, 1])
        gone.pop()
        gone.pop()
        at.dispatch(kernel, calls[1][0], None, [40, 1, 1])
        lost = None
        gone.pop()
        at.dispatch(kernel, calls[2][0], None, [40, 1, 1])
        gone.pop()

    graph = ctx.record_graph(record)
    for _ in range(2):
        for _, y in calls:
            y.zero()
        ctx.submit_blocking(graph)
        for _, y in calls:
            assert (y.read() == 0x3C00).all()  # 1 / sqrt(1 + 1e-6) is 1 in f16
    again = ctx.new_buffer(1 << 20, np.uint8)
    assert (again.read() == 0).all()
    other.sync()


def test_releases_in_a_recording_that_fails():
    import super_gemma_b200 as sg

    ctx = sg.GpuContext(0)
    gone = [ctx.new_buffer(1 << 16, np.uint8)]

    def record(at):
        gone.pop()
        raise ValueError("no graph of this")

    with pytest.raises(ValueError):
        ctx.record_graph(record)
    call, y = _norm(ctx, 3)
    ctx.dispatch_blocking(ctx.load_kernel("rmsnorm_256"), call, None, [3, 1, 1])
    assert (y.read() == 0x3C00).all()


def test_releases_by_another_thread():
    """One thread records and replays, three others make nothing but room: their buffers go at any moment of that."""
    import threading

    import super_gemma_b200 as sg

    ctx = sg.GpuContext(0)
    kernel = ctx.load_kernel("rmsnorm_256")
    call, y = _norm(ctx, 40)
    heaps = [[ctx.new_buffer(4096, np.uint8) for _ in range(150)] for _ in range(3)]
    def drop(heap):
        while heap:
            heap.pop()

    threads = [threading.Thread(target=drop, args=(heap,)) for heap in heaps]
    for t in threads:
        t.start()
    graphs = []
    for _ in range(20):
        graphs.append(ctx.record_graph(lambda at: [at.dispatch(kernel, call, None, [40, 1, 1]) for _ in range(4)]))
        ctx.submit(graphs[-1])
    for t in threads:
        t.join()
    ctx.sync()
    assert (y.read() == 0x3C00).all()
