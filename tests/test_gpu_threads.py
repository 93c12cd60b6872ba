"""Host threads that share a context: the launches of one call stand together on its
stream, so that what one leaves in the context's workspace for the next is not
overwritten by another thread's."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from decoder_forms import Batch
from test_gpu_pages import attention_scalars, attention_symbol, halves, upload_batch

pytestmark = pytest.mark.gpu

ROUNDS = 60


def paged(ipus, ctx, kind):
    """(launch into a buffer, its bytes) of an attention of two launches: split
    blocks and their join, or shared keys and the decode that joins them."""
    if kind == "split keys":
        b, heads, key_heads, width = Batch(np.random.default_rng(41), [70, 33], [4100, 1500], 16), 4, 1, 64
    else:
        b = Batch(np.random.default_rng(42), [1] * 300, [1003] * 300, 16, shared=1000)
        heads, key_heads, width = 16, 4, 64
    cache = halves(ipus, (b.pages, 2, key_heads, b.page_rows, width), 1)
    q = halves(ipus, (b.rows, heads, width), 2)
    ins = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    scalars = attention_scalars(b, heads, key_heads, width, 1)
    return (lambda out: ctx.launch(attention_symbol(b), out, ins, scalars)), q.nbytes, ins


def beside(ipus, ctx, kind):
    """The same of an operator that another thread runs, in the same workspace."""
    if kind == "split product":
        M, N, K = 8, 1024, 4096
        ins = [ctx.upload(ipus.synth_f16(n, 61, t, ipus.UNIFORM)) for t, n in ((1, M * K), (2, K * N))]
        return (lambda out: ctx.launch("ipu_stack_gemm_f16", out, ins, [1, M, N, K, 0, 0, 0, 0])), M * N * 2, ins
    if kind == "decode attention":
        streams, keys, d = 4, 2048, 64
        ins = [ctx.upload(ipus.synth_f16(streams * n * d, 62, t, ipus.NORMAL, 1.0)) for t, n in enumerate((1, keys, keys))]
        return (lambda out: ctx.launch("ipu_stack_flash_attention_online_f16", out, ins,
                                       [streams, 1, keys, d, d, 0, 0, 0])), streams * d * 4, ins
    return paged(ipus, ctx, kind)


def run_threads(*jobs):
    failed, gate = [], threading.Barrier(len(jobs))

    def guarded(job):
        try:
            gate.wait(30)
            job()
        except BaseException as e:  # noqa: BLE001 - reported by the test's thread
            failed.append(e)

    threads = [threading.Thread(target=guarded, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed, failed
    assert not any(t.is_alive() for t in threads)


@pytest.mark.parametrize("second", ["split product", "decode attention", "split keys", "shared keys"])
@pytest.mark.parametrize("first", ["split keys", "shared keys"])
def test_two_threads_on_one_context(ipus, ctx, first, second):
    runs, want, held = [], [], []
    for launch, size, ins in (paged(ipus, ctx, first), beside(ipus, ctx, second)):
        alone = ctx.alloc(size)
        launch(alone)
        want.append(alone.download(np.uint16))
        alone.free()
        outs = [ctx.alloc(size) for _ in range(ROUNDS)]
        runs.append((launch, outs))
        held += ins
    ctx.sync()

    def job(launch, outs):
        def go():
            for out in outs:
                launch(out)
        return go

    run_threads(*(job(*r) for r in runs))
    ctx.sync()
    for (_, outs), bits in zip(runs, want):
        for i, out in enumerate(outs):
            assert np.array_equal(out.download(np.uint16), bits), i
    for buf in held + [o for _, outs in runs for o in outs]:
        buf.free()


def session(ipus, ctx):
    """A package whose product is split, and its result."""
    M, N, K = 8, 256, 4096
    g = ipus.ComputeGraph()
    g.set_outputs([g.gemm(g.host_input("x", [M, K]), g.parameter("w", [K, N]))])
    package = ipus.build_package(g, ipus.PackageConfig(compute_precision="f32"))
    s = package.session(ctx)
    s.write("x", ipus.synth_f32(M * K, 76, 1, 0, 1.0).reshape(M, K))
    s.write("w", ipus.synth_f32(K * N, 76, 2, 0, 1.0).reshape(K, N))
    name = package.outputs[0].name
    s.run_sync()
    return s, name, s.read(name).copy()


@pytest.mark.parametrize("kind", ["split keys", "shared keys"])
def test_a_session_beside_a_thread(ipus, ctx, kind):
    """Captured by one thread while another launches, whose launches are not
    recorded, and replayed between them."""
    launch, size, ins = paged(ipus, ctx, kind)
    s, name, bits = session(ipus, ctx)
    outs = [ctx.alloc(size) for _ in range(ROUNDS)]
    launch(outs[0])
    want = outs[0].download(np.uint16)
    ctx.memset(outs[0], 0xFF)
    ctx.sync()

    def replay():
        s.capture()
        for _ in range(ROUNDS):
            s.run()

    def work():
        for out in outs:
            launch(out)

    run_threads(replay, work)
    ctx.sync()
    assert np.array_equal(s.read(name), bits)
    for i, out in enumerate(outs):
        assert np.array_equal(out.download(np.uint16), want), i
        ctx.memset(out, 0xFF)
    # The graph holds the session's own launches and no others.
    s.run_sync()
    assert np.array_equal(s.read(name), bits)
    assert all(np.all(out.download(np.uint16) == 0xFFFF) for out in outs)
    s.close()
    for buf in ins + outs:
        buf.free()


def test_copies_beside_captures(ipus, ctx):
    """Copies, fills and waits of one thread are in no other thread's graph, and end no capture."""
    x = np.arange(4096, dtype=np.uint32)
    a, b = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    kept = []

    def capture():
        for _ in range(8):
            s, name, bits = session(ipus, ctx)
            s.capture()
            s.run_sync()
            kept.append((s, name, bits))

    def copy():
        for i in range(150):
            ctx.write(a, x + np.uint32(i))
            ctx.memset(b, i % 256)
            ctx.sync()
            assert np.array_equal(a.download(np.uint32), x + np.uint32(i))
            assert np.all(b.download(np.uint8) == i % 256)

    run_threads(capture, copy)
    ctx.write(a, x)
    ctx.memset(b, 0xFF)
    for s, name, bits in kept:
        s.run_sync()
        assert np.array_equal(s.read(name), bits)
    assert np.array_equal(a.download(np.uint32), x) and np.all(b.download(np.uint8) == 0xFF)
    for s, _, _ in kept:
        s.close()
    a.free()
    b.free()
