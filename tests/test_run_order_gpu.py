"""A handle's runs follow one another whatever streams they are given: its
workspaces hold what a run packs. Observed by completion: work that a first
run waits for holds back the second as well."""
import threading

import pytest
import torch

import momiru_b200 as mb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
V = mb.DeviceView.from_torch
PER_THREAD = 2  # the value of cudaStreamPerThread, in every thread its own stream


def packing_layer():
    """A layer whose operands TMA cannot read: each run packs them into the handle's workspace."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    lhs, rhs = (torch.randn(*s, generator=g, device="cuda").bfloat16() for s in ((77, 515), (515, 1001)))
    out = torch.empty(77, 1001, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    op = mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out))
    assert "mmr_pack_kernel" in op.plan
    return op


def held_back(op, stream, ms=200):
    """A run of `op` behind `ms` of other work on `stream`; the event after it."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 1e6))  # about a cycle a nanosecond or less
        op.replay(stream.cuda_stream)
        done = torch.cuda.Event()
        done.record(stream)
    return done


def test_per_thread_streams_of_two_threads():
    op = packing_layer()
    seen, started, ended = {}, threading.Event(), threading.Event()

    def first():  # lives until the second is done, and its stream with it
        try:
            seen["done"] = held_back(op, torch.cuda.ExternalStream(PER_THREAD))
        finally:
            started.set()
        ended.wait(60)

    t = threading.Thread(target=first)
    t.start()
    started.wait(60)

    def second():
        stream = torch.cuda.ExternalStream(PER_THREAD)
        op.replay(PER_THREAD)
        stream.synchronize()
        seen["first was done"] = seen["done"].query()

    u = threading.Thread(target=second)
    u.start()
    u.join()
    ended.set()
    t.join()
    op.quiesce_or_abort(20)
    op.close()
    assert seen["first was done"]


def test_streams_of_different_values():
    op = packing_layer()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    done = held_back(op, s1)
    op.replay(s2.cuda_stream)
    s2.synchronize()
    assert done.query()
    op.quiesce_or_abort(20)
    op.close()


def test_runs_from_many_threads():
    """Sixteen threads, each with runs and waits of its own on one handle; the result is one run's."""
    op = packing_layer()
    out = op._views[2].torch_view()
    op.replay()
    op.quiesce_or_abort(20)
    want = out.clone()
    failed = []

    def work(i):
        try:
            for _ in range(20):
                op.replay(PER_THREAD if i % 2 else None)
                op.quiesce_or_abort(20)
        except Exception as e:  # reported by the assertion below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(16)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and torch.equal(out, want)
    op.close()
