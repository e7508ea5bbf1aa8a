"""Two host threads whose calls use one stream, and so one cached scratch (GPU)."""

from __future__ import annotations

import sys
import threading

import pytest
import torch

import representax_amd as rx
from representax_amd import ops
from tests.helpers import DEVICE

pytestmark = pytest.mark.gpu


def _run(work):
    """Each of ``work`` in a thread of its own, the interpreter switching often."""

    failed = []

    def guarded(fn):
        try:
            fn()
        except BaseException as error:  # reported by the main thread
            failed.append(error)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        started = [threading.Thread(target=guarded, args=(fn,)) for fn in work]
        for t in started:
            t.start()
        for t in started:
            t.join(timeout=60)
    finally:
        sys.setswitchinterval(interval)
    assert not failed, failed[0]


def test_split_products_of_two_threads_keep_their_sums():
    """A split product is two launches over the scratch: its partial sums, then theirs."""

    g = torch.Generator(device=DEVICE).manual_seed(3)
    jobs = []
    for m, n, k in ((200, 130, 5000), (96, 300, 4100)):
        a, b = (torch.randn((r, k), generator=g, device=DEVICE).to(torch.bfloat16) for r in (m, n))
        jobs.append((rx.mxfp4_quantize(a), rx.mxfp4_quantize(b)))
    with ops.tuning(mx_tile=5, mx_splits=4):
        want = [rx.mxfp4_matmul(a, b, torch.float32) for a, b in jobs]
        torch.cuda.synchronize()
        wrong = [None, None]

        def work(i):
            def go():
                off = torch.zeros((), dtype=torch.bool, device=DEVICE)
                for _ in range(300):
                    off |= (rx.mxfp4_matmul(*jobs[i], torch.float32) != want[i]).any()
                wrong[i] = bool(off)
            return go

        _run([work(0), work(1)])
    assert wrong == [False, False]
