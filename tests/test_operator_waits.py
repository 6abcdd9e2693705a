"""The give-up path of the bounded waits in the kernels of linear and latent attention.

Every wait has a limit.  When it runs out the kernel stops loading, lets its roles run to their ends inside their tensors, waits for
what is in flight and returns; ``operator_status`` then reports it.  A test-only hook makes that happen without any fault: one call
loads nothing, and the first wait for its tiles has a limit of a few milliseconds.
"""
import threading
import time

import pytest
import torch

import flashkda_b200 as lib
from flashkda_b200 import _lib
from test_attention_calls import CALLS, chunk_call, decode_call, results

gpu = pytest.mark.gpu
WAITING = sorted(set(CALLS) - {"step"})


def test_the_hook_takes_a_limit_within_its_range():
    L = _lib.lib()
    assert [L.fkda_operator_test_starve(ms) for ms in (0, -1, 1001)] == [2, 2, 2]


@gpu
@pytest.mark.parametrize("name", WAITING)
def test_a_starved_call_is_reported_and_the_next_one_succeeds(name):
    call, outs = CALLS[name]()
    want = results(call, outs)
    assert lib.operator_status() == 0
    guards = [torch.full_like(outs[0], 7.0) for _ in range(2)]     # (other tensors of the process)
    assert _lib.lib().fkda_operator_test_starve(3) == 0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    call()
    assert lib.operator_status() == 9
    dt = time.perf_counter() - t0
    assert dt < 2.0, f"{dt:.2f} s with a limit of 3 ms"
    assert all(bool((x == 7.0).all()) for x in guards)
    got = results(call, outs)
    assert lib.operator_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_the_hook_is_for_one_call_on_its_thread():
    call, outs = chunk_call()
    want = results(call, outs)
    assert _lib.lib().fkda_operator_test_starve(3) == 0
    call()
    call()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    assert lib.operator_status() == 9 and lib.operator_status() == 0


@gpu
def test_every_thread_is_told():
    """A thread that asks first does not take the report away from another, nor does one that asks again get it twice."""
    call, outs = decode_call()
    want = results(call, outs)
    ask, answers = [threading.Event() for _ in range(2)], []

    def other():
        answers.append(lib.operator_status())      # (whatever there was before)
        answers.append(lib.operator_status())
        ask[0].set()
        ask[1].wait(30)
        answers.append(lib.operator_status())
        answers.append(lib.operator_status())

    t = threading.Thread(target=other)
    t.start()
    ask[0].wait(30)
    lib.operator_status()
    assert _lib.lib().fkda_operator_test_starve(3) == 0
    call()
    assert lib.operator_status() == 9 and lib.operator_status() == 0
    ask[1].set()
    t.join()
    assert answers[1:] == [0, 9, 0]
    assert all(torch.equal(a, b) for a, b in zip(results(call, outs), want))
    assert lib.operator_status() == 0
