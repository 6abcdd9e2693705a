"""Linear and latent attention called in the ways of a serving process: from a fresh thread, from threads at once, captured in a fresh
process, behind other work, with many short sequences, with broadcast views."""
import subprocess
import sys
import threading

import pytest
import torch

import flashkda_b200 as lib
from attention_testlib import SCALE, assert_within, check_linear, latent_decode_oracle, latent_prompt_oracle, linear_inputs, paged

pytestmark = pytest.mark.gpu


def step_call():
    d = linear_inputs([1] * 5, 4, seed=1)
    hT = torch.zeros(5, 4, 128, 128, device="cuda")
    return lambda: lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, d["out"], d["h0"], hT), [d["out"], hT]


def chunk_call(T=300, H=4):
    d = linear_inputs([T], H, seed=2)
    hT = torch.zeros(1, H, 128, 128, device="cuda")
    return lambda: lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, d["out"], d["h0"], hT), [d["out"], hT]


def segment_call():
    return chunk_call(900, 2)


def prompt_call(T=400, H=3):
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    q, k, r, v = rnd(1, T, H, 192), rnd(1, T, H, 128), rnd(1, T, 64), rnd(1, T, H, 128)
    out, lse = torch.zeros_like(v), torch.zeros(1, T, H, device="cuda")
    return lambda: lib.latent_attention_fwd(q, k, r, v, SCALE, out, lse), [out, lse]


def decode_call():
    cache, table, lens, _ = paged([700, 3, 90], 32)
    q = torch.randn(3, 2, 8, 576, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).bfloat16()
    out, lse = torch.zeros(3, 2, 8, 512, device="cuda").bfloat16(), torch.zeros(3, 2, 8, device="cuda")
    return lambda: lib.latent_attention_decode(q, cache, table, lens, SCALE, out, lse), [out, lse]


CALLS = {"step": step_call, "chunk": chunk_call, "segment": segment_call, "prompt": prompt_call, "decode": decode_call}


def results(call, outs):
    for o in outs:
        o.zero_()
    call()
    torch.cuda.synchronize()
    return [o.clone() for o in outs]


@pytest.mark.parametrize("name", sorted(CALLS))
def test_first_call_of_a_thread(name):
    call, outs = CALLS[name]()
    want = results(call, outs)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    errors = []

    def run():
        try:
            call()
        except Exception as e:
            errors.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not errors
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_threads_with_a_stream_each_at_once():
    """All operators beside one another, each thread on a stream of its own, with scratch of the calls' own."""
    made = [CALLS[name]() for name in sorted(CALLS)]
    want = [results(*m) for m in made]
    errors = []

    def run(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    call()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(m[0],)) for m in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and lib.operator_status() == 0
    for (_, outs), w in zip(made, want):
        assert all(torch.equal(o, x) for o, x in zip(outs, w))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_captured_without_a_workspace_and_behind_other_work(name):
    """Scratch from the graph's own pool; the inputs' last write and the outputs' first read are nodes beside the call's."""
    call, outs = CALLS[name]()
    want = results(call, outs)
    total = torch.zeros((), device="cuda", dtype=torch.float64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for o in outs:
            o.fill_(3.0)
        call()
        total.copy_(sum(o.double().nan_to_num(0, 0, 0).sum() for o in outs))
    for _ in range(3):
        for o in outs:
            o.zero_()
        total.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert float(total) == float(sum(o.double().nan_to_num(0, 0, 0).sum() for o in outs))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_captured_as_the_first_call_of_a_process(name):
    code = f"""
import sys, torch
sys.path[:0] = ["tests", "."]
from test_attention_calls import CALLS, results
call, outs = CALLS[{name!r}]()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    call()
g.replay()
torch.cuda.synchronize()
got = [o.clone() for o in outs]
assert all(torch.equal(a, b) for a, b in zip(got, results(call, outs)))
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("n", [600, 1000])
def test_many_short_packed_sequences(n):
    """More sequences than the kernels put in order."""
    lens = [2 + i % 3 for i in range(n)]
    d = linear_inputs(lens, 2, seed=5, packed=True)
    hT = torch.zeros(n, 2, 128, 128, device="cuda")
    lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, d["out"], d["h0"], hT, d["cu"])
    some = [0, 1, n // 2, n - 2, n - 1]
    at = torch.tensor([0] + lens).cumsum(0).tolist()
    for i in some:
        e = {x: d[x][:, at[i]:at[i + 1]] for x in "qkvg"} | dict(cu=None, h0=d["h0"][i:i + 1])
        check_linear(e, [lens[i]], 1.0, d["out"][:, at[i]:at[i + 1]], hT[i:i + 1])
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).bfloat16()
    T = sum(lens)
    q, k, r, v = rnd(1, T, 2, 192), rnd(1, T, 2, 128), rnd(1, T, 64), rnd(1, T, 2, 128)
    out = torch.zeros_like(v)
    lib.latent_attention_fwd(q, k, r, v, SCALE, out, None, d["cu"])
    for i in some:
        s = slice(at[i], at[i + 1])
        want, _, bound, _ = latent_prompt_oracle(q[0, s], k[0, s], r[0, s], v[0, s], SCALE)
        assert_within(out[0, s], want, bound, f"sequence {i}")


def test_many_short_caches():
    n = 2500
    lens = [i % 70 for i in range(n)]
    cache, table, L, rows = paged(lens, 16, filler=float("nan"))
    q = torch.randn(n, 1, 3, 576, device="cuda").bfloat16()
    out, lse = torch.full((n, 1, 3, 512), 7.0, device="cuda").bfloat16(), torch.full((n, 1, 3), 7.0, device="cuda")
    lib.latent_attention_decode(q, cache, table, L, SCALE, out, lse)
    for b in [0, 1, 5, 69, 70, 71, 1234, n - 1]:
        want, wlse, bound, lb = latent_decode_oracle(q[b], rows[b], SCALE)
        assert_within(out[b], want, bound, f"sequence {b}")
        assert_within(lse[b], wlse, lb, f"lse {b}")
    empty = L == 0
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == float("-inf")).all())
    assert bool(torch.isfinite(out.float()).all())


def test_a_cache_without_pages_and_without_a_table():
    q = torch.randn(2, 1, 3, 576, device="cuda").bfloat16()
    out, lse = torch.full((2, 1, 3, 512), 7.0, device="cuda").bfloat16(), torch.zeros(2, 1, 3, device="cuda")
    lib.latent_attention_decode(q, torch.empty(0, 16, 576, device="cuda").bfloat16(), torch.empty(2, 0, dtype=torch.int32, device="cuda"),
                                torch.tensor([5, 0], dtype=torch.int32, device="cuda"), SCALE, out, lse)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    lib.latent_attention_decode(q[:0], torch.empty(0, 16, 576, device="cuda").bfloat16(), torch.empty(0, 0, dtype=torch.int32, device="cuda"),
                                torch.empty(0, dtype=torch.int32, device="cuda"), SCALE, out[:0], lse[:0])


def test_the_same_page_in_many_rows_of_the_table():
    """A shared prefix: sequences whose first pages are the same."""
    cache, table, lens, rows = paged([256, 96, 96], 32)
    table[1, :2], table[2, :2] = table[0, :2], table[0, :2]
    rows[1], rows[2] = torch.cat([rows[0][:64], rows[1][64:]]), torch.cat([rows[0][:64], rows[2][64:]])
    q = torch.randn(3, 1, 5, 576, device="cuda").bfloat16()
    out = torch.empty(3, 1, 5, 512, device="cuda").bfloat16()
    lib.latent_attention_decode(q, cache, table, lens, SCALE, out)
    for b in range(3):
        want, _, bound, _ = latent_decode_oracle(q[b], rows[b], SCALE)
        assert_within(out[b], want, bound, f"sequence {b}")


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_no_tokens_at_all(packed, kind):
    """The state goes through, and becomes zero where none comes in."""
    e = lambda *s: torch.empty(*s, device="cuda").bfloat16()
    n = 3
    h0 = torch.randn(n, 2, 128, 128, device="cuda").to(kind)
    hT = torch.full_like(h0, 7.0)
    B = 1 if packed else n
    cu = torch.zeros(n + 1, dtype=torch.int64, device="cuda") if packed else None
    args = e(B, 0, 2, 128), e(B, 0, 2, 128), e(B, 0, 2, 128), torch.empty(B, 0, 2, device="cuda"), 1.0, e(B, 0, 2, 128)
    lib.linear_attention_fwd(*args, h0, hT, cu)
    assert torch.equal(hT, h0)
    lib.linear_attention_fwd(*args, None, hT, cu)
    assert bool((hT == 0).all())
    lib.latent_attention_fwd(e(B, 0, 2, 192), e(B, 0, 2, 128), e(B, 0, 64), e(B, 0, 2, 128), 1.0, e(B, 0, 2, 128), None, cu, cu)


def test_decays_broadcast_over_tokens_or_heads():
    d = linear_inputs([130], 4, seed=7)
    for g in (-torch.rand(1, 1, 4, device="cuda").expand(1, 130, 4), -torch.rand(1, 130, 1, device="cuda").expand(1, 130, 4)):
        d["g"] = g
        hT = torch.zeros(1, 4, 128, 128, device="cuda")
        lib.linear_attention_fwd(d["q"], d["k"], d["v"], g, 0.3, d["out"], d["h0"], hT)
        check_linear(d, [130], 0.3, d["out"], hT)


def test_growing_states_and_negative_scales():
    """Decays above one are not refused, nor is a scale of any sign."""
    d = linear_inputs([100], 2, seed=8, strong=-0.01)
    hT = torch.zeros(1, 2, 128, 128, device="cuda")
    lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], -0.7, d["out"], d["h0"], hT)
    check_linear(d, [100], -0.7, d["out"], hT)


def test_cumulative_lengths_that_run_backwards_stay_in_bounds():
    """Nothing sensible comes out for such sequences, but nothing outside of the tensors is touched and the others are served."""
    d = linear_inputs([400], 2, seed=9, packed=True)
    guard = torch.full((1, 500, 2, 128), 7.0, device="cuda").bfloat16()
    out, cu = guard[:, 50:450], torch.tensor([0, 300, 100, 10 ** 12, 400], device="cuda")
    h = torch.zeros(4, 2, 128, 128, device="cuda")
    lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, out, h, h, cu)
    assert bool((guard[:, :50] == 7.0).all()) and bool((guard[:, 450:] == 7.0).all())
    q, k, r = (torch.randn(1, 400, *s, device="cuda").bfloat16() for s in ((2, 192), (2, 128), (64,)))
    guard.fill_(7.0)
    lib.latent_attention_fwd(q, k, r, k, SCALE, out, None, cu)
    torch.cuda.synchronize()
    assert bool((guard[:, :50] == 7.0).all()) and bool((guard[:, 450:] == 7.0).all())
    want, _, bound, _ = latent_prompt_oracle(q[0, :300], k[0, :300], r[0, :300], k[0, :300], SCALE)
    e = torch.empty_like(k)
    lib.latent_attention_fwd(q, k, r, k, SCALE, e, None, torch.tensor([0, 300, 400], device="cuda"))
    assert_within(e[0, :300], want, bound, "first sequence")
    assert lib.operator_status() == 0


@pytest.mark.parametrize("bad", [2 ** 31 - 1, -5, 10 ** 6])
def test_page_numbers_that_are_none_read_page_0(bad):
    cache, table, lens, rows = paged([64, 64], 32)
    table[1, 1] = bad
    rows[1] = torch.cat([rows[1][:32], cache[0]])
    q = torch.randn(2, 1, 4, 576, device="cuda").bfloat16()
    out = torch.empty(2, 1, 4, 512, device="cuda").bfloat16()
    lib.latent_attention_decode(q, cache.nan_to_num(0), table, lens, SCALE, out)
    for b in range(2):
        want, _, bound, _ = latent_decode_oracle(q[b], rows[b].nan_to_num(0), SCALE)
        assert_within(out[b], want, bound, f"sequence {b}")
