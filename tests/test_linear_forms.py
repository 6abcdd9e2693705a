"""The forms that a linear attention call is served in, chosen by its sizes and types: what they must not change, their values over
many chunks, and what the choice costs."""
import pytest
import torch

import flashkda_b200
from attention_testlib import BF, assert_within, linear_inputs, state_bound

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def call(d, h0=None, hT=None, **kw):
    flashkda_b200.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], SCALE, d["out"], h0, hT, d["cu"], **kw)


def check_head(d, n, at, T, h, h0=None, hT=None, packed=True):
    """One head of one sequence against the recurrence in 64 bits, chunk by chunk: inside a chunk
    o_i = sum over j <= i of exp(G_i - G_j) (q_i . k_j) v_j + exp(G_i) S q_i, and S is what the chunk before left.  The bound is that of
    attention_testlib.linear_oracle, which counts what a chunk rounds to bf16: weights times scores, and the state in front."""
    b, rows = (0, slice(at, at + T)) if packed else (n, slice(0, T))
    group = d["v"].shape[2] // d["q"].shape[2]
    q, k, v = (d[x][b, rows, h if x == "v" else h // group].double() for x in "qkv")
    g = (d["g"][h].expand(T) if d["g"].dim() == 1 else d["g"][b, rows, h]).double().clamp(min=-100.0)
    S = torch.zeros(128, 128, dtype=torch.float64, device="cuda") if h0 is None else h0[n, h].double()
    size = S.abs()
    out, bound = torch.empty_like(v), torch.empty_like(v)
    for c in range(0, T, 64):
        x = slice(c, min(T, c + 64))
        G = g[x].cumsum(0)
        P = ((G[:, None] - G[None]).tril().exp() * (q[x] @ k[x].T)).tril()
        out[x] = SCALE * (P @ v[x] + G.exp()[:, None] * (q[x] @ S.T))
        bound[x] = P.abs() @ v[x].abs() + G.exp()[:, None] * (q[x].abs() @ S.abs().T)
        w = (G[-1] - G).exp()[:, None]
        S = G[-1].exp() * S + (w * v[x]).T @ k[x]
        size = G[-1].exp() * size + (w * v[x].abs()).T @ k[x].abs()
    assert_within(d["out"][b, rows, h], out, SCALE * bound * (BF + 1e-3) + out.abs() * BF + 1e-30, f"out of sequence {n}, head {h}")
    if hT is not None:
        assert_within(hT[n, h], S, state_bound(T, size, S, hT.dtype), f"state of sequence {n}, head {h}")


# (the second one is walked in segments)
@pytest.mark.parametrize("lens,H", [([700], 40), ([700], 2), ([300, 900], 40), ([1, 500, 64], 60)], ids=str)
@pytest.mark.parametrize("first", [None, torch.bfloat16], ids=str)
def test_outputs_do_not_depend_on_the_final_state(lens, H, first):
    """Not on whether one is asked for, and without an initial state not on its type.  Weak decays, so that what a chunk adds to the
    state is still seen in the outputs of many later ones."""
    packed = len(lens) > 1
    d = linear_inputs(lens, H, seed=21, packed=packed, strong=0.01)
    h0 = d["h0"].to(first) if first is not None else None
    finals = [None, torch.zeros_like(d["h0"], dtype=torch.bfloat16)] + ([torch.zeros_like(d["h0"])] if first is None else [])
    outs = []
    for hT in finals:
        d["out"].fill_(7.0)
        call(d, h0, hT)
        outs.append(d["out"].clone())
    assert all(torch.equal(o, outs[0]) for o in outs)
    at = 0
    for n, T in enumerate(lens):
        check_head(d, n, at, T, H - 1, h0, finals[1], packed)
        at += T


def microseconds(call, calls=20):
    best = []
    for _ in range(5):
        torch.cuda.synchronize()
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        for _ in range(calls):
            call()
        end.record()
        end.synchronize()
        best.append(start.elapsed_time(end) / calls * 1e3)
    return min(best[1:])


@pytest.mark.parametrize("n,T,H", [(256, 20, 4), (800, 20, 4)])
def test_many_short_packed_sequences_cost_what_a_fixed_batch_costs(n, T, H):
    """Their chains are walked in the same way, so nothing may be looked up on the way that takes as long (half as much again is left)."""
    times = []
    for packed in (False, True):
        d = linear_inputs([T] * n, H, packed=packed)
        hT = torch.zeros_like(d["h0"])
        times.append(microseconds(lambda: call(d, d["h0"], hT)))
    assert times[1] < 1.5 * times[0], times


def test_packed_single_tokens_cost_about_what_a_fixed_batch_costs():
    """The host cannot know that no sequence is longer, so the kernel for longer ones is there too, and has to leave soon."""
    times = []
    for packed in (False, True):
        d = linear_inputs([1] * 128, 32, packed=packed)
        hT = torch.zeros_like(d["h0"])
        times.append(microseconds(lambda: call(d, d["h0"], hT)))
    assert times[1] < 2 * times[0], times


@pytest.mark.parametrize("lens", [[1] * 60 + [70] + [1] * 39, [1, 0, 2] * 20 + [1] * 40, [1] * 50, [1, 0] * 40, [1, 2, 1, 1], [1, 1, 0, 1], [1] * 70 + [300, 1]],
                         ids=lambda x: f"{len(x)} of {sum(x)}")
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
def test_single_tokens_beside_longer_sequences(lens, kind):
    """Batches on both sides of every line between the kernels, more chains than SMs and fewer, with the state in place."""
    H = 5
    d = linear_inputs(lens, H, seed=22, packed=True)
    d["h0"] = d["h0"].to(kind)
    state = d["h0"].clone()
    call(d, state, state)
    at = 0
    for n, T in enumerate(lens):
        if T == 0:
            assert torch.equal(state[n], d["h0"][n])
        elif n % 3 == 0 or T > 1:
            check_head(d, n, at, T, n % H, d["h0"], state)
        at += T


# one chain per CTA in one piece; in segments of several chunks, fixed and packed; more chains than SMs, in the order of their lengths and,
# with one sequence more than are put in order, as they come
LONG = [([900], 80, 80, 1), ([1500, 1500], 80, 20, 1), ([8192], 32, 32, 2), ([3000, 1, 5000], 16, 4, 2), ([2000, 900, 1, 63, 1500, 700], 48, 12, 3),
        ([340 + 7 * (i % 9) for i in range(64)], 4, 4, 5), ([350 + 7 * (i % 9) for i in range(65)], 4, 2, 5)]


@pytest.mark.parametrize("lens,H,Hk,every", LONG, ids=[f"{len(x[0])} of {sum(x[0])} x {x[1]}" for x in LONG])
@pytest.mark.parametrize("kind", [None, torch.float32, torch.bfloat16], ids=str)
def test_values_over_many_chunks(lens, H, Hk, every, kind):
    """All buffers of the walk used many times over, and states that are handed from segment to segment, against 64 bits."""
    packed = len(set(lens)) > 1
    d = linear_inputs(lens, H, Hk, seed=23, packed=packed, strong=0.05)
    d["h0"] = d["h0"].to(kind or torch.float32)
    hT = torch.full_like(d["h0"], 9.0)
    h0 = d["h0"] if kind else None
    call(d, h0, hT)
    at = 0
    for n, T in enumerate(lens):
        if n % every == 0 or n >= len(lens) - 2:
            for h in sorted({0, H // 2 - 1, H - 1}):
                check_head(d, n, at, T, h, h0, hT, packed)
        at += T
    assert flashkda_b200.operator_status() == 0
