"""The forms that a latent attention call is served in, chosen by its sizes: their values, and what the choice costs."""
import pytest
import torch

import flashkda_b200
from attention_testlib import SCALE, assert_within, latent_prompt_oracle

pytestmark = pytest.mark.gpu


def prompts(lens, prefix, H, seed, packed=True, gap=0):
    """q, k, k_rope, v, all different, and the cumulative lengths."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    keys = [a + b for a, b in zip(lens, prefix)]
    B, T, Tk = (1, sum(lens), sum(keys)) if packed else (len(lens), lens[0], keys[0])
    d = dict(q=rnd(B, T, H, 192), k=rnd(B, Tk, H, 128), k_rope=rnd(B, Tk, 64), v=rnd(B, Tk, H, 128))
    d["out"], d["lse"] = torch.full((B, T, H, 128), 7.0, device="cuda").bfloat16(), torch.full((B, T, H), 7.0, device="cuda")
    d["cu"], d["cu_k"] = (torch.tensor([0] + x).cumsum(0).cuda() if packed else None for x in (lens, keys))
    return d


def call(d):
    flashkda_b200.latent_attention_fwd(d["q"], d["k"], d["k_rope"], d["v"], SCALE, d["out"], d["lse"], d["cu"], d["cu_k"])


def check_heads(d, lens, prefix, heads, only=None):
    at = at_k = 0
    for n, (T, p) in enumerate(zip(lens, prefix)):
        rows, keys = slice(at, at + T), slice(at_k, at_k + T + p)
        at, at_k = at + T, at_k + T + p
        if T == 0 or (only is not None and n not in only):
            continue
        out, lse, bound, lse_bound = latent_prompt_oracle(d["q"][0, rows, heads], d["k"][0, keys, heads], d["k_rope"][0, keys], d["v"][0, keys, heads], SCALE)
        assert_within(d["out"][0, rows, heads], out, bound, f"out of sequence {n}")
        assert_within(d["lse"][0, rows, heads], lse, lse_bound, f"lse of sequence {n}")


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


@pytest.mark.parametrize("n,T,H", [(256, 40, 8), (512, 40, 8)])
def test_many_short_packed_prompts_cost_about_what_a_fixed_batch_costs(n, T, H):
    """As many blocks of rows with the same keys; every block has to find its sequence, which may take as long again."""
    times = []
    for packed in (False, True):
        d = prompts([T] * n, [0] * n, H, 1, packed)
        times.append(microseconds(lambda: call(d)))
    assert times[1] < 2.5 * times[0], times


def uneven(n, mean, seed):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, 2 * mean, (n,), generator=gen).tolist()
    return [x + max(0, mean - sum(lens) // n + 1) for x in lens], torch.randint(0, 900, (n,), generator=gen).tolist()


# batches that are taken in the order of their keys (which is not that of their queries, has ties, and sequences without queries or
# without a prefix), and those just outside: one sequence more or fewer, more rounds of SMs, shorter sequences
ORDERS = {
    "ties and empty ones": ([300, 0, 513, 300, 1, 700, 256, 130], [700, 50, 0, 700, 2000, 0, 1000, 870], 16),
    "7": (*uneven(7, 400, 1), 16), "8": (*uneven(8, 400, 2), 16), "32": (*uneven(32, 260, 3), 8), "33": (*uneven(33, 260, 4), 8),
    "many rounds": (*uneven(20, 300, 5), 32), "short": (*uneven(30, 40, 6), 8)}


@pytest.mark.parametrize("name", ORDERS)
def test_packed_prompts_in_and_out_of_order(name):
    lens, prefix, H = ORDERS[name]
    d = prompts(lens, prefix, H, 7)
    call(d)
    check_heads(d, lens, prefix, slice(0, 2))
    check_heads(d, lens, prefix, slice(H - 1, H))
    assert flashkda_b200.operator_status() == 0
