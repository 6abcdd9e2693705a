"""How far a number that is not finite reaches in linear and latent attention: what sees it, and behind a mask (a weight of 0 times it) the
rows of its block, in its own dimension alone.  Everything else is what it is without it, bit for bit."""
import pytest
import torch

import flashkda_b200 as lib
from attention_testlib import SCALE, linear_inputs, paged

pytestmark = pytest.mark.gpu
BAD = [float("inf"), float("nan")]
H, HEAD, DIM = 3, 1, 77


def linear(d):
    out, hT = torch.full_like(d["out"], 7.0), torch.zeros_like(d["h0"])
    lib.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, out, d["h0"], hT, d["cu"])
    return out, hT


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("T,at", [(200, 100), (200, 191), (1000, 700)])      # (the last one in segments)
@pytest.mark.parametrize("what", ["q", "k", "v", "g"])
def test_linear_attention(what, T, at, bad):
    d = linear_inputs([T], H, seed=31)
    want, state = linear(d)
    d[what][0, at, HEAD, *([DIM] if what != "g" else [])] = bad
    out, hT = linear(d)
    hit = ~torch.isfinite(out[0])
    others = [h for h in range(H) if h != HEAD]
    assert torch.equal(out[0, :, others], want[0, :, others]) and torch.equal(hT[0, others], state[0, others])
    if what == "v":
        chunk = at // 64 * 64
        assert bool(hit[at:, HEAD, DIM].all()) and not bool(hit[:chunk].any())
        out[0, chunk:, HEAD, DIM] = want[0, chunk:, HEAD, DIM]
        assert torch.equal(out, want)
        rows = [r for r in range(128) if r != DIM]
        assert torch.equal(hT[0, HEAD, rows], state[0, HEAD, rows])
    else:
        assert torch.equal(out[0, :at], want[0, :at]) and (bool(hit[at, HEAD].any()) or what == "g")
        if what == "q":
            assert torch.equal(out[0, at + 1:], want[0, at + 1:]) and torch.equal(hT, state)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("T,prefix,at", [(300, 0, 200), (300, 0, 127), (500, 100, 477), (260, 1000, 1100), (100, 30, 120)])
@pytest.mark.parametrize("what", ["k", "k_rope", "v"])
def test_prompts(what, T, prefix, at, bad):
    gen = torch.Generator(device="cuda").manual_seed(32)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    d = dict(q=rnd(1, T, H, 192), k=rnd(1, T + prefix, H, 128), k_rope=rnd(1, T + prefix, 64), v=rnd(1, T + prefix, H, 128))

    def call():
        out, lse = torch.full((1, T, H, 128), 7.0, device="cuda").bfloat16(), torch.zeros(1, T, H, device="cuda")
        lib.latent_attention_fwd(d["q"], d["k"], d["k_rope"], d["v"], SCALE, out, lse)
        return out, lse

    want, want_lse = call()
    if what == "k_rope":
        d[what][0, at, 33] = bad
    else:
        d[what][0, at, HEAD, DIM] = bad
    out, lse = call()
    first = max(0, at - prefix)            # the first row that sees it
    if what == "v":
        assert torch.equal(lse, want_lse) and not bool(torch.isfinite(out[0, first:, HEAD, DIM]).any())
        reach = max(0, first - 255)
        out[0, reach:, HEAD, DIM] = want[0, reach:, HEAD, DIM]
        assert torch.equal(out, want)
    else:
        assert torch.equal(out[0, :first], want[0, :first]) and torch.equal(lse[0, :first], want_lse[0, :first])
        others = [h for h in range(H) if h != HEAD]
        assert what == "k_rope" or torch.equal(out[0, :, others], want[0, :, others])


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dim", [DIM, 540])
@pytest.mark.parametrize("at", [5, 130, 198, 199])
def test_drafted_tokens(at, dim, bad):
    Tq, n = 4, 200
    cache, table, lens, _ = paged([n, 90], 32, seed=33)
    q = torch.randn(2, Tq, H, 576, device="cuda", generator=torch.Generator(device="cuda").manual_seed(34)).bfloat16()

    def call():
        out, lse = torch.full((2, Tq, H, 512), 7.0, device="cuda").bfloat16(), torch.zeros(2, Tq, H, device="cuda")
        lib.latent_attention_decode(q, cache, table, lens, SCALE, out, lse)
        return out, lse

    want, want_lse = call()
    cache[table[0, at // 32], at % 32, dim] = bad
    out, lse = call()
    sees = [i for i in range(Tq) if at < n - Tq + 1 + i]
    blind = [i for i in range(Tq) if i not in sees]
    assert torch.equal(out[1], want[1]) and torch.equal(lse[1], want_lse[1])
    assert torch.equal(lse[0, blind], want_lse[0, blind]) and not bool(torch.isfinite(lse[0, sees]).any() if bad != bad else False)
    if dim >= 512:
        assert torch.equal(out[0, blind], want[0, blind])
    else:
        rest = [x for x in range(512) if x != dim]
        assert torch.equal(out[0, blind][..., rest], want[0, blind][..., rest])
