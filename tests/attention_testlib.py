"""Linear and latent attention in 64 bits, with how far a kernel may be from it, element by element.

Bounds count roundings: half a step of bf16 is 2^-8 of the value, of fp32 2^-24.
"""
import math

import torch

BF = 2.0 ** -8
NEG = float("-inf")


def linear_oracle(q, k, v, g, scale, h0=None):
    """One sequence: q, k [T, Hk, 128], v [T, H, 128], g [T, H] or [H], h0 [H, 128, 128] or None, token by token.
    Returns (out, state, bound of out before its own rounding, sum of magnitudes behind every state element)."""
    T, H = v.shape[:2]
    q, k, v, g = (x.double() for x in (q, k, v, g))
    q, k = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k))
    g = g.expand(T, H).clamp(min=-100.0)
    S = torch.zeros(H, 128, 128, dtype=torch.float64, device=v.device) if h0 is None else h0.double().clone()
    size = S.abs()
    out, bound = torch.zeros_like(v), torch.zeros_like(v)
    for t in range(T):
        if t % 64 == 0:    # what a chunk rounds to bf16: the state in front of it, and its weights times scores
            front, G, rows = S.clone(), torch.zeros_like(g[0]), []
        a = g[t].exp()[:, None, None]
        S = a * S + v[t][:, :, None] * k[t][:, None, :]
        size = a * size + v[t].abs()[:, :, None] * k[t].abs()[:, None, :]
        out[t] = scale * (S @ q[t][:, :, None])[..., 0]
        G = G + g[t]
        rows = [(w * g[t].exp(), j) for w, j in rows] + [(torch.ones_like(g[0]), t)]
        for w, j in rows:
            bound[t] += (w * (q[t] * k[j]).sum(-1).abs())[:, None] * v[j].abs()
        bound[t] += G.exp()[:, None] * (front.abs() @ q[t].abs()[:, :, None])[..., 0]
    # sums of decays over a chunk are exact to 2^-24 of at most 64 of them, each up to 2^7 or so
    return out, S, abs(scale) * bound * (BF + 1e-3), size


def state_bound(T, size, S, dtype):
    """fp32 products of terms that hold 24 bits: a chunk adds at most 16 partial sums, each off by 2^-23 of the magnitudes.  A state that
    leaves in bf16 is made of weighted values in two bf16 terms: the first is x cut off behind 8 bits, which leaves less than 2^(e-7) for
    2^e <= |x|, and the second that rounded to 8 bits, off by at most half of 2^-7 of a number below 2^(e-7), whose leading bit is at most
    2^(e-8): 2^-8 2^(e-8) <= 2^-16 |x|."""
    terms = 2.0 ** -16 if dtype == torch.bfloat16 else 0.0
    return size * ((T // 64 + 2) * 16 * 2.0 ** -23 + terms) + 1e-30 + (S.abs() * BF if dtype == torch.bfloat16 else 0)


def softmax_oracle(scores, values, magnitude):
    """scores [..., n] (masked ones minus infinity), values [n, d] or [..., n, d]; `magnitude`: sums of |q| |k| scale behind the
    scores.  Returns (out, lse, bound of out, bound of lse)."""
    values = torch.where(torch.isnan(values) | torch.isinf(values), 0.0, values)   # (masked everywhere, where a test has such)
    lse = torch.logsumexp(scores, -1) if scores.shape[-1] else torch.full(scores.shape[:-1], NEG, dtype=torch.float64, device=scores.device)
    p = torch.where(scores == NEG, 0.0, (scores - torch.where(lse == NEG, 0.0, lse)[..., None]).exp())
    out, size = p @ values, p @ values.abs()
    # a score is a sum of at most 576 products in fp32, 36 partial sums off by 2^-23 each; exp2 of it adds the rounding of the product
    # with log2(e), 2^-24 of a number of this size, and 2^-22 of its own
    off = 36 * 2.0 ** -23 * magnitude + 2.0 ** -22 * (lse.abs().nan_to_num(0, 0, 0) + 8) + 2.0 ** -21
    return out, lse, size * (BF + 2 * off[..., None]) + out.abs() * BF + 1e-30, off


def assert_within(got, want, bound, what):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= bound)
    if not bool(same.all()):
        at = (~same).nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int((~same).sum())} of {same.numel()} off, first at {at}: {got[tuple(at)].item()} for "
                             f"{want[tuple(at)].item()}, may be {bound.expand_as(want)[tuple(at)].item():.3g} off")


def linear_inputs(lens, H, Hk=None, seed=0, packed=False, decay="token", device="cuda", strong=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    Hk = Hk or H
    B, T = (1, sum(lens)) if packed else (len(lens), lens[0])
    rnd = lambda *s: torch.randn(*s, generator=gen, device=device)
    q, k = (torch.nn.functional.normalize(rnd(B, T, Hk, 128), dim=-1).bfloat16() for _ in range(2))
    v = rnd(B, T, H, 128).bfloat16()
    g = -strong * torch.nn.functional.softplus(rnd(B, T, H)) if decay == "token" else -torch.rand(H, generator=gen, device=device)
    h0 = rnd(len(lens), H, 128, 128)
    cu = torch.tensor([0] + lens).cumsum(0).to(device) if packed else None
    return dict(q=q, k=k, v=v, g=g, h0=h0, cu=cu, out=torch.full((B, T, H, 128), 7.0, device=device).bfloat16())


def check_linear(d, lens, scale, out, hT, state=True, first_state="h0"):
    """Every sequence of a batch against the oracle."""
    at = 0
    for n, T in enumerate(lens):
        b, lo = (0, at) if d["cu"] is not None else (n, 0)
        g = d["g"] if d["g"].dim() == 1 else d["g"][b, lo:lo + T]
        h0 = d[first_state][n] if state else None
        o, S, bound, size = linear_oracle(d["q"][b, lo:lo + T], d["k"][b, lo:lo + T], d["v"][b, lo:lo + T], g, scale, h0)
        assert_within(out[b, lo:lo + T], o, bound + o.abs() * BF + 1e-30, f"out of sequence {n}")
        if hT is not None:
            assert_within(hT[n], S, state_bound(T, size, S, hT.dtype), f"state of sequence {n}")
        at += T


def latent_prompt_oracle(q, k, k_rope, v, scale, causal=True):
    """One sequence: q [T, H, 192], k, v [Tk, H, 128], k_rope [Tk, 64]."""
    T, Tk = q.shape[0], k.shape[0]
    q, k, v = (x.double().transpose(0, 1) for x in (q, k, v))
    key = torch.cat([k, k_rope.double()[None].expand(k.shape[0], -1, -1)], -1)
    scores = scale * q @ key.transpose(1, 2)
    if causal:
        late = torch.arange(Tk, device=q.device)[None] > torch.arange(T, device=q.device)[:, None] + Tk - T
        scores = scores.masked_fill(late, NEG)
    magnitude = (scale * q.abs() @ key.abs().transpose(1, 2)).amax(-1) if Tk else torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    return [x.transpose(0, 1) for x in softmax_oracle(scores, v, magnitude)]


def latent_decode_oracle(q, rows, scale):
    """One sequence: q [Tq, H, 576], rows [len, 576] of the cache."""
    Tq, n = q.shape[0], rows.shape[0]
    q, rows = q.double(), rows.double()
    scores = scale * q @ rows.T
    late = torch.arange(n, device=q.device)[None] >= n - Tq + 1 + torch.arange(Tq, device=q.device)[:, None]
    scores = scores.masked_fill(late[:, None], NEG)
    magnitude = (scale * q.abs() @ rows.abs().T).amax(-1) if n else torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    return softmax_oracle(scores, rows[:, :512], magnitude)


def paged(lens, page, seed=0, device="cuda", spare=2, filler=0.0, width=576):
    """A cache of these lengths on shuffled pages; what no sequence has holds `filler`.  Returns (cache, table, lens, rows of each)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    need = [-(-x // page) for x in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    cache = torch.full((pages, page, width), filler, device=device).bfloat16()
    table = torch.full((len(lens), max(max(need), 1)), -7, dtype=torch.int32)
    at, rows = 0, []
    for b, n in enumerate(lens):
        mine = order[at:at + need[b]]
        table[b, :need[b]] = mine.int()
        at += need[b]
        x = torch.randn(n, width, generator=gen, device=device).bfloat16()
        rows.append(x)
        for i in range(need[b]):
            part = x[i * page:(i + 1) * page]
            cache[mine[i], :part.shape[0]] = part
    return cache, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device), rows


SCALE = 1 / math.sqrt(192)
