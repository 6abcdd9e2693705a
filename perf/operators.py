"""The linear and latent attention operators as measurable cases.

One case is one call of a serving program: a decoding step, a verification step over drafted tokens, a prompt, a packed
batch of prompts.  ``own`` selects between the package's operators and the same mathematics in elementary torch operations.
"""
import math
import random

import torch

own = False

D = 128                      # linear attention: head dimension; latent attention: unrotated part of a key, and a value
LATENT, ROPE = 512, 64       # latent attention: shared vector of a token, rotated part of its key
CHUNK = 128                  # most tokens of a chunk in the plain form of linear attention
NEG = float("-inf")


# ------------------------------------------------------------------------------------------------------------ cases
def _linear(name, lens, H, Hk=None, packed=False, decay="token", state_in="none", state_out="fp32"):
    """Sequences of these lengths, packed or (all equal) side by side; H value heads, Hk heads of queries and keys; decays of every
    token and head, or one constant of each head; the states' types."""
    return {"name": name, "op": "linear", "lens": "+".join(map(str, lens)), "H": H, "Hk": Hk or H, "packed": packed,
            "decay": decay, "state_in": state_in, "state_out": state_out}


def _decode(name, lens, H, Tq=1, page=64):
    """A step of Tq tokens behind every sequence; cache lengths with the new tokens among them."""
    return {"name": name, "op": "decode", "lens": "+".join(map(str, lens)), "H": H, "Tq": Tq, "page": page}


def _prompt(name, lens, H, prefix=None, packed=False):
    """Prompts of these lengths, each behind a prefix whose keys and values are there already."""
    prefix = prefix or [0] * len(lens)
    return {"name": name, "op": "prompt", "lens": "+".join(map(str, lens)), "prefix": "+".join(map(str, prefix)), "H": H,
            "packed": packed}


def _ints(text):
    return [int(x) for x in text.split("+")]


def _ragged(n, lo, hi, seed):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(n)]


def listed():
    return [
        # one user's next token through a linear layer: the smallest call, all of it latency
        _linear("linear_step_single", [1], 32, state_in="fp32"),
        # next token of a serving batch, states kept in bf16: states read and written once
        _linear("linear_step_batch", [1] * 256, 64, state_in="bf16", state_out="bf16"),
        # one prompt of ordinary length with constant decays
        _linear("linear_prompt_single", [777], 32, decay="head"),
        # a packed handful of prompts that continue from states; queries and keys shared by four value heads
        _linear("linear_packed_shared", [1300, 1, 547, 2048, 963, 63, 271, 2999], 32, 8, packed=True, state_in="fp32"),
        # one long prompt of a wide model
        _linear("linear_prefill_8k_wide", [8192], 96, state_in="fp32"),
        # offline throughput: a full batch of long sequences
        _linear("linear_throughput_16k", [16384] * 8, 64, state_in="bf16", state_out="bf16"),
        # one user's next token through a latent layer, in the middle of a conversation
        _decode("latent_decode_single", [2989], 32),
        # next token of a serving batch of uneven conversations
        _decode("latent_decode_batch", _ragged(128, 1, 8192, 3), 64),
        # verification of three tokens behind a few long documents, 128 heads, small pages
        _decode("latent_decode_long_drafts", [131072, 50001, 90017], 128, Tq=3, page=16),
        # one prompt of ordinary length
        _prompt("latent_prompt_single", [777], 32),
        # a packed batch of prompts, some of them behind cached prefixes
        _prompt("latent_prompt_packed", [1300, 1, 547, 2048, 963, 63, 271, 999], 16, [0, 700, 0, 1024, 4001, 0, 129, 0], packed=True),
        # one long prompt
        _prompt("latent_prefill_8k", [8192], 32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more call of the same kinds: sizes over their whole range, odd ones included."""
    kind = rng.choice(["step", "linear", "linear_packed", "decode", "decode", "prompt", "prompt_packed"])
    if kind in ("step", "linear", "linear_packed"):
        H = rng.choice([2, 4, 8, 16, 24, 32, 48, 64, 96])
        Hk = H // rng.choice([1, 1, 2])
        state = rng.choice(["fp32", "bf16"])
        state_in, decay = rng.choice(["none", state]), rng.choice(["token", "head"])
        if kind == "step":
            c = _linear("", [1] * _log_int(rng, 1, 16384 // H), H, Hk, rng.random() < 0.3, decay, state, state)
        elif kind == "linear":
            T = _log_int(rng, 2, min(65536, 3_000_000 // H))
            B = _log_int(rng, 1, max(1, min(32, 4_000_000 // (T * H))))
            c = _linear("", [T] * B, H, Hk, False, decay, state_in, state)
        else:
            n = _log_int(rng, 2, 64)
            top = _log_int(rng, 16, max(17, min(8192, 4_000_000 // (n * H))))
            c = _linear("", [rng.randint(1, top) for _ in range(n)], H, Hk, True, decay, state_in, state)
    elif kind == "decode":
        H = rng.choice([4, 8, 12, 16, 24, 32, 40, 64, 96, 128])
        B = _log_int(rng, 1, 256)
        top = _log_int(rng, 16, min(131072, 500_000 // B))
        c = _decode("", [rng.randint(max(1, top // 8), top) for _ in range(B)], H, rng.choice([1, 1, 1, 2, 4]),
                    rng.choice([16, 32, 64, 128]))
    else:
        H = rng.choice([2, 4, 8, 16, 32, 64])
        if kind == "prompt":
            T = _log_int(rng, 2, min(8192, int(math.sqrt(1.8e9 / H))))
            B = _log_int(rng, 1, max(1, min(16, int(1.8e9 / (T * T * H)))))
            prefix = 0 if rng.random() < 0.5 else _log_int(rng, 1, max(1, min(8192, int(1.8e9 / (T * H * B)) - T)))
            c = _prompt("", [T] * B, H, [prefix] * B)
        else:
            n = _log_int(rng, 2, 32)
            top = _log_int(rng, 16, max(17, min(4096, int(math.sqrt(5e8 / (n * H))))))
            c = _prompt("", [rng.randint(1, top) for _ in range(n)], H, [rng.choice([0, rng.randint(1, top)]) for _ in range(n)], True)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------------------- inputs
def _cumulative(lens, dev):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(dev)


def _padding(lens, dev):
    """[N, longest] token numbers of packed sequences, where they are real, and the way back."""
    top, at, rows, back = max(lens), 0, [], []
    for n, x in enumerate(lens):
        rows.append(torch.clamp(torch.arange(top), max=max(x - 1, 0)) + at)
        back.append(torch.arange(x) + n * top)
        at += x
    real = torch.arange(top)[None] < torch.tensor(lens)[:, None]
    return {"at": torch.stack(rows).clamp(max=max(at - 1, 0)).to(dev), "real": real.to(dev), "back": torch.cat(back).to(dev)}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    bf = torch.bfloat16
    lens, H = _ints(case["lens"]), case["H"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32 if math.prod(shape) < 1 << 28 else bf)

    s = {"case": case}
    if case["op"] == "linear":
        Hk, N, total = case["Hk"], len(lens), sum(lens)
        B, T = (1, total) if case["packed"] else (N, lens[0])
        # queries and keys of norm one, as the layers in front make them
        s["q"], s["k"] = (torch.nn.functional.normalize(randn(B, T, Hk, D).float(), dim=-1).to(bf) for _ in range(2))
        s["v"] = randn(B, T, H, D).to(bf)
        if case["decay"] == "head":      # a geometric row of constants, from half a token's memory to some hundred tokens'
            s["g"] = -torch.exp2(-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H) * (1 + 0.01 * torch.rand(H, generator=gen, device=dev))
        else:                            # the usual gate: -exp(a) softplus(x)
            a = torch.rand(H, generator=gen, device=dev) * 4 - 4
            s["g"] = -torch.exp(a) * torch.nn.functional.softplus(randn(B, T, H).float())
        s["scale"] = D ** -0.5
        kind = {"fp32": torch.float32, "bf16": bf}
        s["h0"] = randn(N, H, D, D).to(kind[case["state_in"]]) if case["state_in"] != "none" else None
        s["hT"] = torch.zeros(N, H, D, D, dtype=kind[case["state_out"]], device=dev) if case["state_out"] != "none" else None
        s["out"] = torch.zeros(B, T, H, D, dtype=bf, device=dev)
        s["cu"] = _cumulative(lens, dev) if case["packed"] else None
        s["pad"] = _padding(lens, dev) if case["packed"] else None
    elif case["op"] == "decode":
        B, Tq, page = len(lens), case["Tq"], case["page"]
        need = [-(-x // page) for x in lens]
        pages = sum(need)
        s["cache"] = randn(pages, page, LATENT + ROPE).to(bf)
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32).cpu()
        table, at = torch.zeros(B, max(need), dtype=torch.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"] = table.to(dev)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q"] = randn(B, Tq, H, LATENT + ROPE).to(bf)
        s["scale"] = (D + ROPE) ** -0.5
        s["out"] = torch.zeros(B, Tq, H, LATENT, dtype=bf, device=dev)
        s["lse"] = torch.zeros(B, Tq, H, dtype=torch.float32, device=dev)
    else:
        prefix = _ints(case["prefix"])
        keys = [a + b for a, b in zip(lens, prefix)]
        B, T, Tk = (1, sum(lens), sum(keys)) if case["packed"] else (len(lens), lens[0], keys[0])
        s["q"] = randn(B, T, H, D + ROPE).to(bf)
        s["kv"] = randn(B, Tk, H, 2 * D).to(bf)      # keys and values leave one projection side by side
        s["k_rope"] = randn(B, Tk, ROPE).to(bf)
        s["scale"] = (D + ROPE) ** -0.5
        s["out"] = torch.zeros(B, T, H, D, dtype=bf, device=dev)
        s["lse"] = torch.zeros(B, T, H, dtype=torch.float32, device=dev)
        s["cu"] = _cumulative(lens, dev) if case["packed"] else None
        s["cu_k"] = _cumulative(keys, dev) if case["packed"] else None
        if case["packed"]:
            s["pad"], s["pad_k"] = _padding(lens, dev), _padding(keys, dev)
        s["n_q"], s["n_k"] = torch.tensor(lens, device=dev), torch.tensor(keys, device=dev)
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        import flashkda_b200 as lib
        if op == "linear":
            lib.linear_attention_fwd(s["q"], s["k"], s["v"], s["g"], s["scale"], s["out"], s["h0"], s["hT"], s["cu"])
            return {"out": s["out"], "final_state": s["hT"]}
        if op == "decode":
            lib.latent_attention_decode(s["q"], s["cache"], s["table"], s["lens"], s["scale"], s["out"], s["lse"])
        else:
            lib.latent_attention_fwd(s["q"], s["kv"][..., :D], s["k_rope"], s["kv"][..., D:], s["scale"], s["out"], s["lse"],
                                     s["cu"], s["cu_k"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "linear":
        return _plain_linear(s)
    return _plain_decode(s) if op == "decode" else _plain_prompt(s)


def _plain_linear(s):
    q, k, v, g, pad = s["q"], s["k"], s["v"], s["g"], s["pad"]
    H = v.shape[2]
    if g.dim() == 1:
        g = g.expand(v.shape[:3])
    if pad is not None:                # packed sequences side by side; padding adds nothing and does not decay
        q, k, v, g = (x[0][pad["at"]] for x in (q, k, v, g))
        k, g = k * pad["real"][..., None, None], g * pad["real"][..., None]
    N, T = v.shape[:2]
    C = min(CHUNK, T)
    n = -(-T // C)

    def chunks(x):                     # [N, H, chunks, C, ...] in 32 bits (decays in 64: their sums go through exp)
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, n * C - T))
        x = x.reshape(N, n, C, *x.shape[2:]).transpose(2, 3).transpose(1, 2)
        return x.double() if x.dim() == 4 else x.float().repeat_interleave(H // x.shape[1], 1)

    q, k, v, G = chunks(q), chunks(k), chunks(v), chunks(g).cumsum(-1)
    lower = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    P = (q @ k.transpose(-1, -2)) * torch.where(lower, G[..., :, None] - G[..., None, :], NEG).exp().float()
    local = (v * (G[..., -1:] - G).exp().float()[..., None]).transpose(-1, -2) @ k       # [N, H, chunks, V, K]
    first = torch.zeros(N, H, 1, D, D, device=q.device) if s["h0"] is None else s["h0"].float()[:, :, None]
    total = torch.nn.functional.pad(G[..., -1].cumsum(-1), (1, 0))                         # decay up to each chunk
    upto = torch.ones(n + 1, n + 1, dtype=torch.bool, device=q.device).tril()
    carry = torch.where(upto, total[..., :, None] - total[..., None, :], NEG).exp().float()
    states = (carry @ torch.cat([first, local], 2).flatten(3)).view(N, H, n + 1, D, D)   # in front of each chunk, and the last
    out = P @ v + (q @ states[:, :, :-1].transpose(-1, -2)) * G.exp().float()[..., None]
    out = (s["scale"] * out).transpose(1, 2).transpose(2, 3).reshape(N, n * C, H, D)[:, :T]
    if pad is not None:
        out = out.flatten(0, 1)[pad["back"]][None]
    hT = None if s["hT"] is None else states[:, :, -1].to(s["hT"].dtype)
    return {"out": out.to(torch.bfloat16), "final_state": hT}


def _softmax_values(scores, values):
    """softmax(scores) values over the last axis, and the logarithm of the sum; rows of minus infinities give 0 and -inf."""
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == NEG, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    out = (p @ values) / torch.where(total == 0, 1.0, total)
    return out, (total.log() + torch.where(top == NEG, 0.0, top))[..., 0]


def _plain_decode(s):
    q, cache, table, lens = s["q"], s["cache"], s["table"].long(), s["lens"].long()
    B, Tq, H, _ = q.shape
    page = cache.shape[1]
    pos = torch.arange(table.shape[1] * page, device=q.device)
    rows = cache[table[:, pos // page], pos % page].float()                              # [B, positions, 576]
    scores = s["scale"] * (q.float().reshape(B, Tq * H, -1) @ rows.transpose(1, 2))
    seen = lens[:, None] - Tq + 1 + torch.arange(Tq, device=q.device)                     # positions that a new token sees
    scores = torch.where(pos < seen.repeat_interleave(H, 1)[..., None], scores, NEG)
    out, lse = _softmax_values(scores, rows[..., :LATENT])
    return {"out": out.view(B, Tq, H, LATENT).to(torch.bfloat16), "lse": lse.view(B, Tq, H)}


def _plain_prompt(s):
    q, kv, k_rope = s["q"], s["kv"], s["k_rope"]
    if s["cu"] is not None:
        q, kv, k_rope = q[0][s["pad"]["at"]], kv[0][s["pad_k"]["at"]], k_rope[0][s["pad_k"]["at"]]
    H = q.shape[2]
    k = torch.cat([kv[..., :D], k_rope[:, :, None].expand(-1, -1, H, -1)], -1)
    scores = s["scale"] * (q.float().transpose(1, 2) @ k.float().permute(0, 2, 3, 1))
    i, j = torch.arange(q.shape[1], device=q.device), torch.arange(kv.shape[1], device=q.device)
    n_q, n_k = s["n_q"][:, None, None, None], s["n_k"][:, None, None, None]
    scores = torch.where((j <= i[:, None] + n_k - n_q) & (j < n_k), scores, NEG)
    out, lse = _softmax_values(scores, kv[..., D:].float().transpose(1, 2))
    out, lse = out.transpose(1, 2), lse.transpose(1, 2)
    if s["cu"] is not None:
        out, lse = (x.flatten(0, 1)[s["pad"]["back"]][None] for x in (out, lse))
    return {"out": out.to(torch.bfloat16), "lse": lse.contiguous()}


# ------------------------------------------------------------------------------------------------ what a pass takes
def work(case):
    lens, H = _ints(case["lens"]), case["H"]
    n = sum(lens)
    if case["op"] == "linear":
        width = {"none": 0, "bf16": 2, "fp32": 4}
        state = len(lens) * H * D * D * (width[case["state_in"]] + width[case["state_out"]])
        g = 4 * H * (1 if case["decay"] == "head" else n)
        # products of the chunked form with 64 tokens in a chunk (half of q k^T and of its product with v are masked); a single
        # token: the state once for the update and once for the output
        per = 4 * D * D + (2 * 64 * D if max(lens) > 1 else 0)
        return {"bytes": n * 512 * (case["Hk"] + H) + g + state, "flops": n * H * per}
    if case["op"] == "decode":
        Tq = case["Tq"]
        rows = len(lens) * Tq * H
        seen = sum(max(0, x - j) for x in lens for j in range(Tq)) * H
        return {"bytes": n * 2 * (LATENT + ROPE) + rows * (2 * (2 * LATENT + ROPE) + 4), "flops": 2 * (2 * LATENT + ROPE) * seen}
    prefix = _ints(case["prefix"])
    pairs = sum(x * p + x * (x + 1) // 2 for x, p in zip(lens, prefix))
    keys = n + sum(prefix)
    return {"bytes": n * H * (2 * (2 * D + ROPE) + 4) + keys * (H * 4 * D + 2 * ROPE), "flops": 2 * (2 * D + ROPE) * pairs * H}


# ---------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    lens, H = _ints(case["lens"]), case["H"]
    if case["op"] == "linear":
        return _exact_linear(s, case, lens, H)
    return _exact_decode(s, lens, H) if case["op"] == "decode" else _exact_prompt(s, case, lens, H)


def _exact_linear(s, case, lens, H):
    """o_t = scale (sum over s <= t of exp(g_{s+1} + ... + g_t) (q_t . k_s) v_s + exp(g_1 + ... + g_t) S_0 q_t)"""
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    hT = None if s["hT"] is None else torch.zeros(s["hT"].shape, dtype=torch.float64, device="cuda")
    if max(lens) == 1:                 # single tokens: all sequences at once
        q, k = (x.double().reshape(-1, case["Hk"], D).repeat_interleave(H // case["Hk"], 1) for x in (s["q"], s["k"]))
        decay = torch.exp(s["g"].double()).expand(len(lens), H) if s["g"].dim() == 1 else torch.exp(s["g"].double()).reshape(-1, H)
        S = s["v"].double().reshape(-1, H, D)[..., :, None] * k[..., None, :]
        if s["h0"] is not None:
            S = S + decay[..., None, None] * s["h0"].double()
        return {"out": (s["scale"] * (S * q[..., None, :]).sum(-1)).reshape(out.shape), "final_state": S}
    at = 0
    for n, T in enumerate(lens):
        for h in range(H):
            b, lo = (0, at) if case["packed"] else (n, 0)
            hk = h // (H // case["Hk"])
            q, k = (x[b, lo:lo + T, hk].double() for x in (s["q"], s["k"]))
            v = s["v"][b, lo:lo + T, h].double()
            g = s["g"][h].double().expand(T) if s["g"].dim() == 1 else s["g"][b, lo:lo + T, h].double()
            G = torch.cumsum(g, 0)
            S0 = None if s["h0"] is None else s["h0"][n, h].double()
            for i in range(0, T, 8192):
                m = min(T, i + 8192)
                for j in range(0, m, 8192):
                    e = min(m, j + 8192)
                    w = torch.exp((G[i:m, None] - G[None, j:e]).clamp_(max=0.0))
                    w *= q[i:m] @ k[j:e].T
                    if e == m:
                        w = w.tril()
                    out[b, lo + i:lo + m, h] += s["scale"] * (w @ v[j:e])
                if S0 is not None:
                    out[b, lo + i:lo + m, h] += s["scale"] * torch.exp(G[i:m, None]) * (q[i:m] @ S0.T)
            if hT is not None:
                hT[n, h] = (v * torch.exp(G[-1] - G)[:, None]).T @ k
                if S0 is not None:
                    hT[n, h] += torch.exp(G[-1]) * S0
        at += T
    return {"out": out, "final_state": hT}


def _exact_decode(s, lens, H):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    Tq, page = s["q"].shape[1], s["cache"].shape[1]
    for b, n in enumerate(lens):
        used = s["table"][b, :-(-n // page)].long()
        rows = s["cache"].index_select(0, used).flatten(0, 1)[:n].double()
        for j in range(Tq):
            m = n - Tq + 1 + j
            if m <= 0:
                lse[b, j] = NEG
                continue
            x = s["scale"] * (s["q"][b, j].double() @ rows[:m].T)
            lse[b, j] = torch.logsumexp(x, -1)
            out[b, j] = torch.exp(x - lse[b, j][:, None]) @ rows[:m, :LATENT]
    return {"out": out, "lse": lse}


def _exact_prompt(s, case, lens, H):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    at = at_k = 0
    for n, (T, p) in enumerate(zip(lens, _ints(case["prefix"]))):
        b, lo, lo_k = (0, at, at_k) if case["packed"] else (n, 0, 0)
        late = torch.arange(T + p, device="cuda")[None] > torch.arange(T, device="cuda")[:, None] + p
        rope = s["k_rope"][b, lo_k:lo_k + T + p].double()
        for h in range(H):
            q, kv = s["q"][b, lo:lo + T, h].double(), s["kv"][b, lo_k:lo_k + T + p, h].double()
            x = s["scale"] * (q[:, :D] @ kv[:, :D].T + q[:, D:] @ rope.T)
            x.masked_fill_(late, NEG)
            z = torch.logsumexp(x, -1)
            lse[b, lo:lo + T, h] = z
            out[b, lo:lo + T, h] = torch.exp(x - z[:, None]) @ kv[:, D:]
        at, at_k = at + T, at_k + T + p
    return {"out": out, "lse": lse}
