"""Latent attention, expanded and absorbed, against softmax in 64 bits."""
import pytest
import torch

import flashkda_b200
from attention_testlib import SCALE, assert_within, latent_decode_oracle, latent_prompt_oracle, paged
from flashkda_b200 import _lib

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------- on the CPU
def test_there_is_no_cpu_path():
    z = lambda *s: torch.zeros(*s).bfloat16()
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        flashkda_b200.latent_attention_fwd(z(1, 4, 2, 192), z(1, 4, 2, 128), z(1, 4, 64), z(1, 4, 2, 128), 1.0, z(1, 4, 2, 128))
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        flashkda_b200.latent_attention_decode(z(1, 1, 2, 576), z(4, 16, 576), torch.zeros(1, 4).int(), torch.zeros(1).int(), 1.0, z(1, 1, 2, 512))


def prompt_params(**over):
    fake = dict.fromkeys(("q", "k", "k_rope", "v", "out"), 0x1000)
    stride = (4 * 256, 256, 128)
    p = dict(B=1, T=4, Tk=4, H=2, N=1, q_stride=(4 * 384, 384, 192), k_stride=stride, v_stride=stride, out_stride=stride, k_rope_stride=(256, 64),
             scale=1.0, causal=1, **fake)
    p.update(over)
    return _lib.LatentParams(**p)


def decode_params(**over):
    fake = dict.fromkeys(("q", "cache", "block_table", "cache_lens", "out", "workspace"), 0x1000)
    p = dict(B=1, Tq=1, H=2, pages=4, page_size=16, max_pages=4, q_stride=(2 * 576, 576), out_stride=(1024, 512), cache_stride=(16 * 576, 576),
             block_table_stride=4, scale=1.0, workspace_bytes=1 << 40, **fake)
    p.update(over)
    return _lib.LatentDecodeParams(**p)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), 1), (dict(v=None), 1), (dict(cu_seqlens=0x1000), 1), (dict(B=0), 2), (dict(N=3), 2), (dict(T=-1), 2), (dict(Tk=2 ** 31), 2),
    (dict(H=0), 2), (dict(B=2, N=2, cu_seqlens=0x1000, cu_seqlens_k=0x1000), 4), (dict(k=0x1004), 8), (dict(q_stride=(1536, 380, 192)), 8),
    (dict(k_rope_stride=(256, 60)), 8), (dict(out_stride=(1024, 256, 1)), 8), (dict(scale=0.0), 11), (dict(scale=-1.0), 11),
    (dict(scale=float("nan")), 11), (dict(scale=float("inf")), 11)])
def test_refusals_of_the_c_entry_for_prompts(over, status):
    assert _lib.lib().fkda_latent_attention_fwd(prompt_params(**over), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(q=None), 1), (dict(cache_lens=None), 1), (dict(block_table=None), 1), (dict(pages=0), 1), (dict(page_size=8), 2), (dict(page_size=24), 2),
    (dict(B=-1), 2), (dict(max_pages=2 ** 30), 2), (dict(H=70000), 2), (dict(Tq=2 ** 30, H=4), 2), (dict(workspace=None), 5), (dict(workspace=0x1010), 5),
    (dict(workspace_bytes=4096), 5), (dict(q=0x1002), 8), (dict(cache_stride=(16 * 576, 572)), 8), (dict(q_stride=(2 * 576, 577)), 8), (dict(scale=0.0), 11)])
def test_refusals_of_the_c_entry_for_decoding(over, status):
    assert _lib.lib().fkda_latent_attention_decode(decode_params(**over), None) == status


def test_nothing_to_do_launches_nothing():
    L = _lib.lib()
    assert L.fkda_latent_attention_fwd(prompt_params(T=0), None) == 0
    assert L.fkda_latent_attention_decode(decode_params(B=0), None) == 0
    assert L.fkda_last_launch_count() == 0
    assert L.fkda_latent_attention_fwd(None, None) == 1 and L.fkda_latent_attention_decode(None, None) == 1


# ---------------------------------------------------------------------------------------------------------- prompts
def prompt_inputs(B, T, Tk, H, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    return dict(q=rnd(B, T, H, 192), k=rnd(B, Tk, H, 128), k_rope=rnd(B, Tk, 64), v=rnd(B, Tk, H, 128),
                out=torch.full((B, T, H, 128), 7.0, device="cuda").bfloat16(), lse=torch.full((B, T, H), 7.0, device="cuda"))


def prompt(d, scale=SCALE, **kw):
    flashkda_b200.latent_attention_fwd(d["q"], d["k"], d["k_rope"], d["v"], scale, d["out"], d["lse"], **kw)


def check_prompt(d, b, rows, keys, scale=SCALE, causal=True):
    out, lse, bound, lse_bound = latent_prompt_oracle(d["q"][b, rows], d["k"][b, keys], d["k_rope"][b, keys], d["v"][b, keys], scale, causal)
    assert_within(d["out"][b, rows], out, bound, "out")
    if d["lse"] is not None:
        assert_within(d["lse"][b, rows], lse, lse_bound, "lse")


@gpu
@pytest.mark.parametrize("T,Tk", [(1, 1), (1, 128), (1, 129), (127, 127), (128, 128), (129, 129), (255, 300), (256, 256), (257, 257), (130, 700), (511, 640)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(T, Tk, causal):
    d = prompt_inputs(2, T, Tk, 2, T + Tk)
    prompt(d, causal=causal)
    for b in range(2):
        check_prompt(d, b, slice(None), slice(None), causal=causal)
    assert flashkda_b200.operator_status() == 0


@gpu
@pytest.mark.parametrize("T,Tk", [(5, 3), (300, 40), (300, 170), (4, 0), (300, 0)])
def test_rows_that_see_nothing(T, Tk):
    d = prompt_inputs(1, T, Tk, 2, 1)
    prompt(d)
    check_prompt(d, 0, slice(None), slice(None))
    blind = T - Tk
    assert bool((d["out"][:, :blind] == 0).all()) and bool((d["lse"][:, :blind] == float("-inf")).all())


@gpu
@pytest.mark.parametrize("lens,prefix", [([130, 1, 300, 64], [0, 70, 0, 200]), ([0, 5, 0, 257], [3, 0, 0, 1]), ([1] * 40, list(range(40)))], ids=str)
def test_packed_prompts(lens, prefix):
    """NaN in front of, between and behind the rows that the sequences have; rows that none has stay as they were."""
    keys = [a + b for a, b in zip(lens, prefix)]
    T, Tk, extra = sum(lens), sum(keys), 5
    d = prompt_inputs(1, T + extra, Tk + extra, 2, 2)
    for x in ("k", "k_rope", "v"):
        d[x][:, Tk:] = float("nan")
    d["q"][:, T:] = float("nan")
    cu, cu_k = (torch.tensor([0] + x).cumsum(0).cuda() for x in (lens, keys))
    prompt(d, cu_seqlens=cu, cu_seqlens_k=cu_k)
    at = at_k = 0
    for n, m in zip(lens, keys):
        if n:
            check_prompt(d, 0, slice(at, at + n), slice(at_k, at_k + m))
        at, at_k = at + n, at_k + m
    assert bool((d["out"][:, T:] == 7.0).all()) and bool((d["lse"][:, T:] == 7.0).all())


@gpu
def test_a_neighbour_that_is_not_finite():
    lens = [100, 150, 70]
    d = prompt_inputs(1, sum(lens), sum(lens), 2, 3)
    for x in ("q", "k", "k_rope", "v"):
        d[x][:, :100] = float("inf")
        d[x][:, 250:] = float("nan")
    prompt(d, cu_seqlens=torch.tensor([0, 100, 250, 320], device="cuda"))
    check_prompt(d, 0, slice(100, 250), slice(100, 250))


@gpu
@pytest.mark.parametrize("spread", [1e-3, 6.0, 30.0])
def test_flat_and_peaked_scores(spread):
    """Maxima that rise along the keys, so that the running reference moves again and again."""
    d = prompt_inputs(1, 300, 900, 2, 4)
    d["q"] = (d["q"].float() * spread).bfloat16()
    d["k"] = (d["k"].float() * torch.linspace(0.1, 1, 900, device="cuda")[None, :, None, None]).bfloat16()
    prompt(d)
    check_prompt(d, 0, slice(None), slice(None))


@gpu
def test_prompt_views_and_no_lse():
    """Keys and values side by side in one projection, heads in front of tokens in q and out, rope as a slice of the compressed vector."""
    B, T, H = 2, 140, 3
    kv = torch.randn(B, T, H, 256, device="cuda").bfloat16()
    q = torch.randn(B, H, T, 192, device="cuda").bfloat16().transpose(1, 2)
    rope = torch.randn(B, T, 576, device="cuda").bfloat16()[..., 512:]
    out = torch.full((B, H, T, 128), 7.0, device="cuda").bfloat16().transpose(1, 2)
    d = dict(q=q, k=kv[..., :128], v=kv[..., 128:], k_rope=rope, out=out, lse=None)
    prompt(d, 0.05)
    for b in range(B):
        check_prompt(d, b, slice(None), slice(None), 0.05)


@gpu
def test_prompts_join_over_parts_of_the_keys():
    """Softmax over all keys from two calls on halves of them, by their lse."""
    d = prompt_inputs(1, 90, 600, 2, 6)
    whole, parts = d["out"], []
    prompt(d, causal=False)
    for keys in (slice(0, 333), slice(333, 600)):
        e = d | {x: d[x][:, keys] for x in ("k", "k_rope", "v")} | dict(out=torch.empty_like(whole), lse=torch.empty_like(d["lse"]))
        prompt(e, causal=False)
        parts.append(e)
    w = torch.softmax(torch.stack([p["lse"] for p in parts]).double(), 0)[..., None]
    out, lse, bound, _ = latent_prompt_oracle(*(d[x][0] for x in ("q", "k", "k_rope", "v")), SCALE, False)
    joined = sum(a * p["out"].double() for a, p in zip(w, parts))
    assert_within(joined[0], out, 3 * bound, "joined")


# ---------------------------------------------------------------------------------------------------------- decoding
def decode_case(lens, H, Tq=1, page=64, seed=0, filler=0.0):
    cache, table, n, rows = paged(lens, page, seed, filler=filler)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(len(lens), Tq, H, 576, generator=gen, device="cuda").bfloat16()
    return dict(q=q, cache=cache, table=table, lens=n, rows=rows, out=torch.full((len(lens), Tq, H, 512), 7.0, device="cuda").bfloat16(),
                lse=torch.full((len(lens), Tq, H), 7.0, device="cuda"))


def decode(d, scale=SCALE, **kw):
    flashkda_b200.latent_attention_decode(d["q"], d["cache"], d["table"], d["lens"], scale, d["out"], d["lse"], **kw)


def check_decode(d, scale=SCALE):
    for b, rows in enumerate(d["rows"]):
        out, lse, bound, lse_bound = latent_decode_oracle(d["q"][b], rows, scale)
        # joined parts: two more roundings of fp32 each
        assert_within(d["out"][b], out, bound, f"out of sequence {b}")
        if d["lse"] is not None:
            assert_within(d["lse"][b], lse, lse_bound, f"lse of sequence {b}")


@gpu
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 128])
def test_cache_lengths_and_pages(n, page):
    """Pages that end inside a tile, and NaN wherever no sequence has a token."""
    d = decode_case([n, max(1, n - 7)], 16, page=page, seed=n, filler=float("nan"))
    decode(d)
    check_decode(d)
    assert flashkda_b200.operator_status() == 0


@gpu
@pytest.mark.parametrize("H", [1, 5, 16, 32, 33, 64, 65, 96, 128])
@pytest.mark.parametrize("Tq", [1, 2, 4])
def test_heads_and_drafted_tokens(H, Tq):
    d = decode_case([3, 200, 1, 131], H, Tq, 32, seed=H, filler=float("nan"))
    decode(d)
    check_decode(d)


@gpu
@pytest.mark.parametrize("lens", [[0], [0, 0, 70], [70, 0, 0, 1], [0, 130]], ids=str)
def test_sequences_without_tokens(lens):
    d = decode_case(lens, 8, 2)
    decode(d)
    check_decode(d)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((d["out"][b] == 0).all()) and bool((d["lse"][b] == float("-inf")).all())


@gpu
@pytest.mark.parametrize("lens,H", [([20000], 32), ([9000, 3, 64 * 148, 1], 64), ([500] * 150, 16), ([64] * 300, 16), (list(range(1, 400, 3)), 8)], ids=lambda x: str(x)[:20])
def test_cuts_through_sequences(lens, H):
    d = decode_case(lens, H, seed=7)
    decode(d)
    check_decode(d)


@gpu
@pytest.mark.parametrize("spread", [1e-3, 8.0, 40.0])
def test_decode_flat_and_peaked_scores(spread):
    d = decode_case([5000, 700], 40, seed=8)
    d["q"] = (d["q"].float() * spread).bfloat16()
    decode(d)
    check_decode(d)


@gpu
def test_decode_views():
    """A cache and its rows inside wider ones, heads of q and out inside wider rows."""
    d = decode_case([100, 333], 6, 3, 32, seed=9)
    wide = torch.zeros(d["cache"].shape[0], 2, 32, 584, device="cuda").bfloat16()
    wide[:, 1, :, :576] = d["cache"]
    q = torch.zeros(2, 3 * 6, 640, device="cuda").bfloat16()
    q[..., 64:] = d["q"].flatten(1, 2)
    d["cache"], d["q"] = wide[:, 1, :, :576], q.unflatten(1, (3, 6))[..., 64:]
    d["out"] = torch.zeros(2, 20, 520, device="cuda").bfloat16()[:, 1:19, :512].unflatten(1, (3, 6))
    table = torch.zeros(2, 40, dtype=torch.int32, device="cuda")
    table[:, :d["table"].shape[1]] = d["table"]
    d["table"] = table[:, :d["table"].shape[1]]
    d["lse"] = None
    decode(d)
    check_decode(d)


@gpu
def test_a_length_beyond_the_table_counts_as_its_end():
    d = decode_case([128, 64], 4, seed=10)
    d["lens"] = torch.tensor([1000, -5], dtype=torch.int32, device="cuda")
    d["rows"][1] = d["rows"][1][:0]
    decode(d)
    check_decode(d)


@gpu
def test_decode_repeats_bit_for_bit_on_two_streams_at_once():
    d = decode_case([3000, 17, 900], 32, seed=11)
    decode(d)
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            e = d | dict(out=torch.zeros_like(d["out"]), lse=torch.zeros_like(d["lse"]))
            for _ in range(20):
                decode(e)
            outs.append(e)
    torch.cuda.synchronize()
    for e in outs:
        assert torch.equal(e["out"], d["out"]) and torch.equal(e["lse"], d["lse"])


@gpu
def test_decode_captured_with_its_own_workspace_and_longer_caches_at_replay():
    d = decode_case([200, 900], 16, seed=12)
    ws = torch.empty(flashkda_b200.latent_decode_workspace_size(2, 1, 16), dtype=torch.uint8, device="cuda")
    full = d["lens"].clone()
    d["lens"].copy_(torch.tensor([3, 70]))
    decode(d, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(d, workspace=ws)
    d["lens"].copy_(full)
    ws.fill_(255)
    graph.replay()
    torch.cuda.synchronize()
    check_decode(d)


@gpu
@pytest.mark.parametrize("change,match", [
    (dict(q=lambda x: x.float()), "q must be bfloat16"), (dict(q=lambda x: x[..., :512]), "q must be"), (dict(cache=lambda x: x[:, :8]), "multiple of 16"),
    (dict(cache=lambda x: x[..., :512]), "cache must be"), (dict(table=lambda x: x.long()), "block_table must be int32"), (dict(table=lambda x: x[:1]), "block_table must be"),
    (dict(lens=lambda x: x.long()), "cache_lens must be int32"), (dict(out=lambda x: x[:, :, :2]), "out must be"), (dict(lse=lambda x: x.double()), "lse must be float32"),
    (dict(lse=lambda x: x[:, :, :2]), "lse must be"), (dict(q=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)), "heads apart"),
    (dict(cache=lambda x: torch.zeros(x.shape[0], x.shape[1], 577, device="cuda").bfloat16()[..., :576]), "16-byte aligned"), (dict(lens=lambda x: x.cpu()), "must be on CUDA"),
])
def test_decode_refusals(change, match):
    d = decode_case([20, 30], 4, 2, 16)
    for name, f in change.items():
        d[name] = f(d[name])
    with pytest.raises(RuntimeError, match=match):
        decode(d)
    with pytest.raises(RuntimeError, match="workspace must be"):
        decode(decode_case([20, 30], 4), workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="scale must be positive"):
        decode(decode_case([20, 30], 4), scale=0.0)


@gpu
@pytest.mark.parametrize("change,match", [
    (dict(q=lambda x: x[..., :128]), "q must be"), (dict(k=lambda x: x[:, :, :1]), "k must be"), (dict(k_rope=lambda x: x[..., :32]), "k_rope must be"),
    (dict(v=lambda x: x.half()), "v must be bfloat16"), (dict(out=lambda x: x[:, :3]), "out must be"), (dict(lse=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)), "lse must be contiguous"),
])
def test_prompt_refusals(change, match):
    d = prompt_inputs(1, 4, 6, 2)
    for name, f in change.items():
        d[name] = f(d[name])
    with pytest.raises(RuntimeError, match=match):
        prompt(d)
    d = prompt_inputs(1, 4, 6, 2)
    cu = torch.tensor([0, 4], device="cuda")
    for kw, why in ((dict(cu_seqlens=cu), "as many tokens"), (dict(cu_seqlens_k=cu), "needs cu_seqlens"),
                    (dict(cu_seqlens=cu, cu_seqlens_k=torch.tensor([0, 4, 6], device="cuda")), "same length")):
        with pytest.raises(RuntimeError, match=why):
            prompt(d, **kw)


# ---------------------------------------------------------------------------------------------------------- together
@gpu
def test_a_model_of_linear_and_latent_layers_generates():
    """A KDA layer, a linear layer and a latent layer: a prompt, then tokens one by one with the states and the cache that it left;
    every layer of every step against its oracle on the inputs that it had."""
    from attention_testlib import check_linear
    T, new, H, page = 150, 3, 4, 16
    gen = torch.Generator(device="cuda").manual_seed(13)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    up_k, up_v = (rnd(H, 128, 512).bfloat16() / 16 for _ in range(2))
    kda, lin = torch.zeros(1, H, 128, 128, device="cuda"), torch.zeros(1, H, 128, 128, device="cuda")
    cache = torch.full((12, page, 576), float("nan"), device="cuda").bfloat16()
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).int()[None].cuda()
    x = rnd(1, T, H, 128).bfloat16()
    at = 0
    for step in range(1 + new):
        n = x.shape[1]
        # KDA
        y = torch.empty_like(x)
        flashkda_b200.fwd(x, x, x, x, x[..., 0].contiguous(), 0.1, y, torch.zeros(H, device="cuda"), torch.zeros(H, 128, device="cuda"), -5.0, kda, kda)
        # linear
        unit = torch.nn.functional.normalize(y.float(), dim=-1).bfloat16()
        d = dict(q=unit, k=unit.flip(-1), v=y, g=-torch.rand(1, n, H, generator=gen, device="cuda"), cu=None, h0=lin.clone())
        z = torch.empty_like(x)
        flashkda_b200.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], 1.0, z, lin, lin)
        check_linear(d, [n], 1.0, z, lin)
        # latent: the compressed vectors go into the cache
        latent = (z.flatten(2)[:, :, :512].float() + 0.1 * rnd(1, n, 512)).bfloat16()
        rope, q_rope = rnd(1, n, 64).bfloat16(), rnd(1, n, H, 64).bfloat16()
        pos = torch.arange(at, at + n, device="cuda")
        cache[table[0, pos // page].long(), pos % page] = torch.cat([latent, rope], -1)[0]
        at += n
        q = z.float()
        if step == 0:
            k, v = (torch.einsum("btc,hdc->bthd", latent.float(), w.float()).bfloat16() for w in (up_k, up_v))
            full = torch.cat([q, q_rope.float()], -1).bfloat16()
            out = torch.empty_like(x)
            flashkda_b200.latent_attention_fwd(full, k, rope, v, SCALE, out)
            want, _, bound, _ = latent_prompt_oracle(full[0], k[0], rope[0], v[0], SCALE)
            assert_within(out[0], want, bound, "latent prompt")
        else:
            absorbed = torch.cat([torch.einsum("bthd,hdc->bthc", q, up_k.float()), q_rope.float()], -1).bfloat16()
            wide = torch.empty(1, n, H, 512, device="cuda").bfloat16()
            lens = torch.tensor([at], dtype=torch.int32, device="cuda")
            flashkda_b200.latent_attention_decode(absorbed, cache, table, lens, SCALE, wide)
            rows = cache[table[0].long()].flatten(0, 1)[:at]
            want, _, bound, _ = latent_decode_oracle(absorbed[0], rows, SCALE)
            assert_within(wide[0], want, bound, "latent decode")
            out = torch.einsum("bthc,hdc->bthd", wide.float(), up_v.float()).bfloat16()
        x = out[:, -1:].contiguous()


@gpu
def test_absorbed_and_expanded_forms_agree():
    """The last token of a prompt through both forms: queries times the keys' expansion on one side, expanded keys on the other.  With
    expansions that copy numbers both have the same products, so they differ by the weights' and the outputs' roundings alone."""
    T, H = 300, 2
    gen = torch.Generator(device="cuda").manual_seed(14)
    latent, rope = torch.randn(1, T, 512, generator=gen, device="cuda").bfloat16(), torch.randn(1, T, 64, generator=gen, device="cuda").bfloat16()
    q = torch.randn(1, T, H, 192, generator=gen, device="cuda").bfloat16()
    k = torch.stack([latent[..., 128 * h:128 * h + 128] for h in range(H)], 2)
    v = torch.stack([latent[..., 256 + 128 * h:384 + 128 * h] for h in range(H)], 2)
    out = torch.empty(1, T, H, 128, device="cuda").bfloat16()
    flashkda_b200.latent_attention_fwd(q, k, rope, v, SCALE, out)
    absorbed = torch.zeros(1, 1, H, 576, device="cuda").bfloat16()
    for h in range(H):
        absorbed[0, 0, h, 128 * h:128 * h + 128] = q[0, -1, h, :128]
    absorbed[..., 512:] = q[:, -1:, :, 128:]
    cache = torch.zeros(19, 16, 576, device="cuda").bfloat16()
    cache.view(-1, 576)[:T] = torch.cat([latent, rope], -1)[0]
    wide = torch.empty(1, 1, H, 512, device="cuda").bfloat16()
    flashkda_b200.latent_attention_decode(absorbed, cache, torch.arange(19, dtype=torch.int32, device="cuda")[None],
                                          torch.tensor([T], dtype=torch.int32, device="cuda"), SCALE, wide)
    want, _, bound, _ = latent_prompt_oracle(q[0], k[0], rope[0], v[0], SCALE)
    got = torch.stack([wide[0, 0, h, 256 + 128 * h:384 + 128 * h] for h in range(H)])
    assert_within(got, want[-1], bound[-1], "absorbed")
    assert_within(out[0, -1], want[-1], bound[-1], "expanded")
