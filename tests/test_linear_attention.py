"""Linear attention with a decay for each head against its recurrence in 64 bits."""
import pytest
import torch

import flashkda_b200
from attention_testlib import check_linear, linear_inputs
from flashkda_b200 import _lib

gpu = pytest.mark.gpu
SCALE = 128 ** -0.5


def call(d, scale=SCALE, h0=None, hT=None, **kw):
    flashkda_b200.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], scale, d["out"], h0, hT, d["cu"], **kw)


# ---------------------------------------------------------------------------------------------------------- on the CPU
def cpu_args(**over):
    d = dict(q=torch.zeros(1, 4, 2, 128).bfloat16(), k=torch.zeros(1, 4, 2, 128).bfloat16(), v=torch.zeros(1, 4, 2, 128).bfloat16(),
             g=torch.zeros(1, 4, 2), out=torch.zeros(1, 4, 2, 128).bfloat16())
    d.update(over)
    return d["q"], d["k"], d["v"], d["g"], 1.0, d["out"]


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        flashkda_b200.linear_attention_fwd(*cpu_args())
    with pytest.raises(RuntimeError, match="q must be a torch.Tensor"):
        flashkda_b200.linear_attention_fwd(*cpu_args(q=None))


def params(**over):
    fake = dict.fromkeys(("q", "k", "v", "g", "out"), 0x1000)
    stride = (4 * 256, 256, 128)
    p = dict(B=1, T=4, H=2, Hk=2, N=1, q_stride=stride, k_stride=stride, v_stride=stride, out_stride=stride, g_stride=(8, 2, 1), scale=1.0, **fake)
    p.update(over)
    return _lib.LinearParams(**p)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), 1), (dict(g=None), 1), (dict(B=0), 2), (dict(T=-1), 2), (dict(H=3), 2), (dict(Hk=0), 2), (dict(H=70000, Hk=1), 2), (dict(N=2), 2),
    (dict(T=2 ** 31), 2), (dict(state_dtype=2), 3), (dict(B=2, N=3, cu_seqlens=0x1000), 4), (dict(q=0x1008), 8), (dict(out=0x1002), 8),
    (dict(initial_state=0x1008), 8), (dict(q_stride=(1024, 252, 128)), 8), (dict(k_stride=(1024, 256, 0)), 8), (dict(v_stride=(1024, -256, 128)), 8),
    (dict(out_stride=(1024, 256, 4)), 8)])
def test_refusals_of_the_c_entry(over, status):
    assert _lib.lib().fkda_linear_attention_fwd(params(**over), None) == status


def test_nothing_to_do_launches_nothing():
    L = _lib.lib()
    assert L.fkda_linear_attention_fwd(None, None) == 1
    assert L.fkda_linear_attention_fwd(params(T=0), None) == 0 and L.fkda_last_launch_count() == 0


@pytest.mark.parametrize("B,T,H,N,packed", [(1, 0, 1, 1, False), (1, 0, 1, 3, True), (3, 0, 2, 3, False), (1, 1, 1, 1, False), (1, 1, 200, 1, False), (1, 10 ** 9, 1, 1, False),
                                            (1, 10 ** 9, 1, 64, True), (64, 10 ** 6, 2, 64, False), (1, 5, 2, 10, True)])
def test_workspace_size_of_any_call(B, T, H, N, packed):
    size = flashkda_b200.linear_attention_workspace_size(B, T, H, N, packed)
    rows = 148 + 2 * N     # segments that all SMs together walk, and the packed sequences' last ones
    assert 0 <= size <= rows * H * (128 * 128 + 1) * 4
    if T < 64 * 10:
        assert size == 0


def test_workspace_size_of_a_latent_step():
    assert flashkda_b200.latent_decode_workspace_size(0, 1, 4) == 0
    for B, Tq, H in ((1, 1, 1), (3, 4, 128), (36864, 1, 64)):
        tiles = -(-Tq * H // 64)
        size = flashkda_b200.latent_decode_workspace_size(B, Tq, H)
        assert size % 4 == 0 and size <= max(148, tiles) * 2 * 64 * 513 * 4 + 16 * B


# ---------------------------------------------------------------------------------------------------------- on the GPU
@gpu
@pytest.mark.parametrize("T", [1, 2, 15, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("state", ["none", "fp32", "bf16"])
def test_lengths_and_states(T, state):
    d = linear_inputs([T, T], 3, seed=T)
    kind = torch.float32 if state != "bf16" else torch.bfloat16
    d["h0"] = d["h0"].to(kind)
    hT = torch.full((2, 3, 128, 128), 9.0, device="cuda", dtype=kind)
    call(d, h0=None if state == "none" else d["h0"], hT=hT)
    check_linear(d, [T, T], SCALE, d["out"], hT, state != "none")
    assert flashkda_b200.operator_status() == 0


@gpu
@pytest.mark.parametrize("H,Hk", [(4, 1), (6, 3), (5, 5)])
@pytest.mark.parametrize("decay", ["token", "head"])
def test_shared_heads_and_constant_decays(H, Hk, decay):
    d = linear_inputs([97], H, Hk, seed=H, decay=decay)
    hT = torch.zeros(1, H, 128, 128, device="cuda")
    call(d, hT=hT)
    check_linear(d, [97], SCALE, d["out"], hT, False)


@gpu
@pytest.mark.parametrize("lens", [[1, 1, 1], [1, 2, 1, 1], [0, 5, 0, 64], [70, 1, 130, 3, 64], [0, 0], [1, 0, 1, 1]], ids=str)
def test_packed_sequences(lens):
    d = linear_inputs(lens, 2, seed=3, packed=True)
    extra = 3      # rows behind the last sequence stay as they were
    grow = lambda x: torch.cat([x, torch.full_like(x[:, :1].expand(-1, extra, *x.shape[2:]) if x.shape[1] else x.new_zeros(1, extra, *x.shape[2:]), float("nan"))], 1)
    T = sum(lens)
    for name in ("q", "k", "v", "g"):
        d[name] = grow(d[name])
    d["out"] = torch.full((1, T + extra, 2, 128), 7.0, device="cuda").bfloat16()
    hT = torch.zeros(len(lens), 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    check_linear(d, lens, SCALE, d["out"], hT)
    assert bool((d["out"][:, T:] == 7.0).all())


@gpu
@pytest.mark.parametrize("strong", [1e-4, 8.0, 60.0])
def test_weak_and_strong_decays(strong):
    d = linear_inputs([190], 2, seed=5, strong=strong)
    hT = torch.zeros(1, 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    check_linear(d, [190], SCALE, d["out"], hT)


@gpu
@pytest.mark.parametrize("T", [1, 100])
def test_minus_infinity_starts_afresh(T):
    d = linear_inputs([T], 2, seed=6)
    d["g"][:, T // 2] = float("-inf")
    d["g"][:, 0] = -1e30
    hT = torch.zeros(1, 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    check_linear(d, [T], SCALE, d["out"], hT)


@gpu
@pytest.mark.parametrize("T", [1, 77])
def test_views_of_wider_tensors(T):
    """q, k, v as slices of one projection, heads in front of tokens in out, decays as a column of a wider tensor."""
    H = 3
    wide = torch.randn(2, T, 3 * H * 128 + 8, device="cuda").bfloat16()
    q, k, v = (wide[..., 8 + i * H * 128:8 + (i + 1) * H * 128].unflatten(-1, (H, 128)) for i in range(3))
    g = -torch.rand(2, H, T, 2, device="cuda")[..., 1].transpose(1, 2)
    out = torch.full((2, H, T, 128), 7.0, device="cuda").bfloat16().transpose(1, 2)
    d = dict(q=q, k=k, v=v, g=g, cu=None, out=out)
    hT = torch.zeros(2, H, 128, 128, device="cuda")
    call(d, 0.01, hT=hT)
    check_linear(d, [T, T], 0.01, out, hT, False)


@gpu
@pytest.mark.parametrize("T", [1, 70])
def test_state_in_place_and_continued(T):
    """Two calls with the state handed over in one buffer are the call on both stretches."""
    d = linear_inputs([2 * T], 2, seed=8)
    state = d["h0"].clone()
    for part in (slice(0, T), slice(T, 2 * T)):
        flashkda_b200.linear_attention_fwd(*(d[x][:, part] for x in "qkvg"), SCALE, d["out"][:, part], state, state)
    hT = torch.zeros_like(state)
    whole = d["out"].clone()
    check_linear(d, [2 * T], SCALE, d["out"], state)
    d["out"] = whole
    call(d, h0=d["h0"], hT=hT)
    check_linear(d, [2 * T], SCALE, d["out"], hT)


SEGMENTED = [([770], "fp32"), ([705], "none"), ([1000, 1000], "bf16"), ([700, 1, 90, 0, 1450], "fp32"), ([2, 2300, 64], "none")]


@gpu
@pytest.mark.parametrize("lens,state", SEGMENTED, ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_few_long_chains_in_segments(lens, state, in_place):
    packed = len(set(lens)) > 1
    d = linear_inputs(lens, 2, 1, seed=14, packed=packed, strong=0.1)
    d["h0"] = d["h0"].to(torch.bfloat16 if state == "bf16" else torch.float32)
    T = sum(lens) if packed else lens[0]
    size = flashkda_b200.linear_attention_workspace_size(1 if packed else len(lens), T, 2, len(lens), packed)
    assert size > 0
    state0 = d["h0"].clone() if state != "none" else None
    hT = state0 if in_place and state0 is not None else torch.full_like(d["h0"], 9.0)
    call(d, h0=state0, hT=hT, workspace=torch.full((size,), 255, dtype=torch.uint8, device="cuda"))
    assert flashkda_b200.last_launch_count() == 3
    check_linear(d, lens, SCALE, d["out"], hT, state != "none")
    # without a final state, and in scratch of the call's own
    want = d["out"].clone()
    d["out"].zero_()
    call(d, h0=d["h0"] if state != "none" else None)
    assert torch.equal(d["out"], want)


@gpu
def test_segments_captured_and_replayed_with_other_lengths():
    lens = [700, 1, 90, 0, 1450]
    d = linear_inputs(lens, 2, seed=15, packed=True)
    ws = torch.empty(flashkda_b200.linear_attention_workspace_size(1, sum(lens), 2, 5, True), dtype=torch.uint8, device="cuda")
    hT = torch.zeros(5, 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, h0=d["h0"], hT=hT, workspace=ws)
    other = [3, 1200, 64, 300, 674]
    d["cu"].copy_(torch.tensor([0] + other).cumsum(0))
    d["out"].fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    check_linear(d, other, SCALE, d["out"], hT)
    with pytest.raises(RuntimeError, match="workspace must be"):
        call(d, h0=d["h0"], hT=hT, workspace=ws[:-1])
    with pytest.raises(RuntimeError, match="workspace missing, misaligned"):
        call(d, h0=d["h0"], hT=hT, workspace=torch.empty(ws.numel() + 64, dtype=torch.uint8, device="cuda")[16:])


@gpu
def test_nothing_of_a_neighbour_or_of_padding_is_used():
    """A sequence between two that hold NaN and infinities."""
    lens = [70, 75, 66]
    d = linear_inputs(lens, 2, seed=9, packed=True)
    for name in ("q", "k", "v", "g"):
        d[name][:, :70] = float("nan")
        d[name][:, 145:] = float("inf")
    hT = torch.zeros(3, 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    e = {x: d[x][:, 70:145] for x in "qkvg"} | dict(cu=None, out=d["out"][:, 70:145], h0=d["h0"][1:2])
    check_linear(e, [75], SCALE, e["out"], hT[1:2])


@gpu
@pytest.mark.parametrize("T", [1, 333])
def test_runs_repeat_bit_for_bit_on_two_streams_at_once(T):
    d = linear_inputs([T] * 3, 4, seed=10)
    hT = torch.zeros(3, 4, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            o, h = torch.zeros_like(d["out"]), torch.zeros_like(hT)
            for _ in range(20):
                flashkda_b200.linear_attention_fwd(d["q"], d["k"], d["v"], d["g"], SCALE, o, d["h0"], h)
            outs.append((o, h))
    torch.cuda.synchronize()
    for o, h in outs:
        assert torch.equal(o, d["out"]) and torch.equal(h, hT)


@gpu
def test_many_long_chains_back_to_back():
    """More chains than SMs, calls behind one another without a pause: no stage of a chunk may be passed twice by another."""
    d = linear_inputs([2000, 900, 1, 63, 1500, 700], 48, 12, seed=13, packed=True)
    hT = torch.zeros(6, 48, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    want, state = d["out"].clone(), hT.clone()
    for _ in range(30):
        call(d, h0=d["h0"], hT=hT)
    assert flashkda_b200.operator_status() == 0
    assert torch.equal(d["out"], want) and torch.equal(hT, state)


@gpu
@pytest.mark.parametrize("lens", [[1, 1], [150, 150], [1, 90, 1]], ids=str)
def test_captured_and_replayed(lens):
    packed = len(set(lens)) > 1
    d = linear_inputs(lens, 2, seed=11, packed=packed)
    hT = torch.zeros(len(lens), 2, 128, 128, device="cuda")
    call(d, h0=d["h0"], hT=hT)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, h0=d["h0"], hT=hT)
    fresh = linear_inputs(lens, 2, seed=12, packed=packed)
    for x in ("q", "k", "v", "g", "h0"):
        d[x].copy_(fresh[x])
    d["out"].zero_(), hT.zero_()
    graph.replay()
    torch.cuda.synchronize()
    check_linear(d, lens, SCALE, d["out"], hT)


@gpu
@pytest.mark.parametrize("change,match", [
    (dict(q=lambda x: x.float()), "q must be bfloat16"), (dict(g=lambda x: x.bfloat16()), "g must be float32"), (dict(k=lambda x: x[:, :3]), "k must be"),
    (dict(out=lambda x: x.cpu()), "out must be on CUDA"), (dict(v=lambda x: x.transpose(1, 3)), "v must be"), (dict(g=lambda x: x[0]), "g must be"),
    (dict(q=lambda x: torch.empty(1, 4, 2, 256, device="cuda").bfloat16()[..., ::2]), "contiguous in its last dimension"),
    (dict(q=lambda x: torch.empty(1, 4, 2, 130, device="cuda").bfloat16()[..., :128]), "16-byte aligned"),
    (dict(k=lambda x: torch.empty(1, 4, 257, device="cuda").bfloat16()[..., 1:].unflatten(-1, (2, 128))), "16-byte aligned"),
    (dict(k=lambda x: x[:, :1].expand(-1, 4, -1, -1)), "16-byte aligned"),
    (dict(h0=lambda x: x.half()), "initial_state must be bfloat16 or float32"), (dict(h0=lambda x: x[:, :1]), "initial_state must be"),
    (dict(h0=lambda x: x.bfloat16()), "must have the same dtype"), (dict(cu=lambda x: torch.tensor([0, 4], device="cuda").int()), "cu_seqlens must be int64"),
    (dict(cu=lambda x: torch.tensor([0], device="cuda")), "at least 2 elements"), (dict(q=lambda x: x[:, :, :0], k=lambda x: x[:, :, :0]), "must divide"),
])
def test_refusals(change, match):
    d = linear_inputs([4], 2)
    hT = torch.zeros(1, 2, 128, 128, device="cuda")
    for name, f in change.items():
        d[name] = f(d[name])
    with pytest.raises(RuntimeError, match=match):
        call(d, h0=d["h0"], hT=hT)
    torch.cuda.synchronize()
