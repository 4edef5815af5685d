"""The operators around the paged cache on the GPU: ``paged_attention_fp8``, ``paged_append`` and ``norm_rotary`` against their
64-bit statements, at sizes that fill the device and at those where they can go wrong, on side streams and in graphs."""
import pytest
import torch

import flag_attn
from flagattention_amd import _abi, _lib
from tests import paged_cache_cases as cases

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,lens,Hq,Hkv,D,block", [
    (BF16, [1], 32, 8, 128, 16),
    (FP16, [300, 0, 1, 2049, 64, 65, 511], 32, 8, 128, 16),
    (BF16, [513, 70, 128, 129], 16, 16, 64, 32),
    (FP16, [4097, 9], 20, 1, 64, 8),              # two blocks of query rows
    (BF16, [700, 33, 0], 40, 2, 128, 24),         # blocks of eight that are no power of two
    (FP16, [255, 258], 6, 2, 128, 20),            # blocks that a lane's eight keys cross
    (BF16, [40, 1000], 12, 1, 256, 64),
    (FP16, [333, 5, 1700], 8, 2, 512, 16),
    (FP16, [100, 77], 4, 4, 32, 16),
    (BF16, [100, 77, 2000], 3, 1, 16, 128),
    (BF16, [50], 5, 1, 16, 7),
    (FP16, [31, 500], 2, 1, 512, 3),
])
@pytest.mark.parametrize("powers", [True, False])
def test_attention_over_codes(dtype, lens, Hq, Hkv, D, block, powers):
    args = cases.attention_inputs(dtype, lens, Hq, Hkv, D, block, seed=11, device="cuda", powers=powers,
                                  table_type=torch.int64 if D == 64 else torch.int32)
    cases.check_attention(args, flag_attn.paged_attention_fp8(*args), "balanced")
    q, *rest, _ = args
    out = torch.full_like(q, torch.nan)
    _abi.paged_attn_e4m3(_lib.get(), out, q, *rest, None, 0)
    cases.check_attention(args, out, "one workgroup per pair")


def test_attention_of_many_short_sequences():
    """More pairs than eight to a workgroup: the other launch."""
    lens = [(37 * i) % 90 for i in range(600)]
    args = cases.attention_inputs(BF16, lens, 16, 8, 64, 16, seed=12, device="cuda")
    cases.check_attention(args, flag_attn.paged_attention_fp8(*args))


def test_lengths_far_past_the_table_end_soon():
    for longest, lens in ((100, [50, 30, 70]), (9000, [50, 30, 9000])):
        args = list(cases.attention_inputs(BF16, lens, 4, 2, 64, 16, seed=19, device="cuda"))
        args[5][0], args[5][2] = 2 ** 31 - 1, 2 ** 31 - 40
        out = flag_attn.paged_attention_fp8(*args[:-1], longest)
        assert out[0].isnan().all() and out[2].isnan().all() and out[1].isfinite().all(), longest


def test_append_refuses_what_it_would_write_to_twice():
    good = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 26, device="cuda")
    ones = [torch.ones(1, 1, device="cuda").expand(*good["key_scales"].shape) for _ in range(2)]
    for change in (dict(value_cache=good["key_cache"]), dict(value_scales=good["key_scales"]), dict(key_scales=ones[0], value_scales=ones[1])):
        with pytest.raises(AssertionError):
            flag_attn.paged_append(**{**good, **change})
            pytest.fail(str(list(change)))


def test_norm_rotary_is_differentiable_once():
    args = cases.rotary_inputs(BF16, 1, 2, 2, 6, 64, 64, 37, device="cuda", grad=True)
    q, k = flag_attn.norm_rotary(**args)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(q.sum() + k.sum(), args["q"], create_graph=True)


def test_offsets_past_32_bits():
    """Caches of 5 GiB each, the blocks in use at both ends."""
    blocks, Hkv, block, D = 20480, 8, 256, 128
    q, kc, vc, ks, vs, lens, table, scale, longest = cases.attention_inputs(FP16, [700, 513], 8, Hkv, D, block, seed=13, device="cuda")
    new = torch.randn(2, 2, Hkv, D, generator=cases.generator("cpu", 14)).to(FP16).cuda()
    cos, sin = cases.tables(800, D, "cuda")
    results = []
    for far in (False, True):
        where = torch.arange(kc.shape[0], device="cuda")
        if far:
            where[1::2] = blocks - where[1::2]
        big = [torch.zeros((blocks if far else kc.shape[0],) + t.shape[1:], dtype=torch.uint8, device="cuda") for t in (kc, vc)]
        scales = [torch.zeros(b.shape[0], Hkv, device="cuda") for b in big]
        for b, t, s, u in zip(big, (kc, vc), scales, (ks, vs)):
            b[where] = t.view(torch.uint8)
            s[where] = u
        big = [b.view(torch.float8_e4m3fn) for b in big]
        rows = where[table.long()]
        flag_attn.paged_append(new[0], new[1], *big, lens, rows, None, *scales, cos, sin)
        results.append(flag_attn.paged_attention_fp8(q, *big, *scales, lens, rows, scale, longest))
        results += [b.view(torch.uint8)[where] for b in big] + [s[where] for s in scales]
    for a, b in zip(results[:5], results[5:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype,olds,news,Hkv,D,block,size,interleaved,pad", [
    (BF16, [0, 5, 16, 31, 200, 63], [1] * 6, 8, 128, 16, 128, False, 0),
    (FP16, [0, 3, 20, 0], [137, 1, 9, 64], 3, 64, 8, 32, True, 50),
    (BF16, [7, 0, 11], [0, 250, 2], 1, 16, 12, 16, False, 0),
    (FP16, [1, 30], [70, 300], 2, 32, 256, 0, False, 0),
    (BF16, [3, 2], [60, 4], 2, 256, 5, 128, True, 0),
    (FP16, [0], [110], 1, 512, 16, 512, False, 0),
])
def test_append(bits, dtype, olds, news, Hkv, D, block, size, interleaved, pad):
    args = cases.append_inputs(dtype, bits, olds, news, Hkv, D, block, size, 21, device="cuda", pad=pad, interleaved=interleaved,
                               ragged=any(n != 1 for n in news))
    cases.check_append(args)


@pytest.mark.parametrize("bits", [8, 16])
def test_append_to_many_sequences(bits):
    """More sequences than lanes, some of them with nothing, and rows behind the last."""
    olds, news = [(7 * i) % 40 for i in range(150)], [(5 * i) % 4 for i in range(150)]
    cases.check_append(cases.append_inputs(BF16, bits, olds, news, 2, 64, 16, 64, 22, device="cuda", pad=9))


@pytest.mark.parametrize("bits", [8, 16])
def test_append_past_many_empty_sequences(bits):
    news = [3, 1, 1] + [0] * 700 + [2] + [0] * 50 + [1, 0, 9] + [0] * 300
    cases.check_append(cases.append_inputs(FP16, bits, [(3 * i) % 7 for i in range(len(news))], news, 2, 64, 8, 32, 29, device="cuda", pad=4))


@pytest.mark.parametrize("rotary", [0, 32, 48, 128])
@pytest.mark.parametrize("olds,news,block", [
    ([(7 * i) % 40 for i in range(80)], [(11 * i) % 60 for i in range(80)], 16),     # a wavefront for a block of a head
    ([(7 * i) % 70 for i in range(40)], [70 + (11 * i) % 60 for i in range(40)], 64),   # a workgroup, also of part of a block
    ([5, 63, 64, 0], [1, 2, 9, 17], 64),                                             # a workgroup, also with rows for one wavefront
])
def test_append_to_8_bits_by_wavefronts_and_by_workgroups(olds, news, block, rotary):
    """Blocks that hold tokens already, with larger and with smaller scales than the new ones need."""
    args = cases.append_inputs(BF16, 8, olds, news, 8, 128, block, rotary, 34, device="cuda", pad=7)
    args["key_scales"][::2] = args["value_scales"][::2] = 2.0 ** -9
    cases.check_append(args)


@pytest.mark.parametrize("values", [1e-3, 40.0, 3e4])
def test_append_makes_room_for_larger_values(values):
    args = cases.append_inputs(FP16 if values < 1e4 else BF16, 8, [9, 3, 0], [1, 4, 30], 2, 64, 16, 64, 23, device="cuda", values=values)
    args["key_scales"][0] = args["value_scales"][0] = 0.0117
    cases.check_append(args)


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_without_a_place_are_not_stored(bits):
    args = cases.append_inputs(FP16, bits, [4, 20, 0, 6, 9], [3, 5, 7, 2, 4], 2, 64, 8, 64, 24, device="cuda")
    args["context_lens"][0] = 0
    args["context_lens"][2] = 3
    args["block_tables"][1, 2] = args["key_cache"].shape[0]
    args["block_tables"][3, 0] = -1
    args["cos"], args["sin"] = args["cos"][:11], args["sin"][:11]
    args["query_starts"][5] = 40
    args["context_lens"][4] = 30
    cases.check_append(args)


def test_values_that_are_not_finite_become_nan_and_leave_the_scale():
    args = cases.append_inputs(BF16, 8, [2, 0], [3, 2], 2, 64, 8, 0, 25, device="cuda")
    args["value"][0, 0, 3], args["value"][1, 1, 5], args["key"][3, 0, 0] = torch.inf, torch.nan, -torch.inf
    args["key"][4] = torch.nan
    args["value"][3:] = 0
    cases.check_append(args)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,B,H,Hk,T,D,size,weight_type,positions,bthd", [
    (BF16, 2, 8, 2, 300, 128, 128, BF16, None, True),
    (BF16, 1, 32, 8, 1025, 128, 128, torch.float32, None, True),
    (FP16, 3, 5, 1, 77, 64, 32, torch.float32, 2, False),
    (BF16, 3, 1, 1, 1, 16, 16, torch.float32, 2, True),
    (FP16, 2, 4, 4, 170, 32, 16, None, 1, True),
    (BF16, 1, 2, 5, 33, 256, 256, BF16, None, False),
    (FP16, 1, 3, 2, 40, 512, 64, FP16, None, True),
])
def test_norm_rotary_and_gradients(interleaved, dtype, B, H, Hk, T, D, size, weight_type, positions, bthd):
    args = cases.rotary_inputs(dtype, B, H, Hk, T, D, size, 31, device="cuda", weight_type=weight_type, positions=positions, bthd=bthd,
                               grad=True)
    cases.check_rotary(args, interleaved, grad=True)


def test_gradients_do_not_depend_on_chance():
    args = cases.rotary_inputs(BF16, 2, 16, 4, 1500, 128, 128, 32, device="cuda", weight_type=torch.float32, grad=True)
    leaves = [args[n] for n in ("q", "k", "q_weight", "k_weight")]

    def step():
        outs = flag_attn.norm_rotary(**args)
        return torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def decoder_step(state, D=128):
    """One token of each sequence: norm and rotation, append, attention over 8 bits."""
    q, k = flag_attn.norm_rotary(state["q"], state["k"], state["cos"], state["sin"], state["lens"] - 1, state["wq"], state["wk"])
    flag_attn.paged_append(k, state["v"], state["kc"], state["vc"], state["lens"], state["table"], None, state["ks"], state["vs"])
    return flag_attn.paged_attention_fp8(q, state["kc"], state["vc"], state["ks"], state["vs"], state["lens"], state["table"],
                                         D ** -0.5, 1000)


def decoder_state(seed, lens=(5, 300, 17, 999, 0, 64), D=128, Hq=16, Hkv=4):
    q, kc, vc, ks, vs, lens, table, _, _ = cases.attention_inputs(BF16, list(lens), Hq, Hkv, D, 16, seed=seed, device="cuda")
    g = cases.generator("cpu", seed)
    k, v = (torch.randn(len(lens), Hkv, D, generator=g).to(BF16).cuda() for _ in range(2))
    cos, sin = cases.tables(1000, D, "cuda")
    w = [torch.ones(D, dtype=BF16, device="cuda") * 1.25, torch.ones(D, dtype=BF16, device="cuda") * 0.5]
    return dict(q=q, k=k, v=v, kc=kc, vc=vc, ks=ks, vs=vs, lens=lens, table=table, cos=cos, sin=sin, wq=w[0], wk=w[1])


def test_a_decoder_step_on_a_side_stream_and_from_graphs():
    """Two graphs of the step on caches of their own, replayed in turn with eager steps between the replays."""
    states = [decoder_state(41), decoder_state(42, lens=(1000, 2, 600, 0, 33, 800))]
    start = [{n: t.clone() for n, t in s.items()} for s in states]
    eager = [decoder_step(s) for s in start]
    args = (None, start[0]["kc"], start[0]["vc"], start[0]["ks"], start[0]["vs"], start[0]["lens"], start[0]["table"], 128 ** -0.5, 1000)
    q, _ = flag_attn.norm_rotary(start[0]["q"], start[0]["k"], start[0]["cos"], start[0]["sin"], start[0]["lens"] - 1, start[0]["wq"], start[0]["wk"])
    cases.check_attention((q,) + args[1:], eager[0])
    torch.cuda.synchronize()
    side, graphs, outs = torch.cuda.Stream(), [], []
    with torch.cuda.stream(side):
        for s, want in zip(states, eager):
            c = {n: t.clone() for n, t in s.items()}
            got = decoder_step(c)
            side.synchronize()
            assert torch.equal(got, want)
    torch.cuda.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decoder_step(s))
        graphs.append(g)
    for turn in range(3):
        for s in states:
            s["lens"] += (s["lens"] > 0).int() * (turn > 0)
            s["q"].copy_(torch.randn(s["q"].shape, generator=cases.generator("cpu", turn)).to(BF16))
            s["lens"].clamp_(max=s["table"].shape[1] * 16)
        copies = [{n: t.clone() for n, t in s.items()} for s in states]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        eager = [decoder_step(c) for c in copies]
        torch.cuda.synchronize()
        for s, c, a, b in zip(states, copies, outs, eager):
            # (bits: the longest sequence outgrows the rotation's tables, and its rows turn to NaN in both)
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), turn
            for n in ("kc", "vc"):
                assert torch.equal(s[n].view(torch.uint8), c[n].view(torch.uint8)), (turn, n)
            assert torch.equal(s["ks"], c["ks"]) and torch.equal(s["vs"], c["vs"]), turn


def test_gradients_from_a_graph():
    args = cases.rotary_inputs(BF16, 1, 8, 2, 200, 64, 64, 51, device="cuda", weight_type=torch.float32, grad=True)
    leaves = [args[n] for n in ("q", "k", "q_weight", "k_weight")]
    dy = [torch.randn_like(args[n]) for n in ("q", "k")]

    def step():
        return torch.autograd.grad(flag_attn.norm_rotary(**args), leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            args["q"].copy_(torch.randn(args["q"].shape, generator=cases.generator("cpu", seed)).to(BF16))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed


def test_a_capture_is_refused_while_an_eager_graph_holds_its_leaves():
    """Refused before anything is recorded: the backward would reach autograd nodes of the eager graph's stream."""
    args = cases.rotary_inputs(BF16, 1, 4, 2, 20, 64, 64, 52, device="cuda", weight_type=torch.float32, grad=True)
    alive = flag_attn.norm_rotary(**args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(g):
            torch.zeros(1, device="cuda")
            flag_attn.norm_rotary(**args)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():
        quiet = flag_attn.norm_rotary(**args)
    assert len(alive) == len(quiet) == 2
    torch.cuda.synchronize()


def test_training_through_flash_attention():
    """Projections, norm and rotation, attention: the gradients of what is in front of the rotation and of its weights."""
    B, H, Hk, T, D = 1, 8, 2, 256, 128
    g = cases.generator("cpu", 61)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(BF16).cuda().transpose(1, 2).requires_grad_() for h in (H, Hk, Hk))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).cuda().requires_grad_() for _ in range(2)]
    cos, sin = cases.tables(T, D, "cuda")
    do = torch.randn(B, H, T, D, generator=g).to(BF16).cuda()
    out = flag_attn.flash_attention(*flag_attn.norm_rotary(q, k, cos, sin, q_weight=w[0], k_weight=w[1]), v, causal=True)
    got = torch.autograd.grad(out, (q, k, v, *w), do)
    from oracle import rotary
    leaves = [t.detach().cpu().double().requires_grad_() for t in (q, k, v, *w)]
    a, b = (rotary.norm_rotary(x, cos.cpu(), sin.cpu(), torch.arange(T)[None], u, 1e-6, False) for x, u in ((leaves[0], leaves[3]), (leaves[1], leaves[4])))
    s = a @ b.repeat_interleave(H // Hk, 1).transpose(2, 3) * D ** -0.5
    s = s.masked_fill(~torch.ones(T, T, dtype=torch.bool).tril(), -torch.inf)
    want = torch.autograd.grad(s.softmax(-1) @ leaves[2].repeat_interleave(H // Hk, 1), leaves, do.cpu().double())
    # bf16 operands of every product: a handful of roundings of 2^-8 behind one another
    for x, y in zip(got, want):
        assert (x.cpu().double() - y).norm() <= 6 * 2.0 ** -8 * y.norm()
