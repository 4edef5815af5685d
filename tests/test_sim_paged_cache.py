"""The operators around the paged cache end to end on the host lane simulator: ``paged_attention_fp8``, ``paged_append`` and
``norm_rotary`` with all of their host logic, CPU tensors, and the kernel sources compiled for the simulator."""
import contextlib

import pytest
import torch

import flag_attn
from flagattention_amd import _lib, paged_fp8
from oracle import paged_attention as oracle_paged
from tests import paged_cache_cases as cases
from tests.sim import simlib

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def simulator_behind_the_public_api(monkeypatch):
    lib = simlib.get()
    monkeypatch.setattr(_lib, "get", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(paged_fp8, "_num_cus", lambda *_: 3)   # workgroups of the balanced launch: few, and each has more
    return lib


# ------------------------------------------------------------------------------------------------ attention ----
@pytest.mark.parametrize("dtype,lens,Hq,Hkv,D,block", [
    (BF16, [1, 0, 70], 4, 2, 128, 16),          # a single key, no keys, a step and a few
    (FP16, [129, 64, 5], 5, 1, 64, 8),          # odd group; a step to the key
    (FP16, [33, 17], 20, 1, 32, 24),            # two blocks of query rows; blocks of eight that are no power of two
    (BF16, [40, 3], 2, 2, 16, 12),              # blocks that a lane's eight keys cross
    (FP16, [21], 3, 1, 256, 5),
    (BF16, [37, 64], 2, 1, 512, 32),
])
def test_attention_over_codes(dtype, lens, Hq, Hkv, D, block):
    args = cases.attention_inputs(dtype, lens, Hq, Hkv, D, block, seed=11, table_type=torch.int64 if D == 64 else torch.int32)
    cases.check_attention(args, flag_attn.paged_attention_fp8(*args))


def test_attention_cut_over_workgroups_and_one_workgroup_per_pair(simulator_behind_the_public_api):
    """Few workgroups for the keys: pairs are cut, a workgroup has the end of one and the beginning of others."""
    from flagattention_amd import _abi
    lib = simulator_behind_the_public_api
    args = cases.attention_inputs(FP16, [700, 0, 260, 1, 513], 6, 3, 64, 16, seed=12, powers=False)
    q, *rest, longest = args
    for wgs in (0, 3, 16):
        out = torch.full_like(q, torch.nan)
        ws = torch.empty(lib.paged_attn_e4m3_workspace(max(1, wgs), 64) // 4) if wgs else None
        _abi.paged_attn_e4m3(lib, out, q, *rest, ws, wgs)
        cases.check_attention(args, out, f"{wgs} workgroups")


def test_keys_behind_the_context_are_not_seen():
    """Whatever the rest of a block and the blocks behind hold, NaN codes too."""
    for block in (16, 12):
        args = list(cases.attention_inputs(BF16, [21, 40], 4, 2, 64, block, seed=13))
        clean = flag_attn.paged_attention_fp8(*args)
        seen = torch.zeros(args[1].shape[0], block, dtype=torch.bool)
        for s, n in enumerate([21, 40]):
            for t in range(n):
                seen[args[6][s, t // block].long(), t % block] = True
        for c in (1, 2):
            codes = args[c].view(torch.uint8).clone()
            codes.permute(0, 2, 1, 3)[~seen] = 0x7F
            args[c] = codes.view(torch.float8_e4m3fn)
        for s in (3, 4):
            args[s] = torch.where(seen.any(1, keepdim=True), args[s], torch.nan)
        assert torch.equal(clean, flag_attn.paged_attention_fp8(*args)) and clean.isfinite().all()


@pytest.mark.parametrize("block", [16, 12])
def test_attention_reads_nothing_for_entries_outside_the_cache(block):
    args = list(cases.attention_inputs(FP16, [50, 30, 70, 9], 4, 2, 64, block, seed=14, table_type=torch.int64))
    args[6][1, 1] = args[1].shape[0]            # a block too far
    args[6][0, 0] = -1
    args[6][3, 4] = 2 ** 40                     # behind its context: not looked at
    args[5][2] = block * args[6].shape[1] + 1   # longer than the table
    out = flag_attn.paged_attention_fp8(*args)
    assert out[:3].isnan().all() and out[3].isfinite().all()
    cases.check_attention(args, out)


@pytest.mark.parametrize("block", [16, 12])
def test_lengths_far_past_the_table_end_soon(simulator_behind_the_public_api, block):
    from flagattention_amd import _abi
    lib = simulator_behind_the_public_api
    args = list(cases.attention_inputs(BF16, [50, 30, 70], 4, 2, 64, block, seed=19))
    args[5][0], args[5][2] = 2 ** 31 - 1, 2 ** 31 - 40
    q, *rest, longest = args
    for wgs in (0, 3, 40):   # a workgroup per pair, a range per wavefront, a piece per workgroup
        out = torch.zeros_like(q)
        ws = torch.empty(lib.paged_attn_e4m3_workspace(max(1, wgs), 64) // 4) if wgs else None
        _abi.paged_attn_e4m3(lib, out, q, *rest, ws, wgs)
        assert out[0].isnan().all() and out[2].isnan().all() and out[1].isfinite().all(), wgs


def test_nan_and_infinities_that_a_row_sees_make_it_nan():
    args = list(cases.attention_inputs(BF16, [40, 40, 40, 40], 4, 2, 64, 16, seed=15))
    args[0][0, 1, 3] = torch.nan
    args[0][1, 2, 0] = torch.inf
    args[1].view(torch.uint8)[args[6][2, 1].long(), 0, 5, 7] = 0x7F
    args[2].view(torch.uint8)[args[6][3, 0].long(), 1, 0, 9] = 0xFF
    out = flag_attn.paged_attention_fp8(*args)
    assert out[0, 1].isnan().all() and out[0, 0].isfinite().all() and out[1, 2].isnan().all() and out[1, 3].isfinite().all()
    assert out[2, :2].isnan().all() and out[2, 2:].isfinite().all() and out[3, 2:, 9].isnan().all() and out[3, :2].isfinite().all()


def test_attention_with_other_strides():
    q, kc, vc, ks, vs, lens, table, scale, longest = cases.attention_inputs(FP16, [37, 18], 4, 2, 64, 16, seed=16)
    want = flag_attn.paged_attention_fp8(q, kc, vc, ks, vs, lens, table, scale, longest)
    both = torch.stack([kc.view(torch.uint8), vc.view(torch.uint8)], 1).permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
    k2, v2 = (both[:, i].view(torch.float8_e4m3fn) for i in (0, 1))        # token before head, keys beside values
    scales = torch.stack([ks, vs], 1)
    wide = torch.zeros(2, 7, 64, dtype=q.dtype)
    wide[:, 1:5] = q
    odd = torch.zeros(2, 4, 65, dtype=q.dtype)
    odd[..., 1:] = q                                                       # rows that the kernel cannot load as they are
    for query in (wide[:, 1:5], odd[..., 1:]):
        out = flag_attn.paged_attention_fp8(query, k2, v2, scales[:, 0], scales[:, 1], lens.long(), table.t().contiguous().t(), scale, longest)
        assert torch.equal(out, want)


def test_attention_refuses():
    good = cases.attention_inputs(FP16, [20, 9], 4, 2, 64, 16, seed=17)
    q, kc, vc, ks, vs, lens, table, scale, longest = good
    bad = {
        "float32 query": (0, q.float()), "16-bit cache": (1, kc.half()), "other value type": (2, vc.half()), "other shape": (2, vc[1:]),
        "double scales": (3, ks.double()), "scales of another shape": (4, vs[:, :1]), "float lengths": (5, lens.float()),
        "lengths of another number": (5, lens[:1]), "16-bit table": (6, table.short()), "table of another number": (6, table[:1]),
        "rows that are not aligned": (1, torch.zeros(kc.shape[:3] + (72,), dtype=torch.uint8).view(kc.dtype)[..., :64]),
        "heads that do not divide": (0, q[:, :3]), "head size": (0, q[..., :48]),
    }
    for what, (i, value) in bad.items():
        args = list(good)
        args[i] = value
        with pytest.raises(AssertionError):
            flag_attn.paged_attention_fp8(*args)
            pytest.fail(what)
    with pytest.raises(AssertionError):
        flag_attn.paged_attention_fp8(q, kc, vc, ks, vs.t().contiguous().t(), lens, table, scale, longest)


def test_attention_with_nothing_to_attend_to():
    q, kc, vc, ks, vs, lens, table, scale, longest = cases.attention_inputs(FP16, [20, 9], 4, 2, 64, 16, seed=18)
    assert flag_attn.paged_attention_fp8(q[:0], kc, vc, ks, vs, lens[:0], table[:0], scale, 0).shape == (0, 4, 64)
    assert (flag_attn.paged_attention_fp8(q, kc, vc, ks, vs, torch.zeros_like(lens), table, scale, 0) == 0).all()
    assert (flag_attn.paged_attention_fp8(q, kc, vc, ks, vs, lens, table[:, :0], scale, 20) == 0).all()
    assert (flag_attn.paged_attention_fp8(q, kc[:0], vc[:0], ks[:0], vs[:0], lens, table, scale, 20) == 0).all()


# --------------------------------------------------------------------------------------------------- append ----
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype,olds,news,Hkv,D,block,size,interleaved,pad", [
    (BF16, [0, 5, 16, 31], [1, 1, 1, 1], 2, 128, 16, 128, False, 0),          # single tokens: fresh and partial blocks
    (FP16, [0, 3, 20], [37, 1, 9], 3, 64, 8, 32, True, 5),                    # over block borders, rows behind the last
    (BF16, [7, 0, 11], [0, 25, 2], 1, 16, 12, 16, False, 0),                  # a sequence without new tokens; odd blocks
    (FP16, [1], [70], 2, 32, 64, 0, False, 0),                                # no rotation, two passes over a block
    (BF16, [3, 2], [6, 4], 1, 256, 5, 128, True, 0),
    (FP16, [0], [11], 1, 512, 16, 512, False, 0),
])
def test_append(bits, dtype, olds, news, Hkv, D, block, size, interleaved, pad):
    args = cases.append_inputs(dtype, bits, olds, news, Hkv, D, block, size, 21, pad=pad, interleaved=interleaved,
                               ragged=pad > 0 or any(n != 1 for n in news))
    cases.check_append(args)


def test_append_by_wavefronts():
    """So many blocks that each of a head has one wavefront; blocks that hold tokens, and rows that fill two of them."""
    olds, news = [(7 * i) % 9 for i in range(120)], [1 + (5 * i) % 5 * (i % 8 == 0) * 4 for i in range(120)]
    args = cases.append_inputs(BF16, 8, olds, news, 5, 128, 12, 128, 28, pad=3)
    args["key_scales"][::2] = args["value_scales"][::2] = 2.0 ** -9
    cases.check_append(args)


@pytest.mark.parametrize("bits", [8, 16])
def test_append_past_many_empty_sequences(bits):
    news = [3, 1, 1] + [0] * 37 + [2] + [0] * 5 + [1, 0, 9, 0, 0]
    cases.check_append(cases.append_inputs(FP16, bits, [(3 * i) % 7 for i in range(len(news))], news, 1, 64, 8, 32, 29, pad=4))


def test_append_makes_room_for_larger_values():
    """Values far above what the block holds: the scale grows, what is there is rounded again, to zero where it falls short."""
    for values in (1e-3, 40.0, 3e4):
        args = cases.append_inputs(FP16 if values < 1e4 else BF16, 8, [9, 3], [1, 4], 2, 64, 16, 64, 22, values=values)
        args["key_scales"][0] = args["value_scales"][0] = 0.0117      # a scale that is no power of two
        cases.check_append(args)


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_without_a_place_are_not_stored(bits):
    args = cases.append_inputs(FP16, bits, [4, 20, 0, 6, 9], [3, 5, 7, 2, 4], 2, 64, 8, 64, 23)
    args["context_lens"][0] = 0                                  # a padding sequence
    args["context_lens"][2] = 3                                  # fewer tokens than rows: the last three
    args["block_tables"][1, 2] = args["key_cache"].shape[0]      # no such block: tokens 16 to 23
    args["block_tables"][3, 0] = -1
    args["cos"], args["sin"] = args["cos"][:11], args["sin"][:11]      # position 11 and on
    args["query_starts"][5] = 40                                 # more rows than there are: the lengths count from there
    args["context_lens"][4] = 30
    cases.check_append(args)
    args["context_lens"][4] = 500                                # behind the table
    cases.check_append(args)


def test_values_that_are_not_finite_become_nan_and_leave_the_scale():
    args = cases.append_inputs(BF16, 8, [2, 0], [3, 2], 2, 64, 8, 0, 24)
    args["value"][0, 0, 3], args["value"][1, 1, 5], args["key"][3, 0, 0] = torch.inf, torch.nan, -torch.inf
    args["key"][4] = torch.nan
    args["value"][3:] = 0                                        # nothing but zeros
    cases.check_append(args)


def test_append_with_other_strides_and_types():
    args = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 25)
    want = cases.check_append(args)
    a = cases.copied(args)
    rows = torch.zeros(11, 6, 64, dtype=FP16)                    # keys and values in one projection
    rows[:, :2], rows[:, 3:5] = a["key"], a["value"]
    a["key"], a["value"] = rows[:, :2], rows[:, 3:5]
    caches = torch.stack([a["key_cache"].view(torch.uint8), a["value_cache"].view(torch.uint8)], 3).contiguous()
    a["key_cache"], a["value_cache"] = (caches[:, :, :, i].view(torch.float8_e4m3fn) for i in (0, 1))
    scales = torch.stack([a["key_scales"], a["value_scales"]])
    a["key_scales"], a["value_scales"] = scales
    a["cos"], a["sin"] = (torch.nn.functional.pad(t, (1, 2))[:, 1:-2] for t in (a["cos"], a["sin"]))
    a["context_lens"], a["query_starts"] = a["context_lens"].long(), a["query_starts"].long()
    a["block_tables"] = a["block_tables"].int().t().contiguous().t()
    flag_attn.paged_append(**a)
    for n in ("key_cache", "value_cache", "key_scales", "value_scales"):
        x, y = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a[n].contiguous(), want[n]))
        assert torch.equal(x, y), n


def test_append_refuses():
    good = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 26)
    plain = cases.append_inputs(FP16, 16, [3, 9], [1, 1], 2, 64, 16, 64, 26, ragged=False)
    bad = [
        (good, dict(key=good["key"].float(), value=good["value"].float())), (good, dict(value=good["value"].bfloat16())),
        (good, dict(value=good["value"][1:])), (good, dict(key_scales=None)), (good, dict(key_scales=None, value_scales=None)),
        (good, dict(key_scales=good["key_scales"].double())), (good, dict(key_scales=good["key_scales"][1:])),
        (good, dict(cos=None)), (good, dict(cos=good["cos"].double(), sin=good["sin"].double())), (good, dict(cos=good["cos"][:, :20], sin=good["sin"][:, :20])),
        (good, dict(cos=torch.cat([good["cos"]] * 2, 1), sin=torch.cat([good["sin"]] * 2, 1))),
        (good, dict(query_starts=None)), (good, dict(query_starts=good["query_starts"][1:])), (good, dict(query_starts=good["query_starts"].float())),
        (good, dict(context_lens=good["context_lens"][1:])), (good, dict(block_tables=good["block_tables"].float())),
        (good, dict(value_cache=good["value_cache"][1:])), (good, dict(key=good["key"][:, :1], value=good["value"][:, :1])),
        (plain, dict(key_cache=plain["key_cache"].bfloat16(), value_cache=plain["value_cache"].bfloat16())),
        (plain, dict(key_scales=good["key_scales"], value_scales=good["value_scales"])),
        (plain, dict(key=plain["key"][:1], value=plain["value"][:1])),
        (plain, dict(key_cache=torch.zeros(6, 2, 16, 65, dtype=FP16)[..., :64], value_cache=torch.zeros(6, 2, 16, 65, dtype=FP16)[..., :64])),
    ]
    for args, change in bad:
        a = cases.copied(args)
        before = a["key_cache"].clone()
        with pytest.raises(AssertionError):
            flag_attn.paged_append(**{**a, **change})
            pytest.fail(str(list(change)))
        assert torch.equal(before.view(torch.uint8), a["key_cache"].view(torch.uint8))


def test_append_refuses_what_it_would_write_to_twice():
    good = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 26)
    one = torch.ones(1, 1).expand(*good["key_scales"].shape)
    for change in (dict(value_cache=good["key_cache"]), dict(value_scales=good["key_scales"]),
                   dict(key_scales=one, value_scales=one.clone().expand_as(one)), dict(key_scales=one, value_scales=one * 1),
                   {n: torch.zeros_like(good["key_cache"])[:1].expand_as(good["key_cache"]) for n in ("key_cache", "value_cache")}):
        with pytest.raises(AssertionError):
            flag_attn.paged_append(**{**good, **change})
            pytest.fail(str(list(change)))


def test_append_of_nothing():
    args = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 27)
    for change in (dict(key=args["key"][:0], value=args["value"][:0], query_starts=torch.zeros(3, dtype=torch.int32)),
                   dict(block_tables=args["block_tables"][:, :0]), dict(context_lens=torch.zeros_like(args["context_lens"]))):
        a = cases.copied(args)
        flag_attn.paged_append(**{**a, **change})
        for n in ("key_cache", "value_cache", "key_scales", "value_scales"):
            assert torch.equal(a[n].view(torch.uint8), args[n].view(torch.uint8)), n


# --------------------------------------------------------------------------------------------------- rotary ----
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,B,H,Hk,T,D,size,weight_type,positions,bthd", [
    (BF16, 2, 4, 2, 9, 128, 128, BF16, None, True),
    (FP16, 1, 3, 1, 17, 64, 32, torch.float32, 2, False),       # half of a head turned, odd sizes
    (BF16, 3, 1, 1, 1, 16, 16, torch.float32, 2, True),         # a single token, one lane per row
    (FP16, 2, 2, 2, 70, 32, 16, None, 1, True),                 # no norm
    (BF16, 1, 2, 5, 3, 256, 256, BF16, None, False),            # more key heads than query heads
    (FP16, 1, 1, 2, 5, 512, 64, FP16, None, True),
])
def test_norm_rotary_and_gradients(interleaved, dtype, B, H, Hk, T, D, size, weight_type, positions, bthd):
    args = cases.rotary_inputs(dtype, B, H, Hk, T, D, size, 31, weight_type=weight_type, positions=positions, bthd=bthd, grad=True)
    cases.check_rotary(args, interleaved, grad=True)


def test_single_tokens_are_rows_of_length_one():
    args = cases.rotary_inputs(FP16, 5, 4, 2, 1, 64, 64, 32, weight_type=FP16, positions=2)
    outs = flag_attn.norm_rotary(**args)
    flat = {n: t[:, :, 0] if n in ("q", "k") else t[:, 0] if n == "positions" else t for n, t in args.items()}
    for a, b in zip(outs, flag_attn.norm_rotary(**{**flat, "positions": flat["positions"].int()})):
        assert b.shape == a[:, :, 0].shape and torch.equal(a[:, :, 0], b)


def test_positions_outside_the_tables_turn_by_nan():
    args = cases.rotary_inputs(FP16, 1, 2, 1, 4, 64, 32, 33, positions=2)
    args["positions"] = torch.tensor([[0, -1, 12, 2 ** 40]])
    q, k = flag_attn.norm_rotary(**args)
    for y in (q, k):
        assert y[0, :, 0].isfinite().all() and y[0, :, 1:, :32].isnan().all() and y[0, :, 1:, 32:].isfinite().all()


def test_gradients_of_part_of_the_outputs_and_inputs():
    """An output without a gradient counts as one of zeros; expanded inputs add theirs up."""
    args = cases.rotary_inputs(BF16, 2, 4, 2, 6, 64, 64, 34, weight_type=torch.float32, grad=True)
    q, k = flag_attn.norm_rotary(**args)
    dy = torch.ones_like(q)
    got = torch.autograd.grad(q, [args[n] for n in ("q", "k", "q_weight", "k_weight")], dy)
    assert (got[1] == 0).all() and (got[3] == 0).all() and got[0].abs().max() > 0
    one = torch.randn(2, 1, 6, 64).to(BF16).requires_grad_()
    a, b = (flag_attn.norm_rotary(**{**args, "k": k})[1] for k in (one.expand(2, 3, 6, 64), one.expand(2, 3, 6, 64).contiguous()))
    assert torch.equal(a, b)
    (ga,), (gb,) = (torch.autograd.grad(t, one, torch.ones_like(t)) for t in (a, b))
    assert torch.equal(ga, gb) and ga.shape == one.shape


def test_norm_rotary_is_differentiable_once():
    args = cases.rotary_inputs(BF16, 1, 2, 2, 6, 64, 64, 37, grad=True)
    q, k = flag_attn.norm_rotary(**args)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(q.sum() + k.sum(), args["q"], create_graph=True)


def test_norm_rotary_of_rows_of_zeros_and_of_nothing():
    args = cases.rotary_inputs(BF16, 2, 4, 2, 6, 64, 64, 35, weight_type=torch.float32, grad=True)
    zeros = torch.zeros_like(args["q"]).requires_grad_()
    q, _ = flag_attn.norm_rotary(**{**args, "q": zeros})
    g = torch.autograd.grad(q, (zeros, args["q_weight"]), torch.ones_like(q))
    assert (q == 0).all() and g[0].isfinite().all() and (g[1] == 0).all()
    empty = {**args, "q": args["q"][:0], "k": args["k"][:0]}
    q, k = flag_attn.norm_rotary(**empty)
    assert q.shape == (0, 4, 6, 64) and k.shape == (0, 2, 6, 64)
    assert (torch.autograd.grad(q.sum() + k.sum(), args["q_weight"])[0] == 0).all()


def test_norm_rotary_refuses():
    good = cases.rotary_inputs(BF16, 2, 4, 2, 6, 64, 64, 36, weight_type=BF16, positions=2)
    single = {n: t[:, :, 0] if n in ("q", "k") else t[:, 0] if n == "positions" else t for n, t in good.items()}
    bad = [
        dict(q=good["q"].float(), k=good["k"].float()), dict(k=good["k"].half()), dict(k=good["k"][:, :, :5]), dict(k=good["k"][:1]),
        dict(k=good["k"][..., :32]), dict(q=good["q"][..., :48], k=good["k"][..., :48]), dict(k=good["k"][:, :0]), dict(k=good["k"][:, :, 0]),
        dict(cos=good["cos"].double()), dict(sin=good["sin"][:, :16]), dict(cos=good["cos"][:, :12], sin=good["sin"][:, :12]),
        dict(cos=good["cos"].requires_grad_()), dict(cos=good["cos"][:0], sin=good["sin"][:0]),
        dict(q_weight=None), dict(q_weight=good["q_weight"].double(), k_weight=good["k_weight"].double()), dict(q_weight=good["q_weight"].float()),
        dict(q_weight=good["q_weight"][:32]), dict(eps=0.0), dict(eps=float("nan")), dict(positions=good["positions"].float()),
        dict(positions=good["positions"][:, :5]), dict(positions=None, cos=good["cos"][:5], sin=good["sin"][:5]),
        {**single, "positions": None},
    ]
    good["cos"] = good["cos"].detach()
    for change in bad:
        with pytest.raises(AssertionError):
            flag_attn.norm_rotary(**{**good, **change})
            pytest.fail(str(list(change)))


# ------------------------------------------------------------------------------------- order of the wavefronts ----
def test_results_do_not_depend_on_how_the_wavefronts_advance(monkeypatch, simulator_behind_the_public_api):
    """Bit for bit under every order that the barriers allow: a missing one would show."""
    from flagattention_amd import _abi
    lib = simulator_behind_the_public_api
    attends = [cases.attention_inputs(FP16, [150, 0, 290], 4, 2, D, 16, seed=51) for D in (64, 128)]
    appends = cases.append_inputs(BF16, 8, [3, 20], [25, 4], 2, 64, 16, 64, 52)
    rotaries = cases.rotary_inputs(BF16, 2, 4, 2, 9, 64, 64, 53, weight_type=torch.float32, grad=True)

    def everything():
        got = []
        for q, *rest, longest in attends:
            for wgs in (0, 3, 20):     # one workgroup per pair, ranges of wavefronts, pieces of workgroups
                out = torch.full_like(q, torch.nan)
                ws = torch.empty(lib.paged_attn_e4m3_workspace(max(1, wgs), q.shape[2]) // 4) if wgs else None
                _abi.paged_attn_e4m3(lib, out, q, *rest, ws, wgs)
                got.append(out)
        a = cases.copied(appends)
        flag_attn.paged_append(**a)
        got += [a[n].view(torch.uint8) for n in ("key_cache", "value_cache", "key_scales", "value_scales")]
        outs = flag_attn.norm_rotary(**rotaries)
        got += outs
        got += torch.autograd.grad(outs, [rotaries[n] for n in ("q", "k", "q_weight", "k_weight")], [torch.ones_like(o) for o in outs])
        return got

    want = everything()
    for schedule, seed in (("ahead", "0"), ("ahead_descending", "0"), ("random", "1"), ("random", "2")):
        monkeypatch.setenv("HWSIM_SCHEDULE", schedule)
        monkeypatch.setenv("HWSIM_SEED", seed)
        assert all(torch.equal(a, b) for a, b in zip(want, everything())), (schedule, seed)


# ------------------------------------------------------------------------------------------------- together ----
def test_a_prompt_and_steps_behind_it():
    """Norm and rotation of the queries, rotation of the keys on their way into the cache, attention: into 8 and 16 bits."""
    D, Hq, Hkv, block, seqs = 64, 4, 2, 16, 2
    cos, sin = cases.tables(64, D)
    table = torch.tensor([[3, 1, 0], [5, 2, 4]])
    g = torch.Generator().manual_seed(41)
    new = lambda rows, heads: torch.randn(rows, heads, D, generator=g).to(FP16)   # noqa: E731
    fp8 = [torch.zeros(6, Hkv, block, D).to(torch.float8_e4m3fn) for _ in range(2)] + [torch.zeros(6, Hkv) for _ in range(2)]
    wide = [torch.zeros(6, Hkv, block, D, dtype=FP16) for _ in range(2)]
    lens = torch.tensor([14, 20], dtype=torch.int32)
    k, v = new(34, Hkv), new(34, Hkv)
    starts = torch.tensor([0, 14, 34], dtype=torch.int32)
    for step in range(4):
        for cache in (fp8, wide):
            flag_attn.paged_append(k, v, *cache[:2], lens, table, starts if step == 0 else None, *cache[2:] or (None, None), cos, sin)
        q, _ = flag_attn.norm_rotary(new(seqs, Hq), new(seqs, Hkv), cos, sin, lens - 1, torch.ones(D, dtype=FP16), torch.ones(D, dtype=FP16))
        args = (q, *fp8, lens, table, D ** -0.5, 48)
        out = flag_attn.paged_attention_fp8(*args)
        cases.check_attention(args, out, f"step {step}")
        # the two caches hold the same rotated keys and values, one to 11 bits, one to 4: what attention makes of them is a
        # mean over keys whose values are off by 2^-4 and whose weights by what that does to the scores
        dense = flag_attn.paged_attention(q, *wide, lens, table, D ** -0.5, 48, num_splits=1)
        assert torch.allclose(dense.float(), oracle_paged(q, *wide, table, lens, D ** -0.5).float(), atol=2e-3, rtol=0)
        assert (dense.float() - out.float()).norm() <= 2 ** -3 * dense.float().norm()
        k, v = new(seqs, Hkv), new(seqs, Hkv)
        lens = lens + 1
