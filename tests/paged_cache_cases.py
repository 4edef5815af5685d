"""Inputs and bounds shared by the simulator's and the GPU's tests of the operators around the paged cache.

Bounds count roundings: a rounding to type t is off by at most finfo(t).eps / 2 relative to the value (e4m3 below its normal
range: half a step of 2^-9), an fp32 operation by 2^-24.  Products of 16-bit numbers and of e4m3 numbers are exact in fp32.
"""
import torch

import flag_attn
from oracle import paged_cache, rotary

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def generator(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def tables(positions, size, device="cpu"):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** -(torch.arange(0, size, 2, dtype=torch.float64) / size)
    return angle.cos().float().to(device), angle.sin().float().to(device)


# ------------------------------------------------------------------------------------------------ attention ----
def fp8_cache(shape, seed, device, powers=True):
    """Codes of normal values and scales (num_blocks, heads)."""
    g = generator("cpu", seed)
    codes = (torch.randn(shape, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-8, -4, shape[:2], generator=g).float()) if powers else torch.rand(shape[:2], generator=g) / 40 + 1e-3
    return codes.to(device), scales.to(device)


def attention_inputs(dtype, lens, Hq, Hkv, D, block, seed, device="cpu", spare=3, powers=True, table_type=torch.int32):
    g = generator("cpu", seed)
    columns = max(1, -(-max(lens) // block))
    num_blocks = len(lens) * columns + spare
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(device)
    (kc, ks), (vc, vs) = (fp8_cache((num_blocks, Hkv, block, D), seed + i, device, powers) for i in (1, 2))
    table = torch.randperm(num_blocks, generator=g)[:len(lens) * columns].reshape(len(lens), columns).to(table_type).to(device)
    return q, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=device), table, D ** -0.5, max(lens)


def check_attention(args, out, name=""):
    """The result rounds once; every probability times its scale has been rounded to bf16 (to two bf16 for fp16 queries) and
    carries the error of its score: (D + 8) fp32 operations on at most `reach`, twice (the row sum has it too); the sums over
    the keys are fp32, one step of 32 to 64 keys after another and four partial sums."""
    q, kc, vc, ks, vs, lens, table, scale, longest = args
    ref, spread, reach = paged_cache.attention_fp8(q, kc, vc, ks, vs, lens, table, scale)
    D, out = q.shape[2], out.detach().cpu()
    assert out.dtype == q.dtype and out.shape == q.shape
    held = half_step(torch.bfloat16) if q.dtype == torch.bfloat16 else half_step(torch.bfloat16) ** 2
    bound = half_step(q.dtype) * ref.abs() * 1.01 + \
        (held + 2 * (D + 8) * U32 * reach + 2.0 ** -20 + (longest / 16 + 16) * U32) * spread + 2.0 ** -25
    wrong = ((out.double() - ref).abs() > bound) | (out.isnan() != ref.isnan())
    assert not wrong.any(), f"{name}: {int(wrong.sum())} of {wrong.numel()}, worst {((out.double() - ref).abs() / bound).nan_to_num().max():.2f} of the bound"


# --------------------------------------------------------------------------------------------------- append ----
def append_inputs(dtype, bits, olds, news, Hkv, D, block, size, seed, device="cpu", pad=0, interleaved=False, ragged=True,
                  values=1.0):
    """olds, news: tokens that each sequence has and gets."""
    g = generator("cpu", seed)
    rows = sum(news) + pad
    totals = [a + b for a, b in zip(olds, news)]
    columns = max(1, -(-max(totals) // block))
    num_blocks = len(olds) * columns + 2
    k, v = ((torch.randn(rows, Hkv, D, generator=g) * values * torch.exp2(torch.randn(rows, Hkv, 1, generator=g))).to(dtype).to(device)
            for _ in range(2))
    if bits == 8:
        (kc, ks), (vc, vs) = (fp8_cache((num_blocks, Hkv, block, D), seed + i, device) for i in (1, 2))
    else:
        kc, vc = (torch.randn(num_blocks, Hkv, block, D, generator=g).to(dtype).to(device) for _ in range(2))
        ks = vs = None
    table = torch.randperm(num_blocks, generator=g)[:len(olds) * columns].reshape(len(olds), columns).to(device)
    starts = torch.tensor([0] + news).cumsum(0).int().to(device) if ragged else None
    cos, sin = tables(max(1, max(totals)), size, device) if size else (None, None)
    return dict(key=k, value=v, key_cache=kc, value_cache=vc, context_lens=torch.tensor(totals, dtype=torch.int32, device=device),
                block_tables=table, query_starts=starts, key_scales=ks, value_scales=vs, cos=cos, sin=sin, interleaved=interleaved)


def copied(args):
    return {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in args.items()}


def check_append(args, name="", exact_scales=True):
    """Runs paged_append on copies of the caches and checks every element of them, those that must not change too."""
    a = copied(args)
    result = flag_attn.paged_append(**a)
    assert result is None
    cpu = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in args.items()}
    num_blocks, Hkv, block, D = cpu["key_cache"].shape
    found = paged_cache.places(cpu["context_lens"], cpu["query_starts"], cpu["key"].shape[0], cpu["block_tables"], block, num_blocks,
                               None if cpu["cos"] is None else cpu["cos"].shape[0])
    dtype = cpu["key"].dtype
    for x, cos, sin in (("key", cpu["cos"], cpu["sin"]), ("value", None, None)):
        before, scales = cpu[x + "_cache"], cpu[x + "_scales"]
        want, want_scales = paged_cache.append(cpu[x], before, scales, found, cos, sin, cpu["interleaved"])
        got = a[x + "_cache"].cpu()
        stored = torch.zeros(num_blocks, block, dtype=torch.bool)
        touched = torch.zeros(num_blocks, dtype=torch.bool)
        for _, _, _, b, slot in found:
            stored[b, slot] = touched[b] = True
        raw = torch.uint8 if scales is not None else torch.int16
        same = (got.view(raw) == before.view(raw)).all(-1)        # (blocks, heads, block)
        if scales is None:
            assert (same | stored[:, None]).all(), f"{name}: {x} cache changed where nothing was stored"
            # one rounding to the type, two products and a sum before it (each at most as large as the pair)
            size = cpu[x].double().abs().amax() * 2 if cos is not None else 0.0
            bad = (got.double() - want).abs() > half_step(dtype) * want.abs() * 1.01 + 4 * U32 * size
            bad &= ~((got.double() == want) | (got.isnan() & want.isnan()))
            assert not (bad & stored[:, None, :, None]).any(), f"{name}: {x} cache"
            continue
        now = a[x + "_scales"].cpu()
        assert torch.equal(now.double(), want_scales), f"{name}: {x} scales"
        grew = now != scales
        assert (same | stored[:, None] | (grew & touched[:, None])[:, :, None]).all(), f"{name}: {x} codes changed where nothing was stored"
        if cos is None:   # nothing but the rounding to e4m3: the same numbers
            equal = (got.double() == want) | (got.double().isnan() & want.isnan())
            assert equal.all(), f"{name}: {x} codes"
        else:             # an fp32 error before the rounding can move a value over a border: a step in place of half of one
            bound = 2.0 ** -3 * want.abs() + 2.0 ** -9
            assert (((got.double() - want).abs() <= bound) | (got.double().isnan() & want.isnan())).all(), f"{name}: {x} codes"
            moved = (got.double() != want) & ~want.isnan()
            assert moved.float().mean() < 1e-3, f"{name}: {x} codes"
    return a


# --------------------------------------------------------------------------------------------------- rotary ----
def rotary_inputs(dtype, B, H, Hk, T, D, size, seed, device="cpu", weight_type=None, positions=None, bthd=True, grad=False):
    """positions: None, 1 (one row for all), 2 (a row per batch entry)."""
    g = generator("cpu", seed)

    def rows(heads):
        t = torch.randn((B, T, heads, D) if bthd else (B, heads, T, D), generator=g).to(dtype).to(device)
        return (t.transpose(1, 2) if bthd else t).requires_grad_(grad)

    q, k = rows(H), rows(Hk)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(weight_type).to(device).requires_grad_(grad) if weight_type else None for _ in range(2))
    where = None
    if positions:
        where = torch.randint(0, 3 * T, (T,) if positions == 1 else (B, T), generator=g).to(device)
    cos, sin = tables(3 * T, size, device)
    return dict(q=q, k=k, cos=cos, sin=sin, positions=where, q_weight=wq, k_weight=wk)


def check_rotary(args, interleaved=False, eps=1e-6, grad=False, name=""):
    a = {n: args[n] for n in ("q", "k", "cos", "sin", "positions", "q_weight", "k_weight")}
    outs = flag_attn.norm_rotary(**a, eps=eps, interleaved=interleaved)
    B, H, T, D = a["q"].shape
    positions = torch.arange(T) if a["positions"] is None else a["positions"].cpu()
    positions = positions.expand(B, T)
    g = generator("cpu", 99)
    gradients = [torch.randn(o.shape, generator=g).to(o.dtype).to(o.device) for o in outs] if grad else None
    if grad:
        leaves = [a[n] for n in ("q", "k", "q_weight", "k_weight") if a[n] is not None]
        got = dict(zip([n for n in ("q", "k", "q_weight", "k_weight") if a[n] is not None],
                       torch.autograd.grad(outs, leaves, gradients, retain_graph=True)))
    for i, (x, w) in enumerate((("q", "q_weight"), ("k", "k_weight"))):
        value = a[x].detach().cpu().double().requires_grad_()
        weight = None if a[w] is None else a[w].detach().cpu().double().requires_grad_()
        ref = rotary.norm_rotary(value, a["cos"].cpu(), a["sin"].cpu(), positions, weight, eps, interleaved)
        out = outs[i].detach().cpu()
        assert out.dtype == a[x].dtype and out.shape == a[x].shape
        # the mean is D fp32 operations (half of their error reaches its root), then a handful on numbers no larger than the row's
        largest = rotary.normalised(value, weight, eps).detach().abs().amax(-1, keepdim=True)
        bound = half_step(out.dtype) * ref.detach().abs() * 1.01 + 2 * (D / 2 + 12) * U32 * largest + 2.0 ** -25
        wrong = ((out.double() - ref.detach()).abs() > bound) | (out.isnan() != ref.detach().isnan())
        assert not wrong.any(), f"{name}: {x}, {int(wrong.sum())} of {wrong.numel()}"
        if not grad:
            continue
        dy = gradients[i].cpu().double()
        want = torch.autograd.grad(ref, (value,) if weight is None else (value, weight), dy)
        dx = got[x].cpu()
        assert dx.dtype == a[x].dtype and dx.shape == a[x].shape
        reach = dy.abs().amax(-1, keepdim=True) * 2
        if weight is not None:   # dx = r (g w - h mean(g w h)), h = x r
            r = 1 / torch.sqrt(value.detach().square().mean(-1, keepdim=True) + eps)
            hat = (value.detach() * r).abs()
            gw = reach * weight.detach().abs().amax()
            reach = r * (gw + hat.amax(-1, keepdim=True) * gw * hat.mean(-1, keepdim=True))
        bound = half_step(dx.dtype) * want[0].abs() * 1.01 + 2 * (2 * D + 16) * U32 * reach + 2.0 ** -25
        assert ((dx.double() - want[0]).abs() <= bound).all(), f"{name}: d{x}"
        if weight is not None:
            dw = got[w].cpu()
            assert dw.dtype == a[w].dtype
            rows = value.numel() // D
            terms = (dy.abs().amax(-1, keepdim=True) * 2 * hat).sum((0, 1, 2))
            bound = (rows + D + 16) * U32 * terms + (half_step(dw.dtype) * 1.01 * want[1].abs() if dw.dtype != torch.float32 else U32 * want[1].abs())
            assert ((dw.double() - want[1]).abs() <= bound).all(), f"{name}: d{w}"
    return outs
