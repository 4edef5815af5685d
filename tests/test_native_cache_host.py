"""The native host path of the operators around the paged cache against the Python form: the launch rule number by number,
and on the GPU the results bit for bit."""
import random

import pytest
import torch

import flag_attn
from flagattention_amd import _lib, append, paged_fp8, rotary
from tests import paged_cache_cases as cases

BF16, FP16 = torch.bfloat16, torch.float16


def test_native_rule_equals_the_python_one():
    native, rng = _lib.native(), random.Random(17)
    for _ in range(2000):
        args = (int(3000 ** rng.random()), rng.choice((1, 2, 3, 8, 16)), rng.choice((1, 2, 4, 5, 16, 17, 40)),
                rng.choice((16, 32, 64, 128, 256, 512)), int(200000 ** rng.random()), rng.choice((256, 304)))
        assert native.e4m3_workgroups(*args) == paged_fp8.choose_workgroups(*args), args


def test_launch_rule():
    """One kernel where a workgroup is done with the longest sequence soon; all compute units where few pairs are long."""
    rule = paged_fp8.choose_workgroups
    assert rule(1, 8, 4, 128, 300, 256) == 0 and rule(1, 8, 4, 128, 4096, 256) == 512
    assert rule(64, 8, 4, 128, 8192, 256) == 512 and rule(300, 16, 1, 64, 700, 256) == 0
    assert rule(3, 4, 12, 256, 120000, 256) == 512 and rule(2, 1, 1, 512, 9000, 256) == 256 and rule(2, 1, 1, 16, 9000, 256) == 1024


class Refuse:
    """Stands for the native path where a call is to be prepared in Python."""
    def __getattr__(self, name):
        return lambda *args: NotImplemented


def same_bits(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.requires_grad == b.requires_grad and \
        torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.gpu
def test_native_calls_equal_the_python_ones(monkeypatch):
    native = _lib.native()
    taken = []

    class Counting:
        def __getattr__(self, name):
            def call(*args):
                out = getattr(native, name)(*args)
                taken.append(out is not NotImplemented)
                return out
            return call

    attends = [cases.attention_inputs(BF16, [300, 0, 7], 8, 2, 128, 16, 71, device="cuda"),
               cases.attention_inputs(FP16, [9000, 33], 4, 1, 64, 20, 72, device="cuda", table_type=torch.int64)]
    appends = [cases.append_inputs(BF16, 8, [3, 0], [1, 1], 2, 128, 16, 128, 73, device="cuda", ragged=False),
               cases.append_inputs(FP16, 16, [3, 0], [10, 5], 2, 64, 8, 0, 74, device="cuda", pad=3)]
    rotaries = [cases.rotary_inputs(BF16, 2, 4, 2, 30, 64, 64, 75, device="cuda", weight_type=torch.float32, grad=True),
                cases.rotary_inputs(FP16, 1, 4, 2, 30, 64, 32, 76, device="cuda", positions=1, grad=True),
                cases.rotary_inputs(FP16, 2, 4, 2, 30, 64, 64, 77, device="cuda", positions=2, weight_type=FP16, bthd=False)]
    single = {n: t[:, :, 0] if n in ("q", "k") else t[:, 0] if n == "positions" else t for n, t in rotaries[2].items()}
    results = []
    for stand_in in (Counting(), Refuse()):
        monkeypatch.setattr(_lib, "native", lambda: stand_in)
        got = [flag_attn.paged_attention_fp8(*a) for a in attends]
        for a in appends:
            c = cases.copied(a)
            flag_attn.paged_append(**c)
            got += [c[n] for n in ("key_cache", "value_cache", "key_scales", "value_scales") if c[n] is not None]
        for a in rotaries + [single]:
            outs = flag_attn.norm_rotary(**a, interleaved=a is rotaries[1])
            got += outs
            if outs[0].requires_grad:
                leaves = [a[n] for n in ("q", "k", "q_weight", "k_weight") if a[n] is not None]
                got += torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
        results.append(got)
    assert all(taken) and len(taken) == 8
    assert len(results[0]) == len(results[1]) and all(same_bits(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_calls_in_error_raise_from_the_python_form():
    q, *rest = cases.attention_inputs(FP16, [20, 9], 4, 2, 64, 16, 78, device="cuda")
    with pytest.raises(AssertionError, match="head_size"):
        flag_attn.paged_attention_fp8(q[..., :48], *rest)
    a = cases.append_inputs(FP16, 8, [3, 9], [4, 7], 2, 64, 16, 64, 79, device="cuda")
    with pytest.raises(AssertionError, match="a row per sequence"):
        flag_attn.paged_append(**{**a, "query_starts": None})
    with pytest.raises(AssertionError, match="on one device"):
        flag_attn.paged_append(**{**a, "key_scales": a["key_scales"].cpu(), "value_scales": a["value_scales"].cpu()})
    r = cases.rotary_inputs(FP16, 2, 4, 2, 6, 64, 64, 80, device="cuda")
    with pytest.raises(AssertionError, match="tables of 5"):
        flag_attn.norm_rotary(r["q"], r["k"], r["cos"][:5], r["sin"][:5])


@pytest.mark.gpu
def test_calls_are_made_in_python_where_something_listens():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Recorder(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    attend = cases.attention_inputs(BF16, [300, 7], 8, 2, 128, 16, 81, device="cuda")
    turn = cases.rotary_inputs(BF16, 2, 4, 2, 30, 64, 64, 82, device="cuda")
    for call in (lambda: flag_attn.paged_attention_fp8(*attend), lambda: flag_attn.norm_rotary(**turn)):
        seen, want = [], call()
        with Recorder():
            got = call()
        assert any("empty" in name for name in seen)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_modules_are_those_of_the_reference_package_name():
    import flag_attn.append
    import flag_attn.paged_fp8
    import flag_attn.rotary
    assert flag_attn.append is append and flag_attn.paged_fp8 is paged_fp8 and flag_attn.rotary is rotary
