"""``norm_rotary``: norm of queries and keys for each head and their rotation by position in one pass, with gradients.

No counterpart in the reference; it makes what its operators take: the queries and keys of ``flash_attention``, the two pairs
of ``piecewise_attention`` (one pair of projections turned by two sets of tables), the queries of ``paged_attention``.
"""
import torch

from . import _abi, _lib
from .append import tables_ready
from .paged import _HEAD_SIZES

__all__ = ["norm_rotary"]


def _result_like(t):
    o = torch.empty_like(t)
    return o if _abi.is_kernel_ready(o) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class NormRotary(torch.autograd.Function):
    """q (B, H, T, D), k (B, Hk, T, D), positions (B, T) or None; the arguments have been checked."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        lib = _lib.get()
        q, k = _abi.kernel_ready(q), _abi.kernel_ready(k)
        q_out, k_out = _result_like(q), _result_like(k)
        if q.shape[0] * q.shape[2] > 0:
            with torch.cuda.device(q.device):
                _abi.fa_norm_rotary(lib, q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, interleaved, eps)
        kept = (None, None) if q_weight is None else (q, k)   # a rotation alone is undone without its input
        ctx.save_for_backward(*kept, q_weight, k_weight, cos, sin, positions)
        ctx.shapes, ctx.eps, ctx.interleaved = (q.shape, k.shape), eps, interleaved
        return q_out, k_out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        if torch.is_grad_enabled():
            raise RuntimeError("norm_rotary is differentiable once: its gradients cannot be part of a graph (create_graph)")
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        lib = _lib.get()
        dq_out, dk_out = _abi.kernel_ready(dq_out), _abi.kernel_ready(dk_out)
        dq, dk = (torch.empty(s, dtype=dq_out.dtype, device=dq_out.device) for s in ctx.shapes)
        dq_weight = dk_weight = workspace = None
        if q_weight is not None:
            dq_weight, dk_weight = torch.empty_like(q_weight), torch.empty_like(k_weight)
        if dq.shape[0] * dq.shape[2] == 0:
            return dq, dk, *(None if w is None else w.zero_() for w in (dq_weight, dk_weight)), None, None, None, None, None
        with torch.cuda.device(dq.device):
            if q_weight is not None:
                nbytes = lib.fa_norm_rotary_workspace(dq.shape[3])
                workspace = torch.empty(nbytes // 4, dtype=torch.float32, device=dq.device)
            _abi.fa_norm_rotary_bwd(lib, q, k, dq_out, dk_out, dq, dk, q_weight, k_weight, dq_weight, dk_weight, workspace,
                                    cos, sin, positions, ctx.interleaved, ctx.eps)
        return dq, dk, dq_weight, dk_weight, None, None, None, None, None


def norm_rotary(q, k, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    """q (batch, heads_q, seqlen, headdim), k (batch, heads_k, seqlen, headdim), float16 or bfloat16, with any strides that
    ``flash_attention`` takes; or single tokens, (num_tokens, heads, headdim) each, as ``paged_attention`` takes queries.

    With ``q_weight`` and ``k_weight`` (headdim,), of the inputs' type or float32, every row (one head of one token) is
    normalised, ``x * rsqrt(mean(x^2) + eps) * weight``.  Then its first ``rotary size`` values are turned by the angles of
    its position: row ``position`` of ``cos`` and ``sin`` (positions, rotary size / 2), float32, in pairs (i, i + size / 2)
    or, ``interleaved``, (2i, 2i + 1).  ``positions`` holds integers (int32 or int64): (seqlen,) or (batch, seqlen), or
    (num_tokens,) for single tokens; without it the position is the token's index.  A position without a row in the tables
    turns by NaN.  All arithmetic is in fp32, rounded once.

    Returns (q_out, k_out), shaped like the inputs.  Differentiable in q, k and the weights, once (not with
    ``create_graph``); cos and sin get no gradient."""
    if q.is_cuda:   # native host path (``csrc/host.cpp``); what it does not take is served below
        out = _lib.native().norm_rotary(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
        if out is not NotImplemented:
            return out
    assert q.dim() in (3, 4) and k.dim() == q.dim(), "q and k: (batch, heads, seqlen, headdim) or (num_tokens, heads, headdim)"
    single = q.dim() == 3
    if single:
        assert positions is not None, "single tokens need positions"
        q, k, positions = q.unsqueeze(2), k.unsqueeze(2), positions.unsqueeze(-1)
    B, H, T, D = q.shape
    assert k.shape[0] == B and k.shape[2] == T and k.shape[3] == D and H > 0 and k.shape[1] > 0
    assert D in _HEAD_SIZES, f"headdim={D}"
    assert q.dtype == k.dtype and q.device == k.device
    _abi.dtype_code(q)   # raises for other types
    assert not (cos.requires_grad or sin.requires_grad), "cos and sin get no gradient"
    cos, sin = tables_ready(cos, sin, D, q.device)
    assert (q_weight is None) == (k_weight is None), "q_weight and k_weight: both or neither"
    if q_weight is not None:
        for w in (q_weight, k_weight):
            assert w.shape == (D,) and w.device == q.device and w.dtype in (q.dtype, torch.float32), \
                f"weights: ({D},) of {q.dtype} or float32"
        assert q_weight.dtype == k_weight.dtype, "q_weight and k_weight must have one type"
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        assert 1e-30 <= eps < float("inf"), f"eps must be positive, got {eps}"
    else:
        eps = 1.0   # not used
    if positions is None:
        assert T <= cos.shape[0], f"{T} tokens, and tables of {cos.shape[0]} positions"
    else:
        assert positions.dtype in (torch.int32, torch.int64), f"positions must be int32 or int64, got {positions.dtype}"
        assert positions.device == q.device, f"positions must be on {q.device}"
        assert positions.shape in ((T,), (B, T)), f"positions: ({T},) or ({B}, {T}), got {tuple(positions.shape)}"
        positions = positions.expand(B, T)
    assert cos.shape[0] > 0 or B * T == 0, "empty tables"
    q_out, k_out = NormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
    return (q_out.squeeze(2), k_out.squeeze(2)) if single else (q_out, k_out)
