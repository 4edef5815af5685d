"""``paged_append``: stores new keys and values in the paged cache that ``paged_attention`` or ``paged_attention_fp8`` reads,
turning the keys by their positions on the way.  No counterpart in the reference, which only reads caches.
"""
import torch

from . import _abi, _lib
from .paged import _HEAD_SIZES
from .paged_fp8 import check_cache, check_cache_layout, check_integers, int32, table_ready

__all__ = ["append"]


def tables_ready(cos, sin, head_size, device):
    """cos and sin as the kernels read them: rows of float32 at 16-byte addresses."""
    assert cos.dim() == 2 and sin.shape == cos.shape, "cos and sin: (positions, rotary size / 2), of one shape"
    assert cos.dtype == sin.dtype == torch.float32, "cos and sin must be float32"
    assert cos.device == sin.device == device, f"cos and sin must be on {device}"
    size = 2 * cos.shape[1]
    assert 0 < size <= head_size and size % 16 == 0, f"the rotary size must be a multiple of 16 up to the head size, got {size}"

    def ready(t):
        return t.stride(1) == 1 and t.stride(0) % 4 == 0 and t.data_ptr() % 16 == 0

    if not (ready(cos) and ready(sin) and cos.stride() == sin.stride()):
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    return cos, sin


def check_written(a, b, name):
    """A pair of tensors that a call writes to."""
    assert a.data_ptr() != b.data_ptr() or a.numel() == 0, f"key_{name} and value_{name} must be tensors of their own"
    assert not any(s == 0 and n > 1 for s, n in zip(a.stride(), a.shape)), f"{name} to be written to must not be expanded"


def append(key, value, key_cache, value_cache, context_lens, block_tables, query_starts=None, key_scales=None,
           value_scales=None, cos=None, sin=None, interleaved=False):
    """Stores ``key`` and ``value`` (rows, heads_kv, head_size), float16 or bfloat16, in ``key_cache`` and ``value_cache``
    (num_blocks, heads_kv, block_size, head_size) in place.

    Sequence s owns rows ``query_starts[s]`` to ``query_starts[s + 1] - 1`` (any integer type, num_seqs + 1 entries that do
    not fall); without ``query_starts`` one row each.  ``context_lens`` (num_seqs,) counts the new tokens, as attention over
    the cache needs it right after: the last row of s goes to position ``context_lens[s] - 1``.  Rows that have no place are
    not stored: rows behind the last sequence's, of negative position (a padding sequence of length 0), behind the block
    table or the rotation's tables, or whose entry in ``block_tables`` (num_seqs, max_blocks_per_seq) is not a block of the
    cache.  The blocks that a call stores to belong to one sequence each, and stand in
    its row of the table once.

    ``cos``, ``sin`` (positions, rotary size / 2), float32: the first ``rotary size`` values of every key are turned by row
    ``position`` of the tables, in pairs (i, i + size / 2) or, ``interleaved``, (2i, 2i + 1).

    A cache of the rows' type takes them rounded once.  A cache of float8_e4m3fn comes with ``key_scales`` and
    ``value_scales`` (num_blocks, heads_kv), float32: a block's scale is the least power of two (2^-118 to 2^120) that keeps
    the largest finite magnitude stored in it within 448; in a block that already holds tokens of the sequence it only grows,
    and where it does what the block holds is rounded again.  Infinities and NaN are stored as NaN.  Not differentiable."""
    if key.is_cuda:   # native host path (``csrc/host.cpp``); what it does not take is served below
        if _lib.native().paged_append(key, value, key_cache, value_cache, context_lens, block_tables, query_starts, key_scales,
                                      value_scales, cos, sin, interleaved) is not NotImplemented:
            return
    assert key.dim() == 3 and key.shape == value.shape and key.dtype == value.dtype, "key and value: (rows, heads_kv, head_size)"
    rows, num_kv_heads, head_size = key.shape
    _abi.dtype_code(key)   # raises for other types
    check_cache_layout(key_cache, value_cache)
    num_blocks, _, block_size, _ = key_cache.shape
    assert key_cache.shape[1] == num_kv_heads and key_cache.shape[3] == head_size, \
        f"rows of {num_kv_heads} heads of {head_size}, and a cache of {tuple(key_cache.shape)}"
    assert head_size in _HEAD_SIZES, f"head_size={head_size}"
    check_written(key_cache, value_cache, "cache")
    assert (key_scales is None) == (value_scales is None), "key_scales and value_scales: both or neither"
    tensors = [value, key_cache, value_cache, block_tables]
    if key_scales is not None:
        check_cache(key_cache, value_cache, key_scales, value_scales)
        check_written(key_scales, value_scales, "scales")
        tensors += [key_scales, value_scales]
    else:
        assert key_cache.dtype == value_cache.dtype == key.dtype, \
            f"without scales the cache has the rows' type: got {key_cache.dtype} and {key.dtype}"
    assert all(t.device == key.device for t in tensors), "all tensors must be on one device"
    block_tables = table_ready(block_tables)
    num_seqs = block_tables.shape[0]
    check_integers("context_lens", context_lens, key.device, (num_seqs,))
    if query_starts is not None:
        check_integers("query_starts", query_starts, key.device, (num_seqs + 1,))
    else:
        assert rows == num_seqs, f"without query_starts a row per sequence: got {rows} rows and {num_seqs} sequences"
    assert (cos is None) == (sin is None), "cos and sin: both or neither"
    if cos is not None:
        cos, sin = tables_ready(cos, sin, head_size, key.device)
    if key.numel() == 0 or num_seqs == 0 or key_cache.numel() == 0 or block_tables.shape[1] == 0 or \
            (cos is not None and cos.shape[0] == 0):   # nothing that has a place
        return
    lib = _lib.get()
    key, value, context_lens = _abi.kernel_ready(key), _abi.kernel_ready(value), int32(context_lens)
    with torch.cuda.device(key.device):
        _abi.paged_append(lib, key, value, key_cache, value_cache, key_scales, value_scales, context_lens,
                          None if query_starts is None else int32(query_starts), block_tables, cos, sin, bool(interleaved))
