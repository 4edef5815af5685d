"""``paged_attention_fp8``: single-token decode over a paged cache of e4m3 codes with a scale for each block and kv head.

No counterpart in the reference; it stands beside ``paged_attention`` and takes its arguments, with the scales behind the
caches.  ``paged_append`` fills such a cache.
"""
import torch

from . import _abi, _lib
from .paged import _HEAD_SIZES, _num_cus

__all__ = ["attention"]


# By head size: microseconds that a workgroup alone on its pair takes for 128 keys (four wavefronts, a step each), and that a
# balanced launch takes before it streams (two kernels, the scan of the context lengths, the merge), with few pairs (an eighth of
# its workgroups) and with more, each of which costs partial results.
_STEP_US = {16: 1.05, 32: 1.05, 64: 1.05, 128: 1.4, 256: 2.2, 512: 4.5}
_FEW_US = {16: 9.5, 32: 9.5, 64: 9.5, 128: 9.5, 256: 12.0, 512: 15.0}
_BALANCED_US = {16: 12.0, 32: 12.0, 64: 12.0, 128: 13.0, 256: 20.0, 512: 15.0}


def choose_workgroups(num_seqs, num_kv_heads, group, head_size, max_context_len, num_cus):
    """Workgroups of the balanced launch, or 0 for one workgroup per (sequence, kv head, 16 query heads), a single kernel
    that the hardware deals out by itself.  That is as long as the longest sequence takes one workgroup and, with many pairs,
    as the keys' bytes take at 5.5 TB/s, of which the part behind the longest one counts.  Lengths are taken to be spread up
    to the longest.  Measured, one per pair against balanced (us, lengths uniform up to the longest, D = 128):
    8 pairs of up to 512 keys 8.6 / 9.8, of 1024 13.4 / 10.3; 256 pairs of 1024 17.4 / 19.1, of 2048 31 / 24; 512 pairs of
    1024 21 / 27, of 2048 35.5 / 37.1, of 4096 67 / 64, of 8192 133 / 100; 2048 pairs of 2048 104 / 117; D = 64: 256 pairs of
    1024 14.1 / 13.8, 512 16.3 / 17.7, 4096 61 / 74; D = 32: 256 pairs of 1024 11.3 / 13.1, of 2048 21 / 15; D = 256: 4 pairs
    of 256 9.4 / 12.0, of 512 14 / 12, 512 pairs of 1024 31 / 35, of 2048 54 / 62, 256 pairs of 2048 39 / 36; D = 512: 96 pairs
    of 512 23 / 23, of 1024 56 / 28.
    A compute unit holds four workgroups up to head size 64, two up to 256 and one above."""
    pairs = num_seqs * num_kv_heads * (-(-group // 16))
    stream = pairs * max_context_len * head_size / 5.5e6
    wgs = num_cus * (4 if head_size <= 64 else 2 if head_size <= 256 else 1)
    fixed = (_FEW_US if 8 * pairs <= wgs else _BALANCED_US)[head_size]
    alone = 3.0 + _STEP_US[head_size] * (-(-max_context_len // 128)) + 0.6 * stream
    return 0 if alone <= fixed + stream else wgs


def check_cache(key_cache, value_cache, key_scales, value_scales):
    """A pair of e4m3 caches (num_blocks, heads_kv, block_size, head_size) and their scales."""
    assert key_cache.dtype == value_cache.dtype == torch.float8_e4m3fn, \
        f"an 8-bit cache holds float8_e4m3fn, got {key_cache.dtype} and {value_cache.dtype}"
    assert key_scales.dtype == value_scales.dtype == torch.float32, "the scales of an 8-bit cache are float32"
    assert key_scales.shape == value_scales.shape == key_cache.shape[:2], \
        f"one scale per block and kv head: got {tuple(key_scales.shape)} for a cache of {tuple(key_cache.shape)}"
    assert key_scales.stride() == value_scales.stride(), "key and value scales must share their strides"


def check_cache_layout(key_cache, value_cache):
    assert key_cache.dim() == 4 and value_cache.shape == key_cache.shape
    assert key_cache.stride() == value_cache.stride(), "key and value cache must share their strides"
    align = 16 // key_cache.element_size()
    assert key_cache.stride(3) == 1 and not any(s % align for n, s in zip(key_cache.shape[:3], key_cache.stride()[:3]) if n > 1) \
        and key_cache.data_ptr() % 16 == 0 and value_cache.data_ptr() % 16 == 0, \
        "cache rows must be 16-byte aligned, with unit stride on the last dimension"


def check_integers(name, t, device, shape):
    assert not t.dtype.is_floating_point and t.dtype not in (torch.bool,), f"{name} must hold integers, got {t.dtype}"
    assert t.device == device, f"{name} must be on {device}, got {t.device}"
    assert t.shape == shape, f"{name} must be {tuple(shape)}, got {tuple(t.shape)}"


def int32(t):
    """Contiguous 32-bit integers, as the kernels read them."""
    return (t if t.dtype == torch.int32 else t.to(torch.int32)).contiguous()


def table_ready(block_tables):
    assert block_tables.dim() == 2 and block_tables.dtype in (torch.int32, torch.int64), "block_tables: two dimensions, int32 or int64"
    return block_tables if block_tables.stride(1) == 1 else block_tables.contiguous()


def attention(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, attn_scale,
              max_context_len):
    """query (num_seqs, heads_q, head_size), float16 or bfloat16; key_cache / value_cache (num_blocks, heads_kv, block_size,
    head_size), float8_e4m3fn with identical strides; key_scales / value_scales (num_blocks, heads_kv), float32: a code c
    stands for ``c * scale``.  context_lens (num_seqs,) of any integer type; block_tables (num_seqs, max_blocks_per_seq)
    int32 or int64; max_context_len bounds the context lengths (it decides how the work is dealt out, not what is read).

    Returns out shaped like ``query``; a sequence of context length 0 gets a zero row, and so does every one where the
    cache or the table is empty.  A key whose block number is not one of the cache's, or whose column is not in the table,
    makes the rows that see it NaN; nothing is read for it (and a length past the table's end takes no longer than one key past it).  Not differentiable."""
    if query.is_cuda:   # native host path (``csrc/host.cpp``); what it does not take is served below
        out = _lib.native().paged_fp8(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables,
                                      attn_scale, max_context_len)
        if out is not NotImplemented:
            return out
    num_seqs, num_q_heads, head_size = query.shape
    check_cache(key_cache, value_cache, key_scales, value_scales)
    check_cache_layout(key_cache, value_cache)
    num_blocks, num_kv_heads, block_size, _ = key_cache.shape
    assert key_cache.shape[3] == head_size, f"head_size={head_size}, and a cache of {key_cache.shape[3]}"
    assert head_size in _HEAD_SIZES, f"head_size={head_size}"
    assert num_kv_heads > 0 and num_q_heads % num_kv_heads == 0
    assert all(t.device == query.device for t in (key_cache, value_cache, key_scales, value_scales, block_tables)), \
        "all tensors must be on one device"
    check_integers("context_lens", context_lens, query.device, (num_seqs,))
    block_tables = table_ready(block_tables)
    assert block_tables.shape[0] == num_seqs
    _abi.dtype_code(query)   # raises for other types
    if query.numel() == 0 or num_blocks == 0 or block_size == 0 or block_tables.shape[1] == 0:   # nothing to launch
        return torch.zeros_like(query)
    lib = _lib.get()
    query = _abi.kernel_ready(query)
    context_lens = int32(context_lens)
    out = torch.empty_like(query)
    if not _abi.is_kernel_ready(out):
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    with torch.cuda.device(query.device):
        num_wgs = choose_workgroups(num_seqs, num_kv_heads, num_q_heads // num_kv_heads, head_size, int(max_context_len),
                                    _num_cus(lib, query.device))
        workspace = None
        if num_wgs > 0:
            nbytes = lib.paged_attn_e4m3_workspace(num_wgs, head_size)
            workspace = torch.empty(nbytes // 4, dtype=torch.float32, device=query.device)
        _abi.paged_attn_e4m3(lib, out, query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables,
                             attn_scale, workspace, num_wgs)
    return out
