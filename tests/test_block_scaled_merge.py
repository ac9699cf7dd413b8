"""The merge behind attention over the block-scaled cache, chosen by what the rows could have of partials and
done by what they have: every way to it gives the same bits."""

import ctypes
import os

import pytest
import torch

from arctic_platform_amd import _lib
from arctic_platform_amd.forest import make_plan
from arctic_platform_amd.workloads import make_forest_workload
from tests.test_block_scaled_cache import FP8, _check_attention, _random_scales, _used_blocks

# head size, query heads, KV heads, tokens of the sequences (chunks of 32: partials = tokens / 32, rounded up)
CASES = [
    (128, 4, 1, [32 * 17, 32 * 16, 32 * 15 + 1, 0, 5]),  # one wave takes a row of up to 16 partials
    (64, 4, 1, [32 * 33, 32 * 32 - 3, 40]),  # ... 32
    (256, 2, 1, [32 * 9, 32 * 8, 32 * 7 + 1]),  # ... 8
    (128, 4, 1, [32 * 65, 32 * 64, 700]),  # one batch of a workgroup and one more
    (128, 1, 1, [20, 0]),  # short rows under a wide table
]


def _forest(gpu, d, hq, hkv, lens, width):
    from arctic_platform_amd import build_forest_metadata

    g = torch.Generator().manual_seed(d + sum(lens))
    w = make_forest_workload("merge", [max(n, 1) for n in lens], [[i] for i in range(len(lens))], g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    table = torch.zeros(len(lens), max(width, w.block_table.shape[1]), dtype=torch.int32)
    table[:, : w.block_table.shape[1]] = w.block_table
    seq_lens = torch.tensor(lens, dtype=torch.int32)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, seq_lens), powers=True)
    md = build_forest_metadata(table.to(gpu), seq_lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32)
    md.reproducible = True
    return w, scales, table, md


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,lens", CASES)
def test_ways_to_the_merge_agree(gpu, d, hq, hkv, lens):
    from arctic_platform_amd import forest_cascade_decode
    from arctic_platform_amd.ops import forest_cascade_decode_static, forest_pass, merge_partials, prefix_pass, suffix_pass

    w, scales, table, md = _forest(gpu, d, hq, hkv, lens, 64)
    assert md.layout.max_partials >= 16 and len(lens) * hq <= 256
    args, kw = (w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale), dict(block_scales=scales.to(gpu))
    out, lse = forest_cascade_decode(*args, **kw)
    static, static_lse = torch.zeros_like(out), torch.zeros_like(lse)
    forest_cascade_decode_static(*args, out=static, lse=static_lse, **kw)
    prefix_pass(*args, **kw)
    suffix_pass(*args, **kw)
    parts, parts_lse = merge_partials(md, args[0])
    forest_pass(*args, **kw)
    whole, whole_lse = merge_partials(md, args[0])
    wide, _ = forest_cascade_decode(*args, out_dtype=torch.float32, **kw)
    torch.cuda.synchronize()
    for o, l in ((static, static_lse), (parts, parts_lse), (whole, whole_lse), (wide.bfloat16(), lse)):
        assert torch.equal(o, out) and torch.equal(l, lse)
    _check_attention(out, lse, w.q, w.kv_cache, scales, table, range(len(lens)), lens, w.scale, f"lengths {lens}")


@pytest.mark.gpu
def test_passes_over_another_cache_merge_as_before(gpu):
    """The metadata serves a block-scaled cache and one with a scale per head in turn: each merge follows the
    cache of the passes in front of it."""
    from arctic_platform_amd import forest_cascade_decode
    from arctic_platform_amd.ops import forest_pass, merge_partials

    w, scales, _, md = _forest(gpu, 128, 4, 1, [32 * 17, 100], 64)
    q, cache = w.q.to(gpu), w.kv_cache.to(gpu)
    for kw in (dict(block_scales=scales.to(gpu)), dict(), dict(block_scales=scales.to(gpu)), dict(k_scale=torch.full((1,), 0.25).to(gpu))):
        out, lse = forest_cascade_decode(q, cache, md, w.scale, **kw)
        forest_pass(q, cache, md, w.scale, **kw)
        again, again_lse = merge_partials(md, q)
        torch.cuda.synchronize()
        assert torch.equal(again, out) and torch.equal(again_lse, lse), kw


@pytest.mark.gpu
def test_merging_again_what_one_call_attended(gpu):
    """The partial rows of the last forest_cascade_decode, merged once more."""
    from arctic_platform_amd import forest_cascade_decode
    from arctic_platform_amd.ops import merge_partials

    w, scales, _, md = _forest(gpu, 128, 4, 1, [32 * 40, 32 * 29, 100], 64)
    q, cache = w.q.to(gpu), w.kv_cache.to(gpu)
    for kw in (dict(), dict(block_scales=scales.to(gpu)), dict()):
        out, lse = forest_cascade_decode(q, cache, md, w.scale, out_dtype=torch.float32, **kw)
        again, again_lse = merge_partials(md, q, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(again, out) and torch.equal(again_lse, lse), kw


def test_the_merge_of_a_cache_without_separate_passes_is_refused():
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build_library()
    lib, ok = _lib.load_library(), 1 << 20
    plan = make_plan(4, 8, 32, 8, 128)
    for kv_dtype in (_lib.FCA_F32, 4, -1):
        rc = lib.fca_merge_dtype(ctypes.byref(plan), kv_dtype, ok, ok, ok, ok, 32 * 128, 128, _lib.FCA_BF16, None, None)
        assert rc == -2 and f"kv_dtype {kv_dtype}" in lib.fca_last_error().decode()
    assert lib.fca_merge_dtype(ctypes.byref(plan), _lib.FCA_FP8_E4M3_BLOCK, ok, ok, ok, None, 32 * 128, 128, _lib.FCA_BF16, None, None) == -1
