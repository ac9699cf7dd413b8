"""Launches over the block-scaled cache whose waves and workgroups attend several items each: capped grids, so
that a modest batch brings the item lookahead, the drawn tickets, the items shared by two waves and the
ring that runs on from one item into the next into play.  Each launch runs twice on one metadata
workspace (the second finds the counters of the first)."""

import pytest
import torch

from arctic_platform_amd.kv_layout import E4M3_MAX, block_scales_shape, kv_cache_shape
from arctic_platform_amd.workloads import make_forest_workload
from oracle import block_scales as oracle
from tests.test_block_scaled_cache import FP8, _check_attention, _query_runs, _random_scales, _used_blocks

# head size, query heads, KV heads, rows per item, waves or workgroups that take tickets of their own per workgroup launched
KERNELS = [(64, 8, 4, 32, 4), (128, 16, 4, 32, 4), (64, 12, 4, 64, 1), (128, 16, 4, 64, 1), (256, 8, 4, 32, 1)]


def _state(md):
    m, layout = md.meta.cpu(), md.layout
    tickets = int(m[layout.header]) * md.plan.num_kv_heads
    return tickets, int(m[layout.header + 3]), int(m[layout.coop_ctr : layout.coop_ctr + 1024].abs().sum())


def _second_partials(md):
    """Partial rows whose scale points to a second partial."""
    scale = md.partial_lse.view(-1, 2)[:, 1].cpu().view(torch.int32)
    return int(((scale & 0x7FFFFF) >= 32).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows,takers", KERNELS)
@pytest.mark.parametrize("cap", [1, 2, 8])
def test_several_items_each(gpu, d, hq, hkv, rows, takers, cap):
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    g = torch.Generator().manual_seed(d + rows + cap)
    seg = [700 + 300 * i for i in range(6)] + [40 + 29 * i for i in range(18)]
    paths = [[i // 3, 6 + i] for i in range(18)]  # six prompts, three samples each
    w = make_forest_workload("several", seg, paths, g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=cap == 2)
    md = build_forest_metadata(
        w.block_table.to(gpu), w.seq_lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=512, rows_per_item=rows
    )
    md.max_workgroups = cap
    tickets, _, _ = _state(md)
    assert tickets >= 3.5 * cap * takers, tickets
    first = None
    for launch in range(2):
        md.partial_lse.zero_()
        out, lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, block_scales=scales.to(gpu))
        torch.cuda.synchronize()
        _, drawn, claims = _state(md)
        assert drawn == 0 and claims == 0, (drawn, claims)
        # (the 32-row kernel of head size 128 shares its last items where the grid is a multiple of eight)
        assert (_second_partials(md) > 0) == (d == 128 and rows == 32 and cap == 8)
        _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale, f"launch {launch}")
        if d != 128 or rows != 32 or cap != 8:  # (where two waves meet inside a shared item depends on timing)
            assert first is None or torch.equal(out, first)
            first = out
    md.reproducible = True
    out, lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, block_scales=scales.to(gpu))
    again, again_lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, again_lse)
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale, "reproducible")


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows,takers", KERNELS)
def test_several_query_run_items_each(gpu, d, hq, hkv, rows, takers):
    """Verify steps and chunks of a prefill under a cap of one workgroup: items whose last tile shows every row
    another number of tokens, one after the other, short ones (fewer tiles than the ring holds) among them."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.forest import rows_from_query_runs

    g = torch.Generator().manual_seed(d + rows)
    lens, news = [300, 64, 197, 33, 160, 7, 450, 81], [4, 4, 1, 33, 40, 7, 21, 2]
    q, cache, scales, table, starts, row_table, row_lens = _query_runs(g, lens, news, hq, hkv, d, 48)
    rt, rl, rg = rows_from_query_runs(starts.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), sum(news), table.shape[1])
    md = build_forest_metadata(table.to(gpu), rl, row_table=rt, row_group=rg, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=128, rows_per_item=rows)
    md.max_workgroups = 1
    assert _state(md)[0] >= 3 * takers
    for launch in range(2):
        out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, d**-0.5, block_scales=scales.to(gpu))
        torch.cuda.synchronize()
        assert _state(md)[1:] == (0, 0)
        _check_attention(out, lse, q, cache, scales, table, row_table, row_lens, d**-0.5, f"launch {launch}")


def test_codes_that_move_to_a_larger_scale_are_exact():
    """3.25 = 1.625 * 2, a code of any power of two above the subnormals; 100 / 2^-2 = 400 lies half way between
    384 and 416 and goes to the even code, 384 = 96 * 4."""
    d, key = 64, torch.full((2, 1, 64), 3.25, dtype=torch.bfloat16)
    key[1] = 100.0
    cache, scales = torch.zeros(kv_cache_shape(1, 16, 1, d)).to(FP8), torch.zeros(block_scales_shape(1, 1))
    for token in range(2):
        cache, scales = oracle.append_reference(cache, scales, key[token : token + 1], key[token : token + 1], torch.tensor([token]))
        assert float(scales[0, 0, 0]) == (2.0**-7, 2.0**-2)[token] and E4M3_MAX * float(scales[0, 0, 0]) >= float(key[token, 0, 0])
    for rows in oracle.token_rows(cache, scales, torch.tensor([0, 1]), d):
        assert (rows[0] == 3.25).all() and (rows[1] == 96.0).all()
