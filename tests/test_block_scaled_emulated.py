"""The kernels of the block-scaled cache on the CPU emulation (tests/emu), every buffer flush against an
inaccessible page: addresses, and the kernels' own orders -- direct-to-LDS loads that land as late as
the waits allow, waves, workgroups and lanes taken from the last to the first, several workgroups
at a time.  Values are checked against the same restatement as on the GPU."""

import ctypes
import random

import pytest
import torch

from arctic_platform_amd import _lib
from arctic_platform_amd.forest import ForestMetadata, make_plan
from arctic_platform_amd.kv_layout import quantize_blocks
from arctic_platform_amd.workloads import make_forest_workload
from oracle import block_scales as oracle
from tests.test_block_scaled_cache import FP8, _check_attention, _old_state, _query_runs, _random_scales, _rows, _used_blocks
from tests.test_emulated_kernels import EMU_WORKGROUPS, _ok, emu, guarded  # noqa: F401  (emu is a fixture)
from tests.test_gpu_random_forests import random_forest


@pytest.fixture(params=["early", "late", "late-reversed", "late-eight-at-a-time"])
def order(emu, request):  # noqa: F811
    emu.emu_set_dma_late(1 if request.param.startswith("late") else 0)
    emu.emu_set_run_order(7 if request.param.endswith("reversed") else 0)
    emu.emu_set_host_threads(8 if request.param.endswith("time") else 1)
    yield request.param
    emu.emu_set_dma_late(0), emu.emu_set_run_order(0), emu.emu_set_host_threads(1)


def _attend(lib, q, cache, scales, table, row_lens, scale, hq, hkv, d, chunk, rows, row_table=None, row_group=None, reread=0, workgroups=EMU_WORKGROUPS):
    n, mb = q.shape[0], table.shape[1]
    plan = make_plan(n, mb, hq, hkv, d, chunk_tokens=chunk, rows_per_item=rows)
    layout = _lib.FcaMetaLayout()
    _ok(lib, lib.fca_meta_describe(ctypes.byref(plan), ctypes.byref(layout)))
    nm, no, nl = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    _ok(lib, lib.fca_workspace_bytes_dtype(ctypes.byref(plan), _lib.FCA_FP8_E4M3_BLOCK, ctypes.byref(nm), ctypes.byref(no), ctypes.byref(nl)))
    meta = guarded(torch.zeros(nm.value // 4, dtype=torch.int32))
    po = guarded(torch.full((no.value // 2,), float("nan"), dtype=torch.float16))
    pl = guarded(torch.full((nl.value // 4,), float("nan"), dtype=torch.float32))
    bt, sl, qg, sc = guarded(table), guarded(row_lens), guarded(q), guarded(scales)
    kv = guarded(cache.view(torch.uint8))
    if row_table is None:
        _ok(lib, lib.fca_build_metadata(ctypes.byref(plan), bt.data_ptr(), bt.stride(0), sl.data_ptr(), meta.data_ptr(), None))
    else:
        rt, rg = guarded(row_table), guarded(row_group)
        _ok(lib, lib.fca_build_metadata_rows(ctypes.byref(plan), bt.data_ptr(), bt.stride(0), table.shape[0], rt.data_ptr(), rg.data_ptr(), sl.data_ptr(), meta.data_ptr(), 0, None))
    md = ForestMetadata(plan=plan, layout=layout, meta=meta, partial_out=po, partial_lse=pl, block_table=bt, seq_lens=sl)
    md.check()
    t = _lib.FcaTensors(
        qg.data_ptr(), qg.stride(0), qg.stride(1), kv.data_ptr(), kv.data_ptr() + kv.stride(0), kv.stride(1), kv.stride(2),
        _lib.FCA_FP8_E4M3_BLOCK, reread, bt.data_ptr(), bt.stride(0), sc.data_ptr(), None, float(scale), 0, workgroups, 0,
    )
    out, lse = guarded(torch.full((n, hq, d), 3.0).bfloat16()), guarded(torch.full((n, hq), 3.0))
    for _ in range(2):  # (the second launch finds the counters of the first)
        _ok(lib, lib.fca_decode_step(ctypes.byref(plan), ctypes.byref(t), meta.data_ptr(), po.data_ptr(), pl.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), _lib.FCA_BF16, lse.data_ptr(), None))
    assert int(meta[layout.header + 3]) == 0 and int(meta[layout.coop_ctr : layout.coop_ctr + 1024].abs().sum()) == 0
    return out, lse


@pytest.mark.parametrize(
    "seed,hq,hkv,d,depth,fanout,seg,leaf,chunk,rows,workgroups",
    [
        (51, 16, 4, 128, 2, 4, (40, 300), (1, 90), 128, 64, 2),  # several items per workgroup, one and two row tiles
        (52, 8, 2, 64, 2, 4, (1, 200), (1, 70), 96, 64, 2),
        (53, 4, 1, 256, 2, 3, (1, 200), (1, 60), 64, 32, 2),
        (54, 8, 2, 128, 2, 3, (1, 150), (1, 90), 64, 32, 2),
    ],
)
def test_attention(emu, order, seed, hq, hkv, d, depth, fanout, seg, leaf, chunk, rows, workgroups):  # noqa: F811
    seg_len, paths = random_forest(random.Random(seed), depth, fanout, seg, leaf)
    g = torch.Generator().manual_seed(seed)
    w = make_forest_workload("random", seg_len, paths, g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=False)
    out, lse = _attend(emu, w.q, w.kv_cache, scales, w.block_table, w.seq_lens, w.scale, hq, hkv, d, chunk, rows, workgroups=workgroups)
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale, f"seed {seed}")


@pytest.mark.parametrize("d,rows", [(128, 64), (256, 32), (64, 32)])
def test_query_runs_with_a_nan(emu, order, d, rows):  # noqa: F811
    """Runs over shared and own blocks; one value behind the last row of each run's block is NaN, and one
    in the last run, which the rows in front of it do not see."""
    hq, hkv = 4, 2
    g = torch.Generator().manual_seed(d)
    lens, news = [70, 35, 51], [5, 3, 9]
    q, cache, scales, table, starts, row_table, row_lens = _query_runs(g, lens, news, hq, hkv, d, 32)
    clean = cache.clone()
    at = lens[2] - 2  # the last row but one of the third run
    cache.view(torch.uint8)[1, int(table[2, at // 16]), 1].view(d, 16)[d // 2 + 3, at % 16] = 0xFF
    group = torch.tensor([s * table.shape[1] + (n - 1) // 16 for s, n in zip(row_table, row_lens)], dtype=torch.int32)
    out, lse = _attend(
        emu, q, cache, scales, table, torch.tensor(row_lens, dtype=torch.int32), 0.1, hq, hkv, d, 32, rows,
        row_table=torch.tensor(row_table, dtype=torch.int32), row_group=group, reread=1, workgroups=2,
    )
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[-2:, hq // 2 :, d // 2 + 3] = True
    assert torch.equal(out.isnan(), bad) and not lse.isnan().any()
    ref = oracle.attention(q, clean, scales, table, row_table, row_lens, 0.1)[0]
    _check_attention(torch.where(bad, ref.bfloat16(), out), lse, q, clean, scales, table, row_table, row_lens, 0.1, "query runs")


@pytest.mark.parametrize("rows,hkv,max_len", [(32, 4, None), (64, 4, None), (32, 1, 2900)])
def test_nan_keys_in_items_shared_by_two_waves(emu, rows, hkv, max_len):  # noqa: F811
    """NaN keys all over long prompts and private parts: a row is NaN, log-sum-exp included, exactly where
    it sees one, whichever wave of a pair attended the tile that holds it and whichever merge follows."""
    hq, d, chunk = 4 * hkv, 128, 512
    g = torch.Generator().manual_seed(77)
    if max_len is None:
        seg = [700 + 300 * i for i in range(6)] + [40 + 29 * i for i in range(18)]
        paths = [[i // 3, 6 + i] for i in range(18)]
    else:  # one long sequence and short ones: rows with enough partials for the merge of long rows
        seg, paths = [16 * 512 + 77] + [40 + 300 * i for i in range(9)], [[i] for i in range(10)]
    w = make_forest_workload("nan", seg, paths, g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=True)
    clean, cache = w.kv_cache, w.kv_cache.clone()
    bad = torch.zeros(w.num_seqs, hkv, dtype=torch.bool)
    for s in range(0, w.num_seqs, 2):
        at, head = int(torch.randint(0, int(w.seq_lens[s]), (1,), generator=g)), s // 2 % hkv
        blk = int(w.block_table[s, at // 16])
        cache.view(torch.uint8)[0, blk, head].view(d // 16, 16, 16)[3, at % 16, 5] = 0x7F
        for o in range(w.num_seqs):
            where = (w.block_table[o, : (int(w.seq_lens[o]) + 15) // 16] == blk).nonzero()
            bad[o, head] |= bool(len(where)) and int(where[0]) * 16 + at % 16 < int(w.seq_lens[o])
    out, lse = _attend(emu, w.q, cache, scales, w.block_table, w.seq_lens, w.scale, hq, hkv, d, chunk, rows, workgroups=8 if hkv > 1 else 2)
    bad = bad.repeat_interleave(4, dim=1)
    assert torch.equal(lse.isnan(), bad) and torch.equal(out.isnan(), bad[..., None].expand_as(out))
    ref, ref_lse, _, _ = oracle.attention(w.q, clean, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale)
    keep = torch.where(bad[..., None], ref.bfloat16(), out), torch.where(bad, ref_lse.float(), lse)
    _check_attention(*keep, w.q, clean, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale, "nan keys")


@pytest.mark.parametrize("d,hkv,t", [(64, 3, 70), (128, 1, 300), (256, 2, 5)])
def test_append_and_gather(emu, order, d, hkv, t):  # noqa: F811
    g = torch.Generator().manual_seed(t)
    nb = (t + 40) // 16 + 2
    cache, scales = _old_state(g, nb, hkv, d)
    pos = 7 + torch.arange(t)
    slots = (torch.randperm(nb, generator=g)[pos // 16] * 16 + pos % 16).to(torch.int64)
    slots[t // 2], slots[-1] = -1, nb * 16
    if t == 70:
        slots = slots[torch.randperm(t, generator=g)]
    key, value = _rows(g, t, hkv, d), _rows(g, t, hkv, d)
    want, table = oracle.append_reference(cache, scales, key, value, slots)
    kv, sc, sl, k, v = guarded(cache.view(torch.uint8)), guarded(scales), guarded(slots), guarded(key), guarded(value)
    args = (k.stride(0), k.stride(1), t, hkv, d, sl.data_ptr(), kv.data_ptr(), kv.data_ptr() + kv.stride(0), kv.stride(1), kv.stride(2), nb, sc.data_ptr(), None)
    _ok(emu, emu.fca_append_kv_block_scaled(k.data_ptr(), v.data_ptr(), *args))
    assert torch.equal(kv, want.view(torch.uint8))
    assert torch.equal(sc[~table.isnan()], table[~table.isnan()])
    ok, ov = guarded(torch.zeros_like(key)), guarded(torch.zeros_like(value))
    _ok(emu, emu.fca_gather_kv_block_scaled(ok.data_ptr(), ov.data_ptr(), *args))
    rk, rv = oracle.token_rows(want, table, slots, d)
    assert torch.equal(ok, rk.float().bfloat16()) and torch.equal(ov, rv.float().bfloat16())


def test_a_launch_requests_every_block_about_once(emu):  # noqa: F811
    """Bytes the streaming loads ask for against the bytes of the distinct blocks, at a few items per
    workgroup (a short item repeats its last tile up to the depth of the ring)."""
    hq, hkv, d = 8, 1, 128
    g = torch.Generator().manual_seed(3)
    w = make_forest_workload("two", [2000, 700, 800, 900, 400], [[0, 1], [0, 2], [0, 3], [0, 4]], g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8)
    _, scales = quantize_blocks(*(torch.randn(w.kv_cache.shape[1], 16, hkv, d, generator=g) for _ in range(2)))
    for rows in (32, 64):
        emu.emu_take_streamed_bytes.restype = ctypes.c_ulonglong
        emu.emu_take_streamed_bytes()
        _attend(emu, w.q, w.kv_cache, scales, w.block_table, w.seq_lens, w.scale, hq, hkv, d, 512, rows, workgroups=1)
        asked = emu.emu_take_streamed_bytes() / 2
        partials = 4 * 12 * hq * (2 * d + 8) * 3  # (the merge reads its partial rows with streaming loads too)
        assert asked - partials <= 1.25 * w.unique_tokens * 2 * hkv * d, (rows, asked, w.unique_tokens * 2 * hkv * d)


@pytest.mark.parametrize("d,rows,workgroups", [(128, 64, 1), (64, 64, 2), (256, 32, 1), (256, 32, 3)])
def test_long_query_runs_shared_by_two_workgroups(emu, order, d, rows, workgroups):  # noqa: F811
    """Items of 16 to 22 tiles whose last tile shows each row another number of tokens, or none: attended by
    two workgroups, one of which begins with that tile."""
    hq, hkv = 4, 1
    g = torch.Generator().manual_seed(d + workgroups)
    lens, news = [600, 545, 700, 560], [5, 3, 9, 17]
    q, cache, scales, table, starts, row_table, row_lens = _query_runs(g, lens, news, hq, hkv, d, 32)
    clean = cache.clone()
    at = lens[2] - 2
    cache.view(torch.uint8)[1, int(table[2, at // 16]), 0].view(d, 16)[d // 2 + 3, at % 16] = 0xFF
    group = torch.tensor([s * table.shape[1] + (n - 1) // 16 for s, n in zip(row_table, row_lens)], dtype=torch.int32)
    out, lse = _attend(
        emu, q, cache, scales, table, torch.tensor(row_lens, dtype=torch.int32), 0.1, hq, hkv, d, 1024, rows,
        row_table=torch.tensor(row_table, dtype=torch.int32), row_group=group, reread=1, workgroups=workgroups,
    )
    last = torch.tensor([s == 2 and n > at for s, n in zip(row_table, row_lens)])
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[last, :, d // 2 + 3] = True
    assert int(last.sum()) == 2 and torch.equal(out.isnan(), bad) and not lse.isnan().any()
    ref = oracle.attention(q, clean, scales, table, row_table, row_lens, 0.1)[0]
    _check_attention(torch.where(bad, ref.bfloat16(), out), lse, q, clean, scales, table, row_table, row_lens, 0.1, "query runs")
