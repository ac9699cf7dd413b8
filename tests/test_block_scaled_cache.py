"""The KV cache in 8 bits with a scale per block, KV head and plane: writer and reader bit for bit
against their restatement in 64 bits, attention against the same within derived bounds, and the
three together through a decode loop and through the adapter."""

import random

import pytest
import torch

from arctic_platform_amd.kv_layout import (
    block_scale_for, block_scales_shape, dequantize_blocks, kv_cache_shape, pack_blocks, quantize_blocks,
)
from arctic_platform_amd.workloads import make_forest_workload
from oracle import block_scales as oracle
from tests.test_gpu_random_forests import random_forest

FP8 = torch.float8_e4m3fn


# ---- the restatement itself and the host helpers (no GPU) -----------------------------------------


def test_oracle_rounds_as_the_format_does():
    x = torch.cat([torch.randn(4000) * 10.0 ** torch.randint(-4, 3, (4000,)), oracle.VALUES.float(), -oracle.VALUES.float()])
    mid = (oracle.VALUES[1:] + oracle.VALUES[:-1]).float() / 2  # ties
    x = torch.cat([x, mid, -mid]).clamp(-448, 448)
    assert torch.equal(oracle.encode(x.double()), x.to(FP8).view(torch.uint8))
    codes = torch.arange(256, dtype=torch.uint8)
    got, want = oracle.decode(codes), codes.view(FP8).double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("amax", [0.0, 1e-45, 2.0**-92, 447.9, 448.0, 448.1, 1.0, 1.75, 1.7500001, 3.3e38, 2.0**-109, 2.0**-91])
def test_scale_rule(amax):
    a = torch.tensor([amax], dtype=torch.float32)
    assert float(block_scale_for(a)) == oracle.scale_for(float(a))


def test_quantize_blocks_is_what_the_writer_leaves():
    g = torch.Generator().manual_seed(3)
    nb, hkv, d = 5, 2, 64
    k = (torch.randn(nb, 16, hkv, d, generator=g) * torch.exp(2 * torch.randn(nb, 1, hkv, 1, generator=g))).bfloat16()
    v = torch.randn(nb, 16, hkv, d, generator=g).bfloat16()
    v[2, 3, 1, 5], v[2, 4, 1, 5], k[4] = float("inf"), float("nan"), 0.0
    cache, scales = quantize_blocks(k, v)
    empty = torch.zeros(kv_cache_shape(nb, 16, hkv, d)).to(FP8)
    want, table = oracle.append_reference(
        empty, torch.zeros(block_scales_shape(nb, hkv)), k.view(-1, hkv, d), v.view(-1, hkv, d), torch.arange(nb * 16)
    )
    assert torch.equal(cache.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, table)
    kk, vv = dequantize_blocks(cache, scales, d)
    # half a step of e4m3 relative to the value, or half its smallest step times the scale
    for x, y, plane in ((k.float(), kk, 0), (v.float(), vv, 1)):
        bound = torch.maximum(x.abs() * 2.0**-4, scales[:, None, :, plane : plane + 1] * 2.0**-10)
        ok = ((x - y).abs() <= bound) | ~torch.isfinite(x)
        assert ok.all()


def test_a_later_larger_token_moves_the_earlier_codes_exactly():
    """Codes above the subnormals move to a larger power of two without a rounding."""
    d, key = 64, torch.full((2, 1, 64), 3.25, dtype=torch.bfloat16)
    key[1] = 100.0
    cache = torch.zeros(kv_cache_shape(1, 16, 1, d)).to(FP8)
    scales = torch.zeros(block_scales_shape(1, 1))
    cache, scales = oracle.append_reference(cache, scales, key[:1], key[:1], torch.tensor([0]))
    assert float(scales[0, 0, 0]) == 2.0**-7
    cache, scales = oracle.append_reference(cache, scales, key[1:], key[1:], torch.tensor([1]))
    assert float(scales[0, 0, 0]) == 2.0**-2
    k, _ = oracle.token_rows(cache, scales, torch.tensor([0, 1]), d)
    assert (k[0] == 3.25).all() and (k[1] == 96.0).all() or (k[1] == 104.0).all()


# ---- writer and reader --------------------------------------------------------------------------


def _old_state(g, nb, hkv, d):
    """A cache in use: codes and scales of full blocks, a few of them unset or set by somebody else."""
    k, v = (torch.randn(nb, 16, hkv, d, generator=g) * torch.exp(torch.randn(nb, 1, hkv, 1, generator=g)) for _ in range(2))
    cache, scales = quantize_blocks(k, v)
    scales[0] = 0.0
    if nb > 3:
        scales[1], scales[2, 0] = float("nan"), float("inf")
        scales[3] = torch.tensor([0.013, 0.4])  # no power of two
    return cache, scales


def _rows(g, t, hkv, d, spread=1.5):
    return (torch.randn(t, hkv, d, generator=g) * torch.exp(spread * torch.randn(t, 1, 1, generator=g))).bfloat16()


def _append_and_check(gpu, cache, scales, key, value, slots, fused=True):
    """One call on the device against the restatement, bit for bit; returns the new state (host)."""
    from arctic_platform_amd import append_kv

    want, table = oracle.append_reference(cache, scales, key, value, slots)
    t, hkv, d = key.shape
    if fused:  # views of a fused projection's output [T, 2 Hkv + 2 Hkv, D]
        rows = torch.zeros(t, 4 * hkv, d, dtype=torch.bfloat16, device=gpu)
        rows[:, 2 * hkv : 3 * hkv], rows[:, 3 * hkv :] = key.to(gpu), value.to(gpu)
        dk, dv = rows[:, 2 * hkv : 3 * hkv], rows[:, 3 * hkv :]
    else:
        dk, dv = key.to(gpu), value.to(gpu)
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    append_kv(dk, dv, dc, slots.to(gpu), block_scales=ds)
    torch.cuda.synchronize()
    got, gs = dc.cpu(), ds.cpu()
    same = (gs == table) | (gs.isnan() & table.isnan())
    assert same.all(), (gs[~same], table[~same])
    differ = (got.view(torch.uint8) != want.view(torch.uint8)).nonzero()
    assert len(differ) == 0, (len(differ), differ[:4].tolist())
    return got, gs


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv", [(64, 1), (64, 3), (128, 2), (256, 2)])
def test_append_decode_steps(gpu, d, hkv):
    """Five steps of one token per sequence, from the middle of a block over its end, padded."""
    g = torch.Generator().manual_seed(d + hkv)
    nb, seqs = 14, 5
    cache, scales = _old_state(g, nb, hkv, d)
    table = torch.randperm(nb, generator=g)[: 2 * seqs].view(seqs, 2)
    pos = torch.tensor([0, 13, 15, 7, 12])
    for _ in range(5):
        slots = table[torch.arange(seqs), pos // 16] * 16 + pos % 16
        slots = torch.cat([slots[:2], torch.tensor([-1]), slots[2:], torch.tensor([-1, -5])])
        cache, scales = _append_and_check(gpu, cache, scales, _rows(g, 8, hkv, d), _rows(g, 8, hkv, d), slots)
        pos = pos + 1


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv,start,t", [(64, 2, 0, 16), (64, 2, 5, 75), (128, 1, 8, 41), (128, 8, 0, 1), (256, 1, 15, 33), (128, 2, 3, 300)])
def test_append_prompts(gpu, d, hkv, start, t):
    """Runs of consecutive tokens, a padding token inside, off and on block boundaries."""
    g = torch.Generator().manual_seed(100 + t)
    nb = (start + t + 15) // 16 + 3
    cache, scales = _old_state(g, nb, hkv, d)
    table = torch.randperm(nb, generator=g)
    pos = start + torch.arange(t)
    slots = table[pos // 16] * 16 + pos % 16
    if t > 40:
        slots[37] = -1
    _append_and_check(gpu, cache, scales, _rows(g, t, hkv, d), _rows(g, t, hkv, d), slots, fused=start != 8)


@pytest.mark.gpu
@pytest.mark.parametrize("d,seed", [(64, 0), (128, 1), (256, 2), (128, 3)])
def test_append_in_any_order(gpu, d, seed):
    """Tokens of a few blocks scattered over the call, slots that come twice, slots past the cache."""
    g = torch.Generator().manual_seed(seed)
    nb, hkv, t = 6, 2, 150
    cache, scales = _old_state(g, nb, hkv, d)
    slots = torch.randint(0, nb * 16, (t,), generator=g)
    slots[::17], slots[5], slots[6], slots[7] = -1, nb * 16, nb * 16 + 40000, 1 << 40
    if seed == 3:
        slots = torch.where(slots % 16 == 0, slots + 1, slots)  # no block is begun
    _append_and_check(gpu, cache, scales, _rows(g, t, hkv, d), _rows(g, t, hkv, d), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_values_without_a_number(gpu, d):
    """Zeros, infinities, NaN, the smallest and the largest bf16, and a block whose scale has to span both."""
    g = torch.Generator().manual_seed(9)
    cache, scales = _old_state(g, 7, 1, d)
    key, value = _rows(g, 40, 1, d), _rows(g, 40, 1, d)
    key[0:16] = 0.0
    key[17, 0, 3], key[18, 0, 4], key[19, 0, d - 1] = float("inf"), float("-inf"), float("nan")
    value[20] = float("nan")
    value[21:32], value[16:20] = 1e-40, 0.0
    key[33], value[34] = torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).min
    key[35], value[36] = torch.finfo(torch.bfloat16).tiny, -torch.finfo(torch.bfloat16).tiny
    _append_and_check(gpu, cache, scales, key, value, torch.arange(40) + 64)
    # alone in their blocks, behind tokens that are there
    _append_and_check(gpu, cache, scales, key[:3], value[16:19], torch.tensor([64 + 5, 80 + 1, 96 + 0]))
    _append_and_check(gpu, cache, scales, key[19:20], value[20:21], torch.tensor([64 + 5]))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 2, 37, 700])
def test_append_of_slots_behind_others(gpu, t):
    """The slots as a view that begins 8 bytes past a multiple of 16, with slots around it that are not the
    call's, the extreme ones of the type among them."""
    from arctic_platform_amd import append_kv

    g = torch.Generator().manual_seed(t)
    nb, hkv, d = t // 16 + 6, 2, 64
    cache, scales = _old_state(g, nb, hkv, d)
    key, value = _rows(g, t, hkv, d), _rows(g, t, hkv, d)
    around = torch.full((t + 2,), 16, dtype=torch.int64)
    around[1:-1] = 23 + torch.arange(t)
    if t > 2:
        around[3], around[4], around[5] = -(2**63), 2**63 - 1, 16 * nb
    slots = around[1:-1]
    want, table = oracle.append_reference(cache, scales, key, value, slots)
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    view = around.to(gpu)[1:-1]
    assert view.data_ptr() % 16 == 8
    append_kv(key.to(gpu), value.to(gpu), dc, view, block_scales=ds)
    torch.cuda.synchronize()
    assert torch.equal(dc.cpu().view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(ds.cpu().nan_to_num(-1.0), table.nan_to_num(-1.0))


@pytest.mark.gpu
def test_append_nothing(gpu):
    from arctic_platform_amd import append_kv

    g = torch.Generator().manual_seed(1)
    cache, scales = _old_state(g, 4, 2, 64)
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    append_kv(none, none, dc, torch.zeros(0, dtype=torch.int64, device=gpu), block_scales=ds)
    one = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    append_kv(one, one, dc, torch.full((3,), -1, dtype=torch.int64, device=gpu), block_scales=ds)
    torch.cuda.synchronize()
    assert torch.equal(dc.cpu().view(torch.uint8), cache.view(torch.uint8))
    assert torch.equal(ds.cpu().view(torch.int32), scales.view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv", [(64, 3), (128, 2), (256, 1)])
def test_gather_reads_back(gpu, d, hkv):
    """Rows of consecutive tokens, of scattered ones, of padding and of slots past the cache, into
    tensors of the call's own and into strided ones; the rows behind them stay as they were."""
    from arctic_platform_amd.cache import gather_kv

    g = torch.Generator().manual_seed(d)
    nb = 9
    cache, scales = _old_state(g, nb, hkv, d)
    scales[:4] = torch.tensor([0.03, 1.5])
    run = torch.randperm(nb, generator=g)[(3 + torch.arange(60)) // 16] * 16 + (3 + torch.arange(60)) % 16
    for slots in (run, torch.randint(-20, nb * 16 + 20, (77,), generator=g), run[:1], torch.tensor([-1]), torch.arange(32)):
        want = oracle.token_rows(cache, scales, slots, d)
        t = len(slots)
        out = torch.full((2, t + 3, hkv, d + 8), 7.0, dtype=torch.bfloat16).to(gpu)
        views = out[0, :t, :, :d], out[1, :t, :, :d]
        args = cache.to(gpu), slots.to(gpu), d
        for got in (gather_kv(*args, block_scales=scales.to(gpu)), gather_kv(*args, out=views, block_scales=scales.to(gpu))):
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b.float().bfloat16())
        assert (out[:, t:] == 7).all() and (out[..., d:] == 7).all()


@pytest.mark.gpu
def test_a_call_longer_than_a_launch(gpu, request):
    """Calls of more than 32768 tokens have the effect of successive calls: a prompt that goes on over
    the cut, the block at the cut begun in front of it and grown behind it."""
    if request.config.getoption("--on-emulation"):
        pytest.skip("tens of thousands of workgroups: not in the emulation")
    from arctic_platform_amd import append_kv
    from arctic_platform_amd.cache import gather_kv

    g = torch.Generator().manual_seed(77)
    t, d, start = 33000, 64, 4
    nb = (start + t + 15) // 16
    slots = torch.randperm(nb, generator=g)[(start + torch.arange(t)) // 16] * 16 + (start + torch.arange(t)) % 16
    key, value = _rows(g, t, 1, d), _rows(g, t, 1, d)
    caches, tables = [], []
    for pieces in ((slice(0, t),), (slice(0, 32768), slice(32768, t))):
        cache = torch.zeros(kv_cache_shape(nb, 16, 1, d), dtype=torch.uint8, device=gpu).view(FP8)
        table = torch.zeros(block_scales_shape(nb, 1), device=gpu)
        for s in pieces:
            append_kv(key[s].to(gpu), value[s].to(gpu), cache, slots[s].to(gpu), block_scales=table)
        caches.append(cache), tables.append(table)
    torch.cuda.synchronize()
    assert torch.equal(caches[0].view(torch.uint8), caches[1].view(torch.uint8)) and torch.equal(*tables)
    near = slice(32768 - 40, 32768 + 40)  # the oracle on the blocks around the cut
    k, v = gather_kv(caches[0], slots[near].to(gpu), d, block_scales=tables[0])
    for got, rows, plane in ((k, key, 0), (v, value, 1)):
        x, y = rows[near].double(), got.cpu().double()
        s = tables[0].cpu()[slots[near] // 16, :, plane : plane + 1].double()
        # a code that moved to a larger scale stays exact or loses half a step of the subnormals once more
        assert ((x - y).abs() <= torch.maximum(x.abs() * 2.0**-4, s * 2.0**-9)).all()


# ---- attention ----------------------------------------------------------------------------------


def _check_attention(out, lse, q, cache, scales, table, row_table, row_lens, scale, what):
    ref, ref_lse, weight, reach = oracle.attention(q, cache, scales, table, row_table, row_lens, scale)
    d = q.shape[2]
    out, lse = out.detach().cpu().double(), lse.detach().cpu().double()
    # Each probability, times its V scale, is rounded to bf16 (half a step, 2^-8); a partial row to
    # half precision (2^-11 of an element at least 2^-14 of the row's largest, 2^-25 of that below);
    # the sums are fp32 (2^-24 a step: up to 32 k terms here would be 2^-9, in practice the terms'
    # roundings average out and tile sums are short, 2^-13 is granted); the output rounds to bf16.
    # The largest element of a row bounds every element's share of the half-precision floor.
    row_max = weight.amax(dim=-1, keepdim=True)
    tol = weight * (2.0**-8 + 2.0**-11 + 2.0**-13) + row_max * 2.0**-20 + ref.abs() * 2.0**-8
    # A score is off by at most (D + 2) 2^-24 of the sum of its products' magnitudes, which moves every
    # probability and the log-sum-exp by as much; exp2 and log2 of the hardware by 2^-22 or so.
    shift = (d + 2) * 2.0**-24 * reach + 2.0**-20
    tol = tol + 2 * shift[..., None] * weight
    assert torch.equal(lse == float("-inf"), ref_lse == float("-inf")), what
    fine = ref_lse > float("-inf")
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((out - ref).abs() / tol.clamp(min=1e-30)).nan_to_num(nan=1e9).max()))
    lse_tol = shift + 2.0**-22 * ref_lse.abs().nan_to_num(posinf=0)
    off = ((lse - ref_lse).abs() / lse_tol)[fine]
    assert (off <= 1).all(), (what, float(off.max()))
    assert (out[~fine] == 0).all(), what


def _random_scales(g, cache, ids, powers):
    """Scales for the blocks in use; NaN for all others."""
    nb, hkv = cache.shape[1:3]
    s = 0.01 + 0.09 * torch.rand(nb, hkv, 2, generator=g)
    if powers:
        s = block_scale_for(s)
    s = s * torch.exp2(torch.randint(-2, 3, s.shape, generator=g).float())
    unused = torch.ones(nb, dtype=torch.bool)
    unused[ids] = False
    s[unused] = float("nan")
    return s.contiguous()


def _used_blocks(table, lens):
    return sorted({int(b) for s, n in enumerate(lens.tolist()) for b in table[s, : (n + 15) // 16].tolist()})


FORESTS = [
    # seed, Hq, Hkv, D, depth, fanout, segment lengths, leaf lengths, chunk, rows
    (1, 8, 2, 128, 2, 3, (1, 90), (1, 60), 64, 32),
    (2, 8, 8, 128, 2, 3, (1, 200), (1, 40), 128, 32),
    (3, 20, 4, 64, 3, 3, (1, 120), (1, 100), 96, 32),
    (4, 16, 2, 64, 2, 6, (10, 200), (1, 50), 128, 64),
    (5, 32, 8, 128, 2, 5, (30, 260), (1, 80), 256, 64),
    (6, 64, 1, 128, 1, 2, (30, 100), (1, 30), 64, 64),
    (7, 16, 2, 256, 2, 3, (1, 150), (1, 60), 64, 32),
    (8, 3, 3, 256, 1, 4, (1, 70), (1, 70), 32, 32),
    (9, 6, 6, 64, 2, 2, (1, 300), (1, 90), 1024, 32),
    (10, 32, 1, 128, 2, 2, (1, 1100), (1, 40), 1024, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORESTS, ids=lambda c: f"seed{c[0]}")
@pytest.mark.parametrize("levels", [4, 0], ids=["forest", "rows-alone"])
def test_attention_on_random_forests(gpu, case, levels):
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    seed, hq, hkv, d, depth, fanout, seg, leaf, chunk, rows = case
    seg_len, paths = random_forest(random.Random(seed), depth, fanout, seg, leaf)
    g = torch.Generator().manual_seed(seed)
    w = make_forest_workload("random", seg_len, paths, g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    lens = w.seq_lens.clone()
    if len(lens) > 3:
        lens[2] = 0  # a sequence that sees nothing
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, lens), powers=seed % 2 == 0)
    md = build_forest_metadata(
        w.block_table.to(gpu), lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=chunk, rows_per_item=rows,
        cascade=levels > 0,
    )
    if seed % 3 == 0:
        md.max_workgroups = 8
    out, lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    md.check()
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(len(lens)), lens.tolist(), w.scale, f"seed {seed}")


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows,lens", [(64, 4, 1, 32, (1030, 0, 17)), (128, 4, 2, 64, (700, 533)), (256, 2, 1, 32, (560,)), (128, 8, 1, 32, (3000, 40, 2049))])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_attention_on_rows_of_many_partials(gpu, d, hq, hkv, rows, lens, out_dtype):
    """Chunks of one tile: rows of up to 94 partials, next to short and empty ones."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    g = torch.Generator().manual_seed(len(lens) + d)
    w = make_forest_workload("long", list(lens), [[i] for i in range(len(lens))], g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=False)
    md = build_forest_metadata(w.block_table.to(gpu), w.seq_lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32, rows_per_item=rows)
    assert md.layout.max_partials >= 16
    wide = torch.full((len(lens), hq, d + 8), 5.0, dtype=out_dtype).to(gpu)
    out, lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, out=wide[..., 4 : d + 4], block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    assert (wide[..., :4] == 5).all() and (wide[..., d + 4 :] == 5).all()
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(len(lens)), list(lens), w.scale, f"lengths {lens}")


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows,n", [(64, 8, 2, 32, 1), (128, 8, 2, 32, 1), (256, 4, 1, 32, 1), (128, 4, 4, 64, 16), (64, 4, 4, 64, 17), (128, 16, 2, 32, 31), (128, 16, 2, 32, 32), (128, 8, 8, 32, 33)])
def test_attention_on_one_short_sequence(gpu, d, hq, hkv, rows, n):
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    g = torch.Generator().manual_seed(n + d)
    w = make_forest_workload("one", [n], [[0]], g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=False)
    md = build_forest_metadata(w.block_table.to(gpu), w.seq_lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32, rows_per_item=rows)
    out, lse = forest_cascade_decode(w.q.to(gpu), w.kv_cache.to(gpu), md, w.scale, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, [0], [n], w.scale, f"{n} tokens")


def _query_runs(g, lens, news, hq, hkv, d, prefix):
    """Sequences that share `prefix` tokens of blocks and bring `news[i]` query tokens each."""
    shared = prefix // 16
    need = [(n + 15) // 16 for n in lens]
    total = shared + sum(max(0, n - shared) for n in need)
    order = torch.randperm(total + 2, generator=g).tolist()
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32), shared
    for s, n in enumerate(need):
        row = order[: min(shared, n)] + order[at : at + max(0, n - shared)]
        at += max(0, n - shared)
        table[s, :n] = torch.tensor(row, dtype=torch.int32)
    nb = total + 2
    k, v = (torch.randn(nb, 16, hkv, d, generator=g).bfloat16() for _ in range(2))
    cache, scales = quantize_blocks(k, v)
    starts = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32)
    q = torch.randn(sum(news), hq, d, generator=g).bfloat16()
    row_table = [s for s, m in enumerate(news) for _ in range(m)]
    row_lens = [lens[s] - (m - 1 - i) for s, m in enumerate(news) for i in range(m)]
    return q, cache, scales, table, starts, row_table, row_lens


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows,levels", [(128, 8, 2, 64, 4), (128, 8, 2, 32, 4), (64, 4, 1, 64, 4), (64, 6, 3, 32, 0), (256, 8, 2, 32, 4)])
def test_attention_of_query_runs(gpu, d, hq, hkv, rows, levels):
    """Verify steps and prefill chunks, runs that end inside blocks and on their ends."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.forest import rows_from_query_runs

    g = torch.Generator().manual_seed(d + rows)
    lens, news = [100, 64, 97, 33, 160, 7], [4, 4, 1, 33, 40, 7]
    q, cache, scales, table, starts, row_table, row_lens = _query_runs(g, lens, news, hq, hkv, d, 48)
    # behind every sequence's last token the cache holds NaN (where no other sequence shares the block)
    raw = cache.view(torch.uint8)
    for s, n in enumerate(lens):
        if n % 16 and n // 16 >= 48 // 16:
            b = int(table[s, n // 16])
            raw[0, b].view(hkv, d // 16, 16, 16)[:, :, n % 16 :] = 0x7F
            raw[1, b].view(hkv, d, 16)[:, :, n % 16 :] = 0x7F
    dev_table, dev_lens = table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu)
    rt, rl, rg = rows_from_query_runs(starts.to(gpu), dev_lens, sum(news), table.shape[1])
    md = build_forest_metadata(
        dev_table, rl, row_table=rt, row_group=rg, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=64, rows_per_item=rows, max_levels=levels,
    )
    scale = d**-0.5
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, scale, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    md.check()
    _check_attention(out, lse, q, cache, scales, table, row_table, row_lens, scale, "query runs")


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(64, 32), (128, 32), (128, 64), (64, 64), (256, 32)])
@pytest.mark.parametrize("plane", [0, 1])
def test_nan_of_a_later_token_stays_with_the_rows_that_see_it(gpu, d, rows, plane):
    """A run of nine query tokens; the key or value of its sixth holds NaN.  The rows before it do not
    see the token, and their outputs are what they are without it; the rows from it on are NaN in
    every channel (key) or in that channel (value)."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.forest import rows_from_query_runs

    hq, hkv, n, new = 4, 2, 44, 9
    g = torch.Generator().manual_seed(d)
    q, cache, scales, table, starts, row_table, row_lens = _query_runs(g, [n], [new], hq, hkv, d, 0)
    clean = cache.clone()
    at, head, channel = n - new + 5, 1, d - 3
    blk, off = int(table[0, at // 16]), at % 16
    if plane == 0:
        cache.view(torch.uint8)[0, blk, head].view(d // 16, 16, 16)[channel // 16, off, channel % 16] = 0xFF
    else:
        cache.view(torch.uint8)[1, blk, head].view(d, 16)[channel, off] = 0x7F
    rt, rl, rg = rows_from_query_runs(starts.to(gpu), torch.tensor([n], dtype=torch.int32).to(gpu), new, table.shape[1])
    md = build_forest_metadata(table.to(gpu), rl, row_table=rt, row_group=rg, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32, rows_per_item=rows)
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, 0.1, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    out, lse = out.cpu(), lse.cpu()
    sees = torch.zeros(new, hq, d, dtype=torch.bool)
    sees[5:, hq // 2 :, slice(None) if plane == 0 else channel] = True
    assert out[sees].isnan().all() and not out[~sees].isnan().any()
    ref, ref_lse, _, _ = oracle.attention(q, clean, scales, table, row_table, row_lens, 0.1)
    keep_out, keep_lse = torch.where(sees, ref.bfloat16(), out), torch.where(lse.isnan(), ref_lse.float(), lse)
    assert torch.equal(lse.isnan(), sees.all(dim=2))
    _check_attention(keep_out, keep_lse, q, clean, scales, table, row_table, row_lens, 0.1, "rows that do not see it")


@pytest.mark.gpu
def test_entry_points_agree(gpu):
    """The separate passes and the merge, the static variant and fp32 outputs, strided q and out."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.ops import forest_cascade_decode_static, forest_pass, merge_partials, prefix_pass, suffix_pass

    seg_len, paths = random_forest(random.Random(31), 2, 4, (20, 200), (1, 60))
    g = torch.Generator().manual_seed(31)
    w = make_forest_workload("random", seg_len, paths, g, num_q_heads=8, num_kv_heads=2, head_dim=128, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=False)
    md = build_forest_metadata(w.block_table.to(gpu), w.seq_lens.to(gpu), num_q_heads=8, num_kv_heads=2, head_dim=128, chunk_tokens=64)
    md.reproducible = True
    q = torch.zeros(w.num_seqs, 12, 128, dtype=torch.bfloat16).to(gpu)
    q[:, 2:10] = w.q.to(gpu)
    args, kw = (q[:, 2:10], w.kv_cache.to(gpu), md, w.scale), dict(block_scales=scales.to(gpu))
    out, lse = forest_cascade_decode(*args, **kw)
    wide = torch.full((w.num_seqs, 10, 136), 5.0, dtype=torch.bfloat16).to(gpu)
    forest_cascade_decode(*args, out=wide[:, 1:9, :128], **kw)
    static, static_lse = torch.zeros_like(out), torch.zeros_like(lse)
    forest_cascade_decode_static(*args, out=static, lse=static_lse, **kw)
    prefix_pass(*args, **kw)
    suffix_pass(*args, **kw)
    parts, parts_lse = merge_partials(md, args[0])
    forest_pass(*args, **kw)
    whole, whole_lse = merge_partials(md, args[0])
    exact, _ = forest_cascade_decode(*args, out_dtype=torch.float32, **kw)
    torch.cuda.synchronize()
    for o, l in ((static, static_lse), (parts, parts_lse), (whole, whole_lse)):
        assert torch.equal(o, out) and torch.equal(l, lse)
    assert torch.equal(wide[:, 1:9, :128], out) and (wide[:, 0] == 5).all() and (wide[..., 128:] == 5).all()
    assert torch.equal(exact.bfloat16(), out)
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(w.num_seqs), w.seq_lens.tolist(), w.scale, "decode")


@pytest.mark.gpu
def test_decode_loop_and_read_back(gpu):
    """A prompt of every sequence written in one call, four decode steps (append, update of the forest,
    attend), then everything read back: each step against the restatement of the writer's cache."""
    from arctic_platform_amd import append_kv, build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.cache import gather_kv

    g = torch.Generator().manual_seed(5)
    hq, hkv, d, nb = 8, 2, 128, 24
    prompts = [29, 47, 16]
    table = torch.randperm(nb, generator=g)[:12].view(3, 4).to(torch.int32)
    cache, scales = _old_state(g, nb, hkv, d)
    dc, ds, dt = cache.clone().to(gpu), scales.clone().to(gpu), table.to(gpu)
    lens = [0, 0, 0]
    md, rows_k, rows_v, all_slots = None, [], [], []
    for step in range(5):
        news = prompts if step == 0 else [1, 1, 1]
        pos = [(s, lens[s] + i) for s, n in enumerate(news) for i in range(n)]
        slots = torch.tensor([int(table[s, p // 16]) * 16 + p % 16 for s, p in pos])
        key, value = _rows(g, len(pos), hkv, d, 0.7), _rows(g, len(pos), hkv, d, 0.7)
        cache, scales = oracle.append_reference(cache, scales, key, value, slots)
        append_kv(key.to(gpu), value.to(gpu), dc, slots.to(gpu), block_scales=ds)
        lens = [n + m for n, m in zip(lens, news)]
        rows_k.append(key), rows_v.append(value), all_slots.append(slots)
        if step == 0:
            continue
        md = build_forest_metadata(dt, torch.tensor(lens, dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32, out=md, update=md is not None)
        q = torch.randn(3, hq, d, generator=g).bfloat16()
        out, lse = forest_cascade_decode(q.to(gpu), dc, md, 0.09, block_scales=ds)
        torch.cuda.synchronize()
        _check_attention(out, lse, q, cache, scales, table, range(3), lens, 0.09, f"step {step}")
    slots = torch.cat(all_slots)
    k, v = gather_kv(dc, slots.to(gpu), d, block_scales=ds)
    torch.cuda.synchronize()
    unset = scales.isnan()  # (of blocks the loop does not touch)
    assert torch.equal(dc.cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(ds.cpu()[~unset], scales[~unset])
    for got, rows, plane in ((k, torch.cat(rows_k), 0), (v, torch.cat(rows_v), 1)):
        x, y, s = rows.double(), got.cpu().double(), scales[slots // 16, :, plane : plane + 1].double()
        # rounded once to e4m3, and where a scale grew, once more below its subnormals (half a step each)
        assert ((x - y).abs() <= torch.maximum(x.abs() * 2.0**-4, s * 2.0**-9)).all()


@pytest.mark.gpu
def test_captured_and_replayed(gpu, request):
    """Append and attention of a decode step recorded into a graph and replayed on new inputs, with eager
    calls between the replays."""
    if request.config.getoption("--on-emulation"):
        pytest.skip("HIP graphs need a GPU")
    from arctic_platform_amd import append_kv, build_forest_metadata, forest_cascade_decode

    g = torch.Generator().manual_seed(8)
    hq, hkv, d, nb, seqs = 8, 2, 128, 40, 6
    cache, scales = quantize_blocks(*(torch.randn(nb, 16, hkv, d, generator=g) for _ in range(2)))
    table = torch.randperm(nb, generator=g)[: seqs * 5].view(seqs, 5).to(torch.int32)
    lens = torch.tensor([17, 80, 33, 64, 5, 48], dtype=torch.int32)
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    key, value, q = (torch.zeros(seqs, n, d, dtype=torch.bfloat16, device=gpu) for n in (hkv, hkv, hq))
    slots = torch.tensor([int(table[s, (n - 1) // 16]) * 16 + (n - 1) % 16 for s, n in enumerate(lens.tolist())])
    dslots = slots.to(gpu)
    md = build_forest_metadata(table.to(gpu), lens.to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=64)
    out = torch.zeros(seqs, hq, d, dtype=torch.bfloat16, device=gpu)

    def step():
        append_kv(key, value, dc, dslots, block_scales=ds)
        return forest_cascade_decode(q, dc, md, 0.09, out=out, block_scales=ds)[1]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    dc.copy_(cache), ds.copy_(scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse = step()
    dc.copy_(cache), ds.copy_(scales)
    for _ in range(4):
        rows = [_rows(g, seqs, n, d, 0.8) for n in (hkv, hkv, hq)]
        for dst, src in zip((key, value, q), rows):
            dst.copy_(src)
        cache, scales = oracle.append_reference(cache, scales, rows[0], rows[1], slots)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dc.cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(ds.cpu(), scales)
        _check_attention(out, lse, rows[2], cache, scales, table, range(seqs), lens.tolist(), 0.09, "replay")
        again, _ = forest_cascade_decode(q, dc, md, 0.09, block_scales=ds)
        torch.cuda.synchronize()
        _check_attention(again, lse, rows[2], cache, scales, table, range(seqs), lens.tolist(), 0.09, "eager between replays")


# ---- refusals (nothing is launched) -------------------------------------------------------------


def test_c_entry_points_refuse_bad_arguments():
    import ctypes
    import os

    from arctic_platform_amd import _lib
    from arctic_platform_amd.forest import make_plan

    if not os.path.exists(_lib.LIB_PATH):
        _lib.build_library()
    lib = _lib.load_library()
    ok = 1 << 20

    def call(fn, key=ok, ts=8 * 128, hs=128, t=3, h=8, d=128, slots=ok, kc=ok, bs=8 * 16 * 128, ch=16 * 128, nb=4, sc=ok):
        return fn(key, ok, ts, hs, t, h, d, slots, kc, ok + (1 << 16), bs, ch, nb, sc, None)

    for fn in (lib.fca_append_kv_block_scaled, lib.fca_gather_kv_block_scaled):
        assert call(fn, t=0) == 0
        for kw, fragment in [
            (dict(t=-1), "num_tokens must be >= 0"), (dict(h=0), "num_kv_heads >= 1"), (dict(d=96), "head_dim 96"),
            (dict(nb=-1), "num_blocks -1"), (dict(nb=1 << 31), "num_blocks"), (dict(key=ok + 8), "16-byte aligned"), (dict(key=None), "non-NULL"),
            (dict(ts=100), "multiples of 8"), (dict(slots=None), "non-NULL"), (dict(sc=None), "non-NULL"), (dict(sc=ok + 4), "8-byte aligned"),
            (dict(kc=ok + 8), "16-byte aligned"), (dict(ch=16 * 64), "at least one tile"), (dict(bs=8 * 16 * 128 + 8), "16-byte-multiple"),
        ]:
            assert call(fn, **kw) < 0
            assert fragment in lib.fca_last_error().decode(), (kw, lib.fca_last_error())
    plan = make_plan(4, 8, 32, 8, 128)

    def decode(**kw):
        t = _lib.FcaTensors(ok, 32 * 128, 128, ok, ok + (1 << 16), 8 * 16 * 128, 16 * 128, _lib.FCA_FP8_E4M3_BLOCK, 0, ok, 8, ok, None, 0.1)
        for k, v in kw.items():
            setattr(t, k, v)
        # (no metadata: a call whose tensors pass still stops before a launch)
        return lib.fca_decode_step(ctypes.byref(plan), ctypes.byref(t), None, ok, ok, ok, 32 * 128, 128, _lib.FCA_BF16, None, None)

    for kw, fragment in [
        (dict(), "metadata and partial workspaces"), (dict(k_scale_dev=None), "scale table"), (dict(k_scale_dev=ok + 4), "scale table"),
        (dict(v_scale_dev=ok), "no v_scale"), (dict(softmax_scale=0.0), "softmax_scale"), (dict(tile_buffers=3), "tile_buffers 3"),
        (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(kv_head_stride=16 * 64), "smaller than one tile"),
    ]:
        assert decode(**kw) < 0
        assert fragment in lib.fca_last_error().decode(), (kw, lib.fca_last_error())


@pytest.mark.gpu
def test_python_entry_points_refuse_bad_arguments(gpu):
    from arctic_platform_amd import append_kv, build_forest_metadata, forest_cascade_decode
    from arctic_platform_amd.cache import gather_kv

    cache = torch.zeros(kv_cache_shape(6, 16, 2, 128), dtype=torch.uint8).view(FP8).to(gpu)
    scales = torch.ones(block_scales_shape(6, 2)).to(gpu)
    rows = torch.zeros(3, 2, 128, dtype=torch.bfloat16).to(gpu)
    slots = torch.zeros(3, dtype=torch.int64).to(gpu)
    per_head = torch.ones(2).to(gpu)
    md = build_forest_metadata(torch.zeros(1, 2, dtype=torch.int32).to(gpu), torch.tensor([20], dtype=torch.int32).to(gpu), num_q_heads=4, num_kv_heads=2, head_dim=128)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16).to(gpu)
    bf16 = torch.zeros(kv_cache_shape(6, 16, 2, 128), dtype=torch.bfloat16).to(gpu)
    for bad, error in (
        (dict(block_scales=scales[:5]), ValueError), (dict(block_scales=scales.double()), ValueError), (dict(block_scales=scales.transpose(1, 2)), ValueError),
        (dict(block_scales=torch.ones(6, 2, 4).to(gpu)[..., ::2]), ValueError), (dict(block_scales=scales, k_scale=per_head), ValueError),
        (dict(block_scales=scales, v_scale=per_head), ValueError),
    ):
        for call in (
            lambda **kw: append_kv(rows, rows, cache, slots, **kw),
            lambda **kw: gather_kv(cache, slots, 128, **kw),
            lambda **kw: forest_cascade_decode(q, cache, md, 0.1, **kw),
        ):
            with pytest.raises(error):
                call(**bad)
    for call in (
        lambda: append_kv(rows, rows, bf16, slots, block_scales=scales), lambda: gather_kv(bf16, slots, 128, block_scales=scales),
        lambda: forest_cascade_decode(q, bf16, md, 0.1, block_scales=scales), lambda: append_kv(rows.float(), rows.float(), cache, slots, block_scales=scales),
    ):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        forest_cascade_decode(q, cache, md, 0.0, block_scales=scales)
    torch.cuda.synchronize()
    assert (cache.cpu().view(torch.uint8) == 0).all()
