"""The attention backend on a block-scaled 8-bit cache (``kv_cache_dtype="fp8_block"``): its own append,
attention and read-back of a cached context, on the step's K and V, against the 64-bit restatement."""

import types

import pytest
import torch

from arctic_platform_amd.backend import CommonAttentionMetadata, ForestCascadeAttentionBackend
from arctic_platform_amd.config import build_model_config
from arctic_platform_amd.kv_layout import kv_cache_shape
from oracle import block_scales as oracle
from tests.test_block_scaled_cache import _check_attention

FP8 = torch.float8_e4m3fn


def test_dtype_and_table_shape():
    cfg = build_model_config("m", {"kv_cache_dtype": "fp8_block"}, {"zorro_inference": {"enable": True}})
    assert cfg.use_fca and cfg.kv_cache_dtype == "fp8_block"
    with pytest.raises(ValueError, match="fp8_blocks"):
        build_model_config("m", {"kv_cache_dtype": "fp8_blocks"}, {"zorro_inference": {"enable": True}})
    assert tuple(ForestCascadeAttentionBackend.get_kv_block_scales_shape(7, 4)) == (7, 4, 2)


def test_layer_without_a_table_is_refused():
    impl = ForestCascadeAttentionBackend.get_impl_cls()(8, 128, 0.1, 2, kv_cache_dtype="fp8_block")
    rows = torch.zeros(1, 8 * 128, dtype=torch.bfloat16)
    meta = types.SimpleNamespace(num_decode_tokens=1)
    with pytest.raises(ValueError, match="kv_block_scales"):
        impl.forward(types.SimpleNamespace(k_scale=None), rows, rows[:, :256], rows[:, :256], None, meta)


def _common(gpu, table, q_lens, s_lens, slots):
    starts = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    lens = torch.tensor(s_lens, dtype=torch.int32)
    return CommonAttentionMetadata(
        query_start_loc=starts.to(gpu), seq_lens=lens.to(gpu), block_table_tensor=table.to(gpu), slot_mapping=slots.to(gpu),
        num_reqs=len(q_lens), max_query_len=max(q_lens), num_actual_tokens=sum(q_lens), query_start_loc_cpu=starts, seq_lens_cpu=lens,
    )


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 8, 64), (6, 2, 256)])
def test_steps_through_the_backend(gpu, hq, hkv, d):
    """Six requests, two of them behind a cached block of another one, through one layer: short prompts, decode
    steps, a verify step of four tokens each, decodes mixed with a prefill chunk.  The layer also has
    per-head scales, which do not apply."""
    g = torch.Generator().manual_seed(d)
    scale, seqs, width = d**-0.5, 6, 10
    table = torch.randperm(seqs * width + 5, generator=g)[: seqs * width].view(seqs, width).to(torch.int32)
    table[4, :2] = table[5, :2] = table[0, :2]
    cache = torch.randn(kv_cache_shape(seqs * width + 5, 16, hkv, d), generator=g).to(FP8)
    scales = torch.full((seqs * width + 5, hkv, 2), float("nan"))
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    layer = types.SimpleNamespace(k_scale=torch.full((hkv,), 3.0, device=gpu), v_scale=torch.full((hkv,), 5.0, device=gpu), kv_block_scales=ds)
    builder = ForestCascadeAttentionBackend.get_builder_cls()(hq, hkv, d, device=gpu, forest_cascade_attn_configs='{"chunk_tokens": 64}')
    impl = ForestCascadeAttentionBackend.get_impl_cls()(hq, d, scale, hkv, kv_cache_dtype="fp8_block")
    lens = [0, 0, 0, 0, 0, 0]
    for step, q_lens in enumerate(([40, 17, 1, 3, 0, 0], [1, 1, 1, 1, 5, 1], [1] * 6, [4] * 6, [1, 1, 1, 1, 1, 30])):
        if step == 1:
            lens[4] = lens[5] = 32  # (the cached prompt of request 0)
        # requests without a token are not part of the step
        active = [s for s in range(seqs) if q_lens[s] > 0]
        news = [q_lens[s] for s in active]
        pos = [(i, s, lens[s] + j) for i, s in enumerate(active) for j in range(q_lens[s])]
        for s in active:
            lens[s] += q_lens[s]
        slots = torch.tensor([int(table[s, p // 16]) * 16 + p % 16 for _, s, p in pos])
        q, k, v = ((torch.randn(len(pos), h * d, generator=g) * (0.4 + step)).bfloat16() for h in (hq, hkv, hkv))
        cache, scales = oracle.append_reference(cache, scales, k.view(-1, hkv, d), v.view(-1, hkv, d), slots)
        meta = builder.build(0, _common(gpu, table[active], news, [lens[s] for s in active], slots))
        out = impl.forward(layer, q.to(gpu), k.to(gpu), v.to(gpu), dc, meta)
        torch.cuda.synchronize()
        if meta.forest is not None:
            meta.forest.check()
        assert torch.equal(dc.cpu().view(torch.uint8), cache.view(torch.uint8)), f"step {step}"
        assert torch.equal(ds.cpu().nan_to_num(-1.0), scales.nan_to_num(-1.0)), f"step {step}"
        row_seqs, row_lens = [s for _, s, _ in pos], [p + 1 for _, _, p in pos]
        _, lse, _, _ = oracle.attention(q.view(-1, hq, d), cache, scales, table, row_seqs, row_lens, scale)
        _check_attention(
            out.view(-1, hq, d), lse.float(), q.view(-1, hq, d), cache, scales, table, row_seqs, row_lens, scale, f"step {step}"
        )


@pytest.mark.gpu
def test_long_chunk_behind_a_cached_context(gpu):
    """Decodes, a long chunk behind 130 cached tokens, a fresh prompt: K and V of the two prompts are read back
    from the cache just written (context included) for the split-attention kernels."""
    hq, hkv, d = 8, 2, 128
    scale = d**-0.5
    g = torch.Generator().manual_seed(31)
    q_lens, s_lens, width = [1, 1, 600, 300], [50, 17, 730, 300], 48
    table = torch.randperm(4 * width, generator=g).view(4, width).to(torch.int32)
    cache = torch.randn(kv_cache_shape(4 * width, 16, hkv, d), generator=g).to(FP8)
    scales = torch.exp2(torch.randint(-3, 2, (4 * width, hkv, 2), generator=g).float())
    dc, ds = cache.clone().to(gpu), scales.clone().to(gpu)
    pos = [(s, p) for s in range(4) for p in range(s_lens[s] - q_lens[s], s_lens[s])]
    slots = torch.tensor([int(table[s, p // 16]) * 16 + p % 16 for s, p in pos])
    q, k, v = (torch.randn(len(pos), h * d, generator=g).bfloat16() for h in (hq, hkv, hkv))
    builder = ForestCascadeAttentionBackend.get_builder_cls()(hq, hkv, d, device=gpu)
    impl = ForestCascadeAttentionBackend.get_impl_cls()(hq, d, scale, hkv, kv_cache_dtype="fp8_block")
    meta = builder.build(0, _common(gpu, table, q_lens, s_lens, slots))
    assert meta.fresh_start == 2 and meta.context_slots.numel() == 730 + 300
    out = impl.forward(types.SimpleNamespace(kv_block_scales=ds), q.to(gpu), k.to(gpu), v.to(gpu), dc, meta)
    torch.cuda.synchronize()
    cache, scales = oracle.append_reference(cache, scales, k.view(-1, hkv, d), v.view(-1, hkv, d), slots)
    assert torch.equal(dc.cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(ds.cpu(), scales)
    ref, _, weight, reach = oracle.attention(
        q.view(-1, hq, d), cache, scales, table, [s for s, _ in pos], [p + 1 for _, p in pos], scale
    )
    # Probabilities rounded to bf16 (2^-8), the output rounded to bf16 (2^-8), the fp32 score's and sums'
    # roundings as in the decode test; the split kernels' half-precision partials are not involved, their
    # terms are granted all the same.
    row_max = weight.amax(dim=-1, keepdim=True)
    shift = (d + 2) * 2.0**-24 * reach + 2.0**-20
    tol = weight * (2.0**-8 + 2.0**-11 + 2.0**-13 + 2 * shift[..., None]) + row_max * 2.0**-20 + ref.abs() * 2.0**-8
    bad = (out.view(-1, hq, d).cpu().double() - ref).abs() > tol
    assert not bad.any(), int(bad.sum())


@pytest.mark.gpu
def test_two_streams_at_once(gpu, request):
    """Two decode loops on streams of their own, neither the current stream of the thread that waits: each
    has its cache, table and metadata, and both are in flight together."""
    if request.config.getoption("--on-emulation"):
        pytest.skip("streams need a GPU")
    from arctic_platform_amd import append_kv, build_forest_metadata, forest_cascade_decode

    hq, hkv, d, seqs, steps = 8, 2, 128, 4, 6
    loops = []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        table = torch.randperm(40, generator=g)[:24].view(seqs, 6).to(torch.int32)
        rows = torch.randn(steps, 3, seqs, hq, d, generator=g).bfloat16()
        cache = torch.zeros(kv_cache_shape(40, 16, hkv, d)).to(FP8)
        scales = torch.ones(40, hkv, 2)
        slots = torch.tensor([[int(table[s, 0]) * 16 + i for s in range(seqs)] for i in range(steps)])
        on_gpu = [x.to(gpu) for x in (table, rows, cache.clone(), scales.clone(), slots)]
        loops.append((table, rows, cache, scales, slots, on_gpu, torch.cuda.Stream(), []))
    lens = [torch.full((seqs,), i + 1, dtype=torch.int32).to(gpu) for i in range(steps)]
    torch.cuda.synchronize()
    for i in range(steps):
        for *_, (table, rows, cache, scales, slots), stream, outs in loops:
            with torch.cuda.stream(stream):
                k, v = rows[i, 1, :, :hkv], rows[i, 2, :, :hkv]
                append_kv(k, v, cache, slots[i], block_scales=scales)
                md = build_forest_metadata(table, lens[i], num_q_heads=hq, num_kv_heads=hkv, head_dim=d)
                outs.append((md, *forest_cascade_decode(rows[i, 0], cache, md, 0.1, block_scales=scales)))
    torch.cuda.synchronize()
    for table, rows, cache, scales, slots, on_gpu, _, outs in loops:
        for i in range(steps):
            cache, scales = oracle.append_reference(cache, scales, rows[i, 1, :, :hkv], rows[i, 2, :, :hkv], slots[i])
            _check_attention(outs[i][1], outs[i][2], rows[i, 0], cache, scales, table, range(seqs), [i + 1] * seqs, 0.1, f"step {i}")
        assert torch.equal(on_gpu[2].cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(on_gpu[3].cpu(), scales)
