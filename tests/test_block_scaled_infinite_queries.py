"""Query rows whose scores are all minus infinity: their softmax is no number, wherever the sequence ends."""

import pytest
import torch

from arctic_platform_amd.kv_layout import quantize_blocks
from oracle import block_scales as oracle


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32)])
def test_scores_of_minus_infinity(gpu, d, rows):
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    hq, hkv, lens = 4, 1, [1, 17, 31, 32, 40, 70, 0]
    g = torch.Generator().manual_seed(d)
    nb = sum((n + 15) // 16 for n in lens)
    k, v = torch.randn(nb, 16, hkv, d, generator=g), torch.randn(nb, 16, hkv, d, generator=g)
    k[..., 0] = k[..., 0].abs() + 1  # minus infinity times these: every score is minus infinity
    cache, scales = quantize_blocks(k, v)
    table, at = torch.zeros(len(lens), 5, dtype=torch.int32), 0
    for s, n in enumerate(lens):
        need = (n + 15) // 16
        table[s, :need] = torch.arange(at, at + need, dtype=torch.int32)
        at += need
    q = torch.randn(len(lens), hq, d, generator=g)
    q[:, 1, 0] = float("-inf")
    q[:, 2, 3] = float("nan")
    q = q.bfloat16()
    md = build_forest_metadata(table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=32, rows_per_item=rows)
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, 0.1, block_scales=scales.to(gpu))
    torch.cuda.synchronize()
    ref, ref_lse, _, _ = oracle.attention(q, cache, scales, table, range(len(lens)), lens, 0.1)
    assert ref[:-1, 1:3].isnan().all() and not ref[:, 0].isnan().any()
    assert torch.equal(out.cpu().isnan(), ref.isnan()) and torch.equal(lse.cpu().isnan(), ref_lse.isnan())
    assert (out[-1].cpu() == 0).all() and (lse[-1].cpu() == float("-inf")).all()
