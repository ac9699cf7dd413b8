"""How near attention over the block-scaled cache comes to its definition in 64 bits: fp32 outputs, so that
no rounding of the output hides what happens before it."""

import pytest
import torch

from arctic_platform_amd.kv_layout import quantize_blocks
from oracle import block_scales as oracle


def _batch(g, lens, hq, hkv, d, spread):
    """Sequences of their own; the magnitude of the values changes by powers of e^spread from block to block."""
    need = [(n + 15) // 16 for n in lens]
    order = torch.randperm(sum(need) + 2, generator=g).tolist()
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    k, v = (torch.randn(len(order), 16, hkv, d, generator=g) for _ in range(2))
    v = v * torch.exp(spread * torch.randn(len(order), 1, hkv, 1, generator=g))
    return torch.randn(len(lens), hq, d, generator=g).bfloat16(), *quantize_blocks(k, v), table


def _check(out, lse, q, cache, scales, table, lens, scale):
    """out [rows, Hq, D] fp32 against the definition.

    A weight p s_v is a half: half a step, 2^-11 of it (a weight below 2^-21 of the row's largest is
    off by up to 2^-32 of that largest instead, times a code of at most 448: under 2^-23 of the largest
    p s_v 448 a token); a partial row is halves too: 2^-11 of an element (of one below 2^-14 of the row's
    largest, 2^-25 of that).  Their sums are fp32: the terms of a tile are added in one or two
    instructions, 2^-24 a step and 64 tiles at most here, 2^-18 granted.  A score is off by at most
    (D + 2) 2^-24 of the sum of its products' magnitudes, which moves every probability by as much;
    exp2 and log2 of the hardware by 2^-22 or so."""
    ref, ref_lse, weight, reach = oracle.attention(q, cache, scales, table, range(len(lens)), lens, scale)
    d = q.shape[2]
    out, lse = out.detach().cpu().double(), lse.detach().cpu().double()
    shift = (d + 2) * 2.0**-24 * reach + 2.0**-20
    row_max = weight.amax(dim=-1, keepdim=True)
    tol = weight * (2 * 2.0**-11 + 2.0**-18 + 2 * shift[..., None]) + row_max * 2.0**-20
    off = (out - ref).abs() / tol
    assert (off <= 1).all(), (int((off > 1).sum()), float(off.max()))
    assert ((lse - ref_lse).abs() <= shift + 2.0**-22 * ref_lse.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rows", [(64, 8, 2, 32), (64, 4, 1, 64), (128, 8, 2, 32), (128, 4, 1, 64), (256, 4, 1, 32)])
@pytest.mark.parametrize("spread", [0.0, 2.0, 12.0], ids=["even", "uneven", "far-apart"])
def test_weights_keep_eleven_bits(gpu, d, hq, hkv, rows, spread):
    """Short sequences, where a rounded weight shows in the output undiluted, and one of several chunks."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    g = torch.Generator().manual_seed(d + rows)
    lens, scale = [2, 3, 5, 18, 33, 300], d**-0.5
    q, cache, scales, table = _batch(g, lens, hq, hkv, d, spread)
    md = build_forest_metadata(
        table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=128, rows_per_item=rows
    )
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, scale, block_scales=scales.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check(out, lse, q, cache, scales, table, lens, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32)])
@pytest.mark.parametrize("power", [-90, 0, 110])
def test_value_scales_at_the_ends_of_their_range(gpu, d, rows, power):
    """Values of a whole cache around 2^power, blocks a thousandth and a thousand times that among them, and
    scores that make the block with the small scale the one that counts in some rows."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    hq, hkv, scale = 4, 2, 1.5 * d**-0.5
    g = torch.Generator().manual_seed(d + rows + power)
    lens = [40, 100, 17]
    q, cache, scales, table = _batch(g, lens, hq, hkv, d, 0.0)
    step = torch.randint(-1, 2, scales[..., 1].shape, generator=g) * (5 if power else 10)
    scales[..., 1] = scales[..., 1] * torch.exp2((step + power).float())
    md = build_forest_metadata(
        table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=64, rows_per_item=rows
    )
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, scale, block_scales=scales.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check(out, lse, q, cache, scales, table, lens, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(128, 32), (128, 64), (256, 32)])
def test_many_small_weights_beside_a_large_one(gpu, d, rows):
    """One token takes most of the probability and 1023 share the rest, each about 2^-26 of it: their values,
    2^12 times as large, carry a part of the output that must not get lost."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    hq, hkv, n, scale = 4, 1, 1024, 1.0
    g = torch.Generator().manual_seed(d)
    k = torch.zeros(n // 16, 16, hkv, d)
    k[0, 0, 0, 0] = 18.0  # (an e4m3 value; the score of the first token: 18, of the others: 0)
    v = torch.randn(n // 16, 16, hkv, d, generator=g)
    v[1:] = v[1:].abs() * 4096
    cache, scales = quantize_blocks(k, v)
    table = torch.arange(n // 16, dtype=torch.int32).view(1, -1)
    q = torch.zeros(1, hq, d)
    q[..., 0] = 1.0
    q = q.bfloat16()
    md = build_forest_metadata(table.to(gpu), torch.tensor([n], dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=1024, rows_per_item=rows)
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, scale, block_scales=scales.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check(out, lse, q, cache, scales, table, [n], scale)


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32)])
@pytest.mark.parametrize("power", [20, 24, 27, 29])
def test_scores_far_beyond_their_rounding(gpu, d, rows, power):
    """Scores of about 2^power, exact by construction and the same for three tokens of a sequence (one in each of three
    blocks, their V scales far apart), half as large for the others: the output is the mean of three rows."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    hq, hkv, n = 4, 1, 150
    g = torch.Generator().manual_seed(d + power)
    nb = (n + 15) // 16
    k, v = torch.zeros(nb, 16, hkv, d), torch.randn(nb, 16, hkv, d, generator=g)
    k[:, :, :, 0], top = 0.5, [5, 70, 145]
    for t in top:
        k[t // 16, t % 16, :, 0] = 1.0
    v = v * torch.exp2(torch.randint(-30, 31, (nb, 1, 1, 1), generator=g).float())
    cache, scales = quantize_blocks(k, v)
    scales[..., 0], raw = 2.0**-8, cache.view(torch.uint8)[0].view(nb, hkv, d // 16, 16, 16)
    raw[:, :, 0, :, 0] = torch.tensor([0.5, 1.0]).mul(256).to(torch.float8_e4m3fn).view(torch.uint8)[(k[:, :, 0, 0] == 1).long()][:, None]
    table = torch.arange(nb, dtype=torch.int32).view(1, -1)
    q = torch.zeros(1, hq, d)
    q[..., 0] = 1.1015625 * 2.0**power  # (a bf16 number)
    md = build_forest_metadata(table.to(gpu), torch.tensor([n], dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=64, rows_per_item=rows)
    out, lse = forest_cascade_decode(q.bfloat16().to(gpu), cache.to(gpu), md, 1.0, block_scales=scales.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    values = oracle.token_rows(cache, scales, torch.tensor(top), d)[1][:, 0]
    want, weight = values.mean(dim=0), values.abs().mean(dim=0)
    # a third each, exactly (but for 2^-22 of exp2); weights and partial rows are halves, 2^-11 of each
    tol = weight * (2 * 2.0**-11 + 2.0**-18) + weight.max() * 2.0**-20
    assert ((out.cpu().double()[0] - want).abs() <= tol).all()
    assert ((lse.cpu().double() - 1.1015625 * 2.0**power).abs() <= 2.0 ** (power - 22) + 2).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32)])
def test_value_scales_beyond_the_writers(gpu, d, rows):
    """A table of somebody else's: V scales of 2^120 to 2^125 on codes small enough that every value is finite."""
    from arctic_platform_amd import build_forest_metadata, forest_cascade_decode

    hq, hkv, lens, scale = 4, 2, [40, 100, 3], d**-0.5
    g = torch.Generator().manual_seed(d + rows)
    q, cache, scales, table = _batch(g, lens, hq, hkv, d, 0.0)
    raw = cache.view(torch.uint8)
    raw[1] = torch.randint(0x08, 0x41, raw[1].shape, generator=g, dtype=torch.uint8) | (raw[1] & 0x80)  # magnitudes of 2^-6 to 2.25
    scales[..., 1] = torch.exp2(torch.randint(120, 126, scales.shape[:2], generator=g).float())
    md = build_forest_metadata(
        table.to(gpu), torch.tensor(lens, dtype=torch.int32).to(gpu), num_q_heads=hq, num_kv_heads=hkv, head_dim=d, chunk_tokens=64, rows_per_item=rows
    )
    out, lse = forest_cascade_decode(q.to(gpu), cache.to(gpu), md, scale, block_scales=scales.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check(out, lse, q, cache, scales, table, lens, scale)
