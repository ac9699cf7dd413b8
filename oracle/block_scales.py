"""CPU restatement, in 64 bits, of the KV cache held in 8 bits with a scale per block: writing with
scales taken from the data, reading back, and attention over it.

The reference holds none of this (the engine that owns the paged cache is external,
arctic_platform/common/ray_server.py:395-404; the cache dtype it forwards is
common/utils/server_models.py:143-165); the layout and the rule for the scales are this build's
own, so the expected bytes follow from their definition and the writer is checked bit for bit.
"""

from __future__ import annotations

import math

import torch

BLOCK = 16
FP8_MAX = 448.0


def _e4m3_values():
    out = []
    for code in range(0x7F):
        e, m = code >> 3, code & 7
        out.append(m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


VALUES = _e4m3_values()  # of the codes 0 .. 0x7e, ascending


def decode(codes):
    """Bytes -> float64 values (0x7f and 0xff are NaN)."""
    c = codes.long()
    v = torch.cat([VALUES, torch.tensor([math.nan], dtype=torch.float64)])[c & 0x7F]
    return torch.where(c >= 128, -v, v)


def encode(x):
    """float64 values -> bytes: nearest, ties to the even code, saturating; NaN becomes 0x7f."""
    a = x.abs().clamp(max=FP8_MAX)
    a = torch.where(x.isnan(), torch.zeros_like(a), a)
    hi = torch.searchsorted(VALUES, a).clamp(max=0x7E)  # first value >= a
    lo = (hi - 1).clamp(min=0)
    up, down = VALUES[hi] - a, a - VALUES[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(torch.signbit(x), code + 128, code)
    return torch.where(x.isnan(), torch.full_like(code, 0x7F), code).to(torch.uint8)


def scale_for(amax: float) -> float:
    """Smallest power of two s with amax <= 448 s, within [2^-100, 2^120]."""
    s = 2.0**-100
    while amax > FP8_MAX * s and s < 2.0**120:
        s *= 2
    return s


def append_reference(kv_cache, scales, key, value, slot_mapping):
    """Returns (cache, scales) after the write.  Element offsets come straight from the layout."""
    nb, hkv = scales.shape[:2]
    d = key.shape[2]
    raw, table = kv_cache.clone().view(torch.uint8), scales.double().clone()
    blocks: dict = {}
    for t, slot in enumerate(slot_mapping.tolist()):
        if 0 <= slot < nb * BLOCK:
            blocks.setdefault(slot // BLOCK, {})[slot % BLOCK] = t  # a later token replaces an earlier one
    for blk, tokens in blocks.items():
        offs = sorted(tokens)
        idx = [tokens[o] for o in offs]
        for plane, rows in ((0, key), (1, value)):
            for h in range(hkv):
                x = rows[idx, h].double().cpu()
                finite = x.abs()[torch.isfinite(x)]
                new = scale_for(float(finite.max()) if finite.numel() else 0.0)
                old = float(table[blk, h, plane])
                known = 0 not in tokens and old > 0 and math.isfinite(old)
                if known:
                    p2 = 2.0**-100
                    while p2 < old and p2 < 2.0**120:
                        p2 *= 2
                    new = max(new, p2)
                tile = raw[plane, blk, h].view(d // 16, BLOCK, 16) if plane == 0 else raw[plane, blk, h].view(d, BLOCK)
                rest = [o for o in range(BLOCK) if o not in tokens]
                if known and new != old and rest:
                    if plane == 0:
                        tile[:, rest] = encode(decode(tile[:, rest]) * (old / new))
                    else:
                        tile[:, rest] = encode(decode(tile[:, rest]) * (old / new))
                codes = encode(x / new)
                if plane == 0:
                    tile[:, offs] = codes.view(len(offs), d // 16, 16).permute(1, 0, 2)
                else:
                    tile[:, offs] = codes.t()
                table[blk, h, plane] = new
    return raw.view(torch.float8_e4m3fn), table.float()


def token_rows(kv_cache, scales, slots, d):
    """float64 (key, value) rows [T, Hkv, D] of the tokens at ``slots`` (zeros where there is none)."""
    nb, hkv = scales.shape[:2]
    raw = kv_cache.cpu().view(torch.uint8)
    k = torch.zeros(len(slots), hkv, d, dtype=torch.float64)
    v = torch.zeros_like(k)
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < nb * BLOCK:
            continue
        blk, off = divmod(slot, BLOCK)
        sc = scales[blk].double().cpu()
        k[t] = decode(raw[0, blk].view(hkv, d // 16, BLOCK, 16)[:, :, off].reshape(hkv, d)) * sc[:, 0:1]
        v[t] = decode(raw[1, blk].view(hkv, d, BLOCK)[:, :, off]) * sc[:, 1:2]
    return k, v


def attention(q, kv_cache, scales, block_table, row_table, row_lens, softmax_scale):
    """Row r attends to the first ``row_lens[r]`` tokens of table row ``row_table[r]``.

    Returns (out, lse, weight, reach): ``weight`` = sum of p |v| per output and ``reach`` = the
    largest softmax_scale * sum |q| |k| of the row, which error bounds are made of."""
    rows, hq, d = q.shape
    hkv = scales.shape[1]
    g = hq // hkv
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    weight = torch.zeros_like(out)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(rows, hq, dtype=torch.float64)
    table, raw, sc = block_table.cpu(), kv_cache.cpu().view(torch.uint8), scales.cpu().double()
    kept: dict = {}
    for r in range(rows):
        seq, n = int(row_table[r]), int(row_lens[r])
        if n == 0:
            continue
        if seq not in kept:
            longest = max(int(row_lens[i]) for i in range(rows) if int(row_table[i]) == seq)
            ids = table[seq, : (longest + BLOCK - 1) // BLOCK].long()
            k = decode(raw[0, ids]).view(-1, hkv, d // 16, BLOCK, 16).permute(1, 0, 3, 2, 4).reshape(hkv, -1, BLOCK, d)
            v = decode(raw[1, ids]).view(-1, hkv, d, BLOCK).permute(1, 0, 3, 2)
            k = (k * sc[ids, :, 0].t()[..., None, None]).reshape(hkv, -1, d)
            v = (v * sc[ids, :, 1].t()[..., None, None]).reshape(hkv, -1, d)
            kept[seq] = k, v
        k, v = (x[:, :n] for x in kept[seq])
        qq = q[r].double().cpu().view(hkv, g, d)
        s = torch.einsum("hgd,htd->hgt", qq, k) * softmax_scale
        reach[r] = (torch.einsum("hgd,htd->hgt", qq.abs(), k.abs()) * abs(softmax_scale)).amax(dim=-1).reshape(hq)
        top = s.amax(dim=-1, keepdim=True)
        e = torch.exp(s - top)
        total = e.sum(dim=-1, keepdim=True)
        p = e / total
        out[r] = torch.einsum("hgt,htd->hgd", p, v).reshape(hq, d)
        weight[r] = torch.einsum("hgt,htd->hgd", p, v.abs()).reshape(hq, d)
        lse[r] = (top + total.log()).reshape(hq)
    return out, lse, weight, reach
