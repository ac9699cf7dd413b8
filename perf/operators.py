"""What is measured of the paged cache held in 8 bits with one scale per block, KV head and plane.

The cache is the framework's own: ``[2, num_blocks, Hkv, 16 * D]`` float8_e4m3fn (plane 0 = K in
tiles ``[D / 16, 16 tokens, 16]``, plane 1 = V in tiles ``[D, 16 tokens]``), with a scale table
``[num_blocks, Hkv, 2]`` (fp32; K's, V's) beside it: a stored code stands for code * scale.

Three operators:

* ``append``: the new tokens of a step are quantised as they are written.  A block's scale is the
  smallest power of two s with amax <= 448 s over the tokens of the call, or the scale the block
  has, where that is larger; a token at offset 0 begins the block (what it held before is
  forgotten); where the scale of a block grows, the codes of its earlier tokens are rescaled.
* ``gather``: tokens are read back as bf16 rows.
* ``attend``: softmax attention of one query row per (sequence, query token) over such a cache,
  sequences sharing the blocks of common prompts; output and log-sum-exp.

Cases name their sizes; sequence lengths follow from the case alone, values and the places of
blocks from the seed.
"""

import math
import random

import torch

own = False  # False: the plain forms below; True: the framework's operators

BLOCK = 16
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
SCALE_LOW, SCALE_HIGH = -100, 120  # powers of two a block scale lies between
NAN_CODE = 0x7F


# ---- cases ---------------------------------------------------------------------------------------


def listed():
    return [
        # the decode step of a small batch: one new token for each of 8 sequences, most of them in
        # the middle of a block (latency)
        dict(name="append_8_decode", op="append", seqs=8, new=1, ctx=700, hkv=8, d=128, pad=0),
        # the decode step of a full rollout batch
        dict(name="append_512_decode", op="append", seqs=512, new=1, ctx=2000, hkv=8, d=128, pad=0),
        # a long prompt written in one call, starting inside a block, padded batch
        dict(name="append_prompt_8191", op="append", seqs=1, new=8191, ctx=5, hkv=8, d=128, pad=9),
        # a short cached context read back for a prefill chunk, small heads, ragged
        dict(name="gather_257", op="gather", seqs=1, ctx=257, hkv=2, d=64, pad=0),
        # long contexts read back for the chunks of eight requests
        dict(name="gather_8x4093", op="gather", seqs=8, ctx=4093, hkv=8, d=128, pad=0),
        # one short sequence: the smallest decode step (latency)
        dict(name="attend_1x300", op="attend", groups=1, samples=1, prefix=0, suffix=300, new=1, hq=32, hkv=8, d=128, rows=32, chunk=64),
        # one very long sequence: few rows, work split along the cache
        dict(name="attend_1x131071", op="attend", groups=1, samples=1, prefix=0, suffix=131071, new=1, hq=32, hkv=8, d=128, rows=32, chunk=1024),
        # sequences of their own, small heads
        dict(name="attend_48_own_d64", op="attend", groups=48, samples=1, prefix=0, suffix=2500, new=1, hq=8, hkv=2, d=64, rows=32, chunk=256),
        # the rollout batch: 64 prompts of 1024 to 4096 tokens, 8 samples each
        dict(name="attend_64x8", op="attend", groups=64, samples=8, prefix=2560, suffix=512, new=1, hq=32, hkv=8, d=128, rows=32, chunk=1024),
        # long prompts with many samples each: 64-row tiles
        dict(name="attend_8x16_prompt_32768", op="attend", groups=8, samples=16, prefix=32768, suffix=2176, new=1, hq=32, hkv=8, d=128, rows=64, chunk=1024),
        # the verify step of speculative decoding: four query tokens per sequence
        dict(name="attend_verify_16x6", op="attend", groups=16, samples=6, prefix=1500, suffix=400, new=4, hq=32, hkv=8, d=128, rows=64, chunk=512),
        # large heads, few KV heads
        dict(name="attend_32x8_d256", op="attend", groups=32, samples=8, prefix=2560, suffix=512, new=1, hq=16, hkv=2, d=256, rows=32, chunk=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "attend", "attend"])
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8] if d < 256 else [1, 2, 4])
    if op == "append":
        seqs = _log(rng, 1, 512)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, 8192 // seqs))
        return dict(op=op, seqs=seqs, new=new, ctx=_log(rng, 1, 2000), hkv=hkv, d=d, pad=rng.choice([0, 0, rng.randint(1, 40)]))
    if op == "gather":
        seqs = _log(rng, 1, 16)
        return dict(op=op, seqs=seqs, ctx=_log(rng, 1, 32768 // seqs), hkv=hkv, d=d, pad=rng.choice([0, rng.randint(1, 20)]))
    groups, samples = _log(rng, 1, 64), rng.choice([1, 2, 5, 8, 16])
    seqs = groups * samples
    prefix = rng.choice([0, _log(rng, 16, max(32, min(32768, 160000 // groups)))])
    suffix = _log(rng, 1, max(2, min(65536, 200000 // seqs)))
    group = rng.choice([1, 2, 4, 5, 8])
    new = rng.choice([1, 1, 1, 2, 5])
    return dict(
        op=op, groups=groups, samples=samples, prefix=prefix, suffix=suffix, new=new, hq=group * hkv, hkv=hkv, d=d,
        rows=32 if d == 256 else rng.choice([32, 64]), chunk=rng.choice([128, 256, 512, 1024]),
    )


def _near(r, mean):
    """A length between two fifths and eight fifths of the mean (mean itself if it stands alone)."""
    return max(1, int(round(mean * r.uniform(0.4, 1.6))))


def _lengths(case):
    """Lengths of the case's sequences, the same for every seed: for ``attend`` (prefix of every
    group, length of every sequence; with two or more groups one sequence in ninety is empty), for
    the others the tokens a sequence has in the cache."""
    r = random.Random(sum(v * 31**i for i, v in enumerate(case[k] for k in sorted(case) if isinstance(case[k], int))))
    if case["op"] != "attend":
        return [case["ctx"] if case["seqs"] == 1 else _near(r, case["ctx"]) for _ in range(case["seqs"])]
    alone = case["groups"] == 1 and case["samples"] == 1
    prefix = [case["prefix"] if case["groups"] < 16 else _near(r, case["prefix"]) if case["prefix"] else 0 for _ in range(case["groups"])]
    lens = []
    for g in range(case["groups"]):
        for _ in range(case["samples"]):
            n = prefix[g] + (case["suffix"] if alone else _near(r, case["suffix"]))
            lens.append(max(n, case["new"]))
            if not prefix[g] and case["groups"] > 1 and case["new"] == 1 and r.random() < 1 / 90:
                lens[-1] = 0
    return prefix, lens


def _unique_blocks(case):
    """Blocks that hold the tokens of the case's sequences, each counted once."""
    prefix, lens = _lengths(case)
    total, n = 0, case["samples"]
    for g, p in enumerate(prefix):
        total += p // BLOCK + sum(-(-m // BLOCK) - min(p // BLOCK, -(-m // BLOCK)) for m in lens[g * n : (g + 1) * n])
    return total


def work(case):
    hkv, d = case["hkv"], case["d"]
    token = 2 * hkv * d  # codes of one token, K and V
    if case["op"] == "append":
        t = case["seqs"] * case["new"]
        # rows read, codes written, the scales of the blocks touched read and written
        return {"bytes": t * (2 * token + token + 8) + (t / BLOCK + case["seqs"]) * 16 * hkv, "flops": 2 * t * token}
    if case["op"] == "gather":
        t = sum(_lengths(case))
        return {"bytes": t * (token + 2 * token + 8) + t / BLOCK * 8 * hkv, "flops": t * token}
    prefix, lens = _lengths(case)
    blocks, rows = _unique_blocks(case), len(lens) * case["new"]
    return {
        "bytes": blocks * (BLOCK * token + 8 * hkv) + rows * case["hq"] * (4 * d + 4),
        "flops": 4 * sum(lens) * case["new"] * case["hq"] * d,
    }


# ---- inputs --------------------------------------------------------------------------------------


def _tiles(k, v):
    """``[blocks, 16, Hkv, D]`` codes (bytes) -> the cache's tiles."""
    nb, _, h, d = k.shape
    cache = torch.empty(2, nb, h, BLOCK * d, dtype=torch.uint8, device=k.device)
    cache[0].view(nb, h, d // 16, BLOCK, 16).copy_(k.view(nb, BLOCK, h, d // 16, 16).permute(0, 2, 3, 1, 4))
    cache[1].view(nb, h, d, BLOCK).copy_(v.permute(0, 2, 3, 1))
    return cache


def _values(gen, device, shape, spread):
    """Keys or values as a model makes them: some channels larger than the others, some tokens too."""
    x = torch.randn(shape, generator=gen, device=device)
    h, d = shape[-2:]
    channel = torch.exp(0.5 * torch.randn(h, d, generator=gen, device=device))
    token = torch.exp(spread * torch.randn(shape[:-2] + (1, 1), generator=gen, device=device))
    return x.mul_(channel).mul_(token)


def _power_of_two(amax):
    """The smallest power of two s with amax <= 448 s, kept between the format's bounds."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e + 1, e) - 9
    e = torch.where(amax > 0, e, torch.full_like(e, SCALE_LOW)).clamp(SCALE_LOW, SCALE_HIGH)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)  # 2^e, exactly


def _filled_cache(gen, device, nb, h, d):
    """A cache whose blocks are full, and its scales."""
    codes, scales = [], []
    for spread in (0.2, 0.4):
        x = _values(gen, device, (nb, BLOCK, h, d), spread)
        s = _power_of_two(x.abs().amax(dim=(1, 3)))
        codes.append(x.div_(s[:, None, :, None]).to(FP8).view(torch.uint8))
        scales.append(s)
    return _tiles(*codes), torch.stack(scales, dim=-1).contiguous()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    host = random.Random(seed)
    h, d = case["hkv"], case["d"]
    if case["op"] == "attend":
        return _prepare_attend(case, device, gen, host)
    ctx = _lengths(case)
    new = case["new"] if case["op"] == "append" else 0
    spans = [(c % BLOCK, c % BLOCK + new) if new else (0, c) for c in ctx]  # the tokens written or read, in the blocks that hold them
    per = [-(-e // BLOCK) for _, e in spans]
    nb = sum(per) + max(1, sum(per) // 8)
    order = list(range(nb))
    host.shuffle(order)
    slots, at = [], 0
    for (b, e), n in zip(spans, per):
        mine = order[at : at + n]
        at += n
        slots += [mine[p // BLOCK] * BLOCK + p % BLOCK for p in range(b, e)]
    slots += [-1] * case["pad"]  # a batch padded to a fixed size
    slots = torch.tensor(slots, dtype=torch.int64, device=device)
    cache, scales = _filled_cache(gen, device, nb, h, d)
    state = dict(op=case["op"], d=d, cache=cache.view(FP8), scales=scales, slots=slots)
    if new:
        # views of a fused projection's output: query heads, key heads, value heads
        fused = _values(gen, device, (len(slots), 4 * h, d), 0.6).to(torch.bfloat16)
        state |= dict(key=fused[:, 2 * h : 3 * h], value=fused[:, 3 * h :])
    return state


def _prepare_attend(case, device, gen, host):
    h, d, n, new = case["hkv"], case["d"], case["samples"], case["new"]
    prefix, lens = _lengths(case)
    used = _unique_blocks(case)
    nb = used + max(1, used // 8)
    order = list(range(nb))
    host.shuffle(order)
    width = max(1, max(-(-m // BLOCK) for m in lens))
    table, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    ends = []  # (block, first position that no sequence reads)
    for g, p in enumerate(prefix):
        shared = order[at : at + p // BLOCK]
        at += len(shared)
        for s in range(g * n, (g + 1) * n):
            need = -(-lens[s] // BLOCK)
            row = shared[:need] + order[at : at + max(0, need - len(shared))]
            at += max(0, need - len(shared))
            table[s, :need] = torch.tensor(row, dtype=torch.int32)
            if lens[s] % BLOCK:
                ends.append((row[-1], lens[s] % BLOCK))
    cache, scales = _filled_cache(gen, device, nb, h, d)
    # what no sequence reads holds NaN: the blocks of nobody with their scales, positions behind the last token
    rest = torch.tensor(order[at:], dtype=torch.int64, device=device)
    cache[:, rest], scales[rest] = NAN_CODE, float("nan")
    if ends:
        blk = torch.tensor([b for b, _ in ends], dtype=torch.int64, device=device)
        past = torch.arange(BLOCK, device=device) >= torch.tensor([o for _, o in ends], device=device)[:, None]
        k, v = cache[0].view(nb, h, d // 16, BLOCK, 16), cache[1].view(nb, h, d, BLOCK)
        k[blk] = torch.where(past[:, None, None, :, None], NAN_CODE, k[blk])
        v[blk] = torch.where(past[:, None, None, :], NAN_CODE, v[blk])
    rows = len(lens) * new
    q = torch.randn(rows, case["hq"], d, generator=gen, device=device).to(torch.bfloat16)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=device)
    # token i of a sequence's `new` query tokens sees all but the tokens behind it
    row_table = torch.arange(len(lens), device=device, dtype=torch.int32).repeat_interleave(new)
    row_lens = seq_lens.repeat_interleave(new) - (new - 1 - torch.arange(rows, device=device, dtype=torch.int32) % new)
    state = dict(
        op="attend", d=d, cache=cache.view(FP8), scales=scales, q=q, table=table.to(device), seq_lens=seq_lens, row_table=row_table,
        row_lens=row_lens.to(torch.int32).contiguous(), scale=d**-0.5,
    )
    if own:  # the forest of the batch: made once per step, used by every layer's call
        from arctic_platform_amd import build_forest_metadata
        from arctic_platform_amd.forest import rows_from_query_runs

        sizes = dict(num_q_heads=case["hq"], num_kv_heads=h, head_dim=d, chunk_tokens=case["chunk"], rows_per_item=case["rows"])
        if new == 1:
            state["forest"] = build_forest_metadata(state["table"], seq_lens, **sizes)
        else:
            starts = torch.arange(0, rows + 1, new, dtype=torch.int32, device=device)
            run_table, run_lens, run_group = rows_from_query_runs(starts, seq_lens, rows, width)
            state["forest"] = build_forest_metadata(
                state["table"], run_lens, row_table=run_table, row_group=run_group, kv_reread=new > 2, **sizes
            )
    return state


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "gather": _gather, "attend": _attend}[state["op"]](state)


def _run_own(s):
    from arctic_platform_amd import append_kv, forest_cascade_decode
    from arctic_platform_amd.cache import gather_kv

    if s["op"] == "append":
        append_kv(s["key"], s["value"], s["cache"], s["slots"], block_scales=s["scales"])
        return {"cache": s["cache"], "scales": s["scales"]}
    if s["op"] == "gather":
        k, v = gather_kv(s["cache"], s["slots"], s["d"], block_scales=s["scales"])
        return {"key": k, "value": v}
    out, lse = forest_cascade_decode(s["q"], s["cache"], s["forest"], s["scale"], block_scales=s["scales"])
    return {"out": out, "lse": lse}


def _append(s):
    cache, scales, slots, d = s["cache"].view(torch.uint8), s["scales"], s["slots"], s["d"]
    nb, h = scales.shape[:2]
    live = slots >= 0
    blk, off = slots[live] // BLOCK, slots[live] % BLOCK
    rows = torch.stack([s["key"][live], s["value"][live]], dim=-2).float()  # [T, H, 2, D]
    amax = torch.zeros_like(scales).index_reduce_(0, blk, rows.abs().amax(dim=-1), "amax")
    touched = torch.zeros(nb, dtype=torch.bool, device=cache.device).index_fill_(0, blk, True)
    begun = torch.zeros_like(touched).index_fill_(0, blk[off == 0], True)
    new = torch.where(begun[:, None, None], _power_of_two(amax), torch.maximum(scales, _power_of_two(amax)))
    new = torch.where(touched[:, None, None], new, scales)
    # codes of earlier tokens of a block whose scale has grown
    grown = ((new != scales) & ~begun[:, None, None])[..., None]
    ratio = (scales / new)[..., None]
    codes = cache.permute(1, 2, 0, 3)  # [blocks, H, 2, 16 D]
    codes.copy_(torch.where(grown, (codes.view(FP8).float() * ratio).to(FP8).view(torch.uint8), codes))
    scales.copy_(new)
    q = (rows / new[blk][..., None]).to(FP8).view(torch.uint8)
    cache[0].view(nb, h, d // 16, BLOCK, 16)[blk, :, :, off] = q[:, :, 0].reshape(-1, h, d // 16, 16)
    cache[1].view(nb, h, d, BLOCK)[blk, :, :, off] = q[:, :, 1]
    return {"cache": s["cache"], "scales": scales}


def _gather(s):
    cache, scales, d = s["cache"].view(torch.uint8), s["scales"], s["d"]
    nb, h = scales.shape[:2]
    live = (s["slots"] >= 0)[:, None, None]
    slots = s["slots"].clamp(min=0)
    blk, off = slots // BLOCK, slots % BLOCK
    k = cache[0].view(nb, h, d // 16, BLOCK, 16)[blk, :, :, off].reshape(-1, h, d).view(FP8).float()
    v = cache[1].view(nb, h, d, BLOCK)[blk, :, :, off].contiguous().view(FP8).float()
    sc = scales[blk]
    zero = torch.zeros((), device=cache.device)
    return {
        "key": torch.where(live, k * sc[..., 0:1], zero).to(torch.bfloat16),
        "value": torch.where(live, v * sc[..., 1:2], zero).to(torch.bfloat16),
    }


def _attend(s):
    cache, d = s["cache"].view(torch.uint8), s["d"]
    nb, h = s["scales"].shape[:2]
    rows, hq = s["q"].shape[:2]
    blocks = s["table"][s["row_table"].long()].long()  # [R, M]
    seen = (torch.arange(blocks.shape[1] * BLOCK, device=cache.device) < s["row_lens"][:, None])[:, None, :]  # [R, 1, L]
    sc = s["scales"][blocks]  # [R, M, H, 2]
    q = s["q"].float().view(rows, h, hq // h, d)
    k = cache[0].view(nb, h, d // 16, BLOCK, 16)[blocks]  # [R, M, H, D / 16, 16 tokens, 16]
    k = k.permute(0, 2, 1, 4, 3, 5).reshape(rows, h, -1, BLOCK * d).view(FP8).float().mul_(sc[..., 0].transpose(1, 2)[..., None])
    score = torch.matmul(q, k.view(rows, h, -1, d).transpose(2, 3)).mul_(s["scale"])  # [R, H, G, L]
    del k
    score = score.masked_fill_(~seen[:, :, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    v = cache[1].view(nb, h, d, BLOCK)[blocks]  # [R, M, H, D, 16 tokens]
    v = v.permute(0, 2, 1, 4, 3).reshape(rows, h, -1, BLOCK * d).view(FP8).float().mul_(sc[..., 1].transpose(1, 2)[..., None])
    v = v.view(rows, h, -1, d).masked_fill_(~seen[..., None], 0.0)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.where(total > 0, top + total.log(), float("-inf"))
    return {"out": out.view(rows, hq, d).to(torch.bfloat16), "lse": lse.view(rows, hq)}


# ---- the same from the definition, in 64 bits ----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "gather": _exact_gather, "attend": _exact_attend}[s["op"]](s)


def _decode(codes):
    """Bytes of the e4m3 format -> the values they stand for, from the format's definition."""
    c = torch.arange(256, dtype=torch.float64)
    e, m = (c // 8) % 16, c % 8
    v = torch.where(e == 0, m / 8 * 2.0**-6, (1 + m / 8) * 2.0 ** (e - 7))
    v = torch.where((e == 15) & (m == 7), torch.full_like(v, float("nan")), v)
    v = torch.where(c >= 128, -v, v)
    return v.to(codes.device)[codes.long()]


def _round_e4m3(x):
    """The e4m3 value nearest to x, ties to the even one (|x| <= 448)."""
    _, e = torch.frexp(x)
    step = (((e - 1).clamp(min=-6) - 3 + 1023).to(torch.int64) << 52).view(torch.float64)  # a power of two, exactly
    return torch.round(x / step) * step


def _exact_append(s):
    old, slots, d = s["cache"].view(torch.uint8), s["slots"], s["d"]
    scales = s["scales"].double()
    nb, h = scales.shape[:2]
    live = slots >= 0
    blk, off = slots[live] // BLOCK, slots[live] % BLOCK
    # token-major values of every block, NaN where the call writes nothing
    fresh = torch.full((2, nb, BLOCK, h, d), float("nan"), dtype=torch.float64, device=old.device)
    fresh[0, blk, off], fresh[1, blk, off] = s["key"][live].double(), s["value"][live].double()
    written = ~fresh[0, :, :, 0, 0].isnan()  # [blocks, 16]
    amax = torch.where(fresh.isnan(), torch.zeros_like(fresh), fresh.abs()).amax(dim=(2, 4))  # [2, blocks, H]
    _, e = torch.frexp((amax / FP8_MAX).clamp(min=2.0**SCALE_LOW))
    need = ((e + 1023).to(torch.int64) << 52).view(torch.float64)  # a power of two above amax / 448
    need = torch.where((amax <= FP8_MAX * need / 2) & (need > 2.0**SCALE_LOW), need / 2, need).permute(1, 2, 0)
    new = torch.where(written[:, :1, None], need, torch.maximum(need, scales))
    new = torch.where(written.any(dim=1)[:, None, None], new, scales)
    keep = torch.where(written[:, :1, None], torch.ones_like(new), scales / new)  # a begun block keeps no meaning
    k = _decode(old[0]).view(nb, h, d // 16, BLOCK, 16).permute(0, 3, 1, 2, 4).reshape(nb, BLOCK, h, d)
    v = _decode(old[1]).view(nb, h, d, BLOCK).permute(0, 3, 1, 2)
    done = []
    for plane, x in enumerate((k, v)):
        x = torch.where(written[:, :, None, None], fresh[plane] / new[:, None, :, None, plane], x * keep[:, None, :, None, plane])
        done.append(_round_e4m3(x))
    cache = torch.empty(2, nb, h, BLOCK * d, dtype=torch.float64, device=old.device)
    cache[0].view(nb, h, d // 16, BLOCK, 16).copy_(done[0].view(nb, BLOCK, h, d // 16, 16).permute(0, 2, 3, 1, 4))
    cache[1].view(nb, h, d, BLOCK).copy_(done[1].permute(0, 2, 3, 1))
    return {"cache": cache, "scales": new}


def _exact_gather(s):
    cache, d = s["cache"].view(torch.uint8), s["d"]
    nb, h = s["scales"].shape[:2]
    slots = s["slots"]
    index = slots.clamp(min=0)
    blk, off = index // BLOCK, index % BLOCK
    value = _decode(cache.view(2, nb, h, -1)[:, blk])  # whole tiles of every token's block
    sc = s["scales"].double()[blk]
    k = value[0].view(-1, h, d // 16, BLOCK, 16).gather(3, off.view(-1, 1, 1, 1, 1).expand(-1, h, d // 16, 1, 16)).reshape(-1, h, d)
    v = value[1].view(-1, h, d, BLOCK).gather(3, off.view(-1, 1, 1, 1).expand(-1, h, d, 1)).squeeze(-1)
    live = (slots >= 0).double()[:, None, None]
    return {"key": k * sc[..., 0:1] * live, "value": v * sc[..., 1:2] * live}


def _exact_attend(s):
    cache, d = s["cache"].view(torch.uint8), s["d"]
    nb, h = s["scales"].shape[:2]
    rows, hq = s["q"].shape[:2]
    out = torch.zeros(rows, hq, d, dtype=torch.float64, device=cache.device)
    lse = torch.full((rows, hq), float("-inf"), dtype=torch.float64, device=cache.device)
    lens, per = s["row_lens"].tolist(), rows // len(s["seq_lens"])
    for first in range(0, rows, per):  # the rows of one sequence
        longest = max(lens[first : first + per])
        if longest == 0:
            continue
        ids = s["table"][first // per, : -(-longest // BLOCK)].long()
        sc = s["scales"][ids].double()
        k = _decode(cache[0][ids]).view(-1, h, d // 16, BLOCK, 16).permute(1, 0, 3, 2, 4).reshape(h, -1, BLOCK, d) * sc[..., 0].t()[..., None, None]
        v = _decode(cache[1][ids]).view(-1, h, d, BLOCK).permute(1, 0, 3, 2) * sc[..., 1].t()[..., None, None]
        for r in range(first, first + per):
            n = lens[r]
            kk, vv = k.reshape(h, -1, d)[:, :n], v.reshape(h, -1, d)[:, :n]
            score = torch.bmm(s["q"][r].double().view(h, hq // h, d), kk.transpose(1, 2).contiguous()) * s["scale"]
            m = score.amax(dim=-1, keepdim=True)
            e = torch.exp(score - m)
            total = e.sum(dim=-1, keepdim=True)
            out[r] = torch.bmm(e / total, vv.contiguous()).view(hq, d)
            lse[r] = (m + torch.log(total)).view(hq)
    return {"out": out, "lse": lse}
