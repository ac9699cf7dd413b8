"""The writer of the block-scaled cache on calls of more tokens than one workgroup's window: the rule for a
block's scale is that of the whole call, whatever the order of its tokens and however many they are."""

import os

import pytest
import torch

from arctic_platform_amd import _lib
from arctic_platform_amd.kv_layout import block_scales_shape, kv_cache_shape, quantize_blocks
from oracle import block_scales as oracle
from tests.test_block_scaled_cache import FP8, _append_and_check, _old_state, _rows
from tests.test_emulated_kernels import _ok, emu, guarded  # noqa: F401  (emu is a fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["reversed", "halves exchanged"])
def test_a_block_begun_by_a_late_token(gpu, request, order):
    """33000 tokens, the one at offset 0 of every block far behind (or just behind) the others of its block."""
    if request.config.getoption("--on-emulation"):
        pytest.skip("hundreds of workgroups that look at tens of thousands of slots: not in the emulation")
    from arctic_platform_amd import append_kv
    from arctic_platform_amd.cache import gather_kv

    g = torch.Generator().manual_seed(5)
    t, d = 33000, 64
    nb = (t + 15) // 16
    pos = torch.arange(t)
    pos = pos.flip(0) if order == "reversed" else torch.cat([pos[pos % 16 >= 8], pos[pos % 16 < 8]])
    slots = torch.randperm(nb, generator=g)[pos // 16] * 16 + pos % 16
    key, value = _rows(g, t, 1, d), _rows(g, t, 1, d)
    # the blocks were used before, with scales far above what the new tokens need
    cache = torch.full(kv_cache_shape(nb, 16, 1, d), 0x55, dtype=torch.uint8, device=gpu).view(FP8)
    table = torch.full(block_scales_shape(nb, 1), 2.0**30, device=gpu)
    append_kv(key.to(gpu), value.to(gpu), cache, slots.to(gpu), block_scales=table)
    torch.cuda.synchronize()
    # whole blocks (all but the last, which is not full): what quantising them at once gives
    full = slots // 16 != slots[pos == t - 1] // 16
    k, v = torch.zeros(nb, 16, 1, d).bfloat16(), torch.zeros(nb, 16, 1, d).bfloat16()
    k[slots // 16, slots % 16], v[slots // 16, slots % 16] = key, value
    want, scales = quantize_blocks(k, v)
    blocks = (slots[full] // 16).unique()
    assert torch.equal(table.cpu()[blocks], scales[blocks])
    assert torch.equal(cache.cpu().view(torch.uint8)[:, blocks], want.view(torch.uint8)[:, blocks])
    rk, rv = gather_kv(cache, slots.to(gpu), d, block_scales=table)
    for x, y, plane in ((key, rk, 0), (value, rv, 1)):
        s = table.cpu()[slots // 16, :, plane : plane + 1].double()
        # half a step of e4m3 relative to the value, or half its smallest step times the scale
        assert ((x.double() - y.cpu().double()).abs() <= torch.maximum(x.double().abs() * 2.0**-4, s * 2.0**-10)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,t", [(64, 1500), (128, 700), (256, 1030)])
def test_windows_of_many_blocks(gpu, d, t):
    """Every token of a window in another block, the blocks' numbers multiples of a power of two (their places
    in the look-up table meet), blocks shared with other windows in both directions."""
    g = torch.Generator().manual_seed(t)
    nb, hkv = 2048, 1
    used = torch.arange(0, nb, 32)
    cache, scales = _old_state(g, nb, hkv, d)
    slots = used[torch.randint(0, len(used), (t,), generator=g)] * 16 + torch.randint(0, 16, (t,), generator=g)
    slots[::97] = -1
    _append_and_check(gpu, cache, scales, _rows(g, t, hkv, d), _rows(g, t, hkv, d), slots, fused=False)


@pytest.mark.parametrize("host_threads", [1, 8])
def test_order_of_a_call_does_not_matter(emu, host_threads):  # noqa: F811
    """The same tokens in order, reversed and shuffled: the same cache and table, byte for byte."""
    emu.emu_set_host_threads(host_threads)
    g = torch.Generator().manual_seed(2)
    t, hkv, d = 600, 1, 64
    nb = 60
    cache, scales = _old_state(g, nb, hkv, d)
    slots = torch.randperm(nb * 16, generator=g)[:t]
    key, value = _rows(g, t, hkv, d), _rows(g, t, hkv, d)
    want, table = oracle.append_reference(cache, scales, key, value, slots)
    for perm in (torch.arange(t), torch.arange(t).flip(0), torch.randperm(t, generator=g)):
        kv, sc, sl, k, v = guarded(cache.view(torch.uint8)), guarded(scales), guarded(slots[perm]), guarded(key[perm]), guarded(value[perm])
        _ok(emu, emu.fca_append_kv_block_scaled(
            k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), t, hkv, d, sl.data_ptr(), kv.data_ptr(), kv.data_ptr() + kv.stride(0),
            kv.stride(1), kv.stride(2), nb, sc.data_ptr(), None,
        ))
        assert torch.equal(kv, want.view(torch.uint8)) and torch.equal(sc.nan_to_num(-1.0), table.nan_to_num(-1.0))
    emu.emu_set_host_threads(1)


def test_more_tokens_than_a_call_takes_are_refused():
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build_library()
    lib, ok = _lib.load_library(), 1 << 20
    rc = lib.fca_append_kv_block_scaled(ok, ok, 128, 128, (1 << 30) + 1, 1, 128, ok, ok, ok + (1 << 16), 16 * 128, 16 * 128, 4, ok, None)
    assert rc == -2 and "more than one call takes" in lib.fca_last_error().decode(), rc
