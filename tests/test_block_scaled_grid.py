"""The cap of the attention grid (``fca_tensors.max_workgroups``) over the block-scaled cache: what is launched,
counted by the CPU emulation, and that the capped launch is complete."""

import ctypes

import pytest
import torch

from arctic_platform_amd import _lib
from arctic_platform_amd.forest import make_plan
from arctic_platform_amd.workloads import make_forest_workload
from tests.test_block_scaled_cache import FP8, _check_attention, _random_scales, _used_blocks
from tests.test_emulated_kernels import _ok, emu, guarded  # noqa: F401  (emu is a fixture)


@pytest.mark.parametrize("d,hq,hkv,rows", [(64, 8, 4, 32), (128, 8, 4, 32), (64, 8, 4, 64), (128, 8, 4, 64), (256, 8, 4, 32)])
@pytest.mark.parametrize("cap", [1, 3, 0])
def test_a_capped_launch_keeps_to_the_cap(emu, d, hq, hkv, rows, cap):  # noqa: F811
    g = torch.Generator().manual_seed(d + cap)
    w = make_forest_workload("grid", [230, 140, 70, 190, 133], [[0, 1], [0, 2], [3], [4]], g, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=FP8, poison_unused=True)
    scales = _random_scales(g, w.kv_cache, _used_blocks(w.block_table, w.seq_lens), powers=True)
    n, mb = w.block_table.shape
    plan = make_plan(n, mb, hq, hkv, d, chunk_tokens=64, rows_per_item=rows)
    nm, no, nl = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    _ok(emu, emu.fca_workspace_bytes_dtype(ctypes.byref(plan), _lib.FCA_FP8_E4M3_BLOCK, ctypes.byref(nm), ctypes.byref(no), ctypes.byref(nl)))
    meta, po, pl = guarded(torch.zeros(nm.value // 4, dtype=torch.int32)), guarded(torch.zeros(no.value // 2, dtype=torch.float16)), guarded(torch.zeros(nl.value // 4))
    bt, sl, q, kv, sc = guarded(w.block_table), guarded(w.seq_lens), guarded(w.q), guarded(w.kv_cache.view(torch.uint8)), guarded(scales)
    _ok(emu, emu.fca_build_metadata(ctypes.byref(plan), bt.data_ptr(), bt.stride(0), sl.data_ptr(), meta.data_ptr(), None))
    t = _lib.FcaTensors(
        q.data_ptr(), q.stride(0), q.stride(1), kv.data_ptr(), kv.data_ptr() + kv.stride(0), kv.stride(1), kv.stride(2),
        _lib.FCA_FP8_E4M3_BLOCK, 0, bt.data_ptr(), bt.stride(0), sc.data_ptr(), None, float(w.scale), 0, cap, 0,
    )
    _ok(emu, emu.fca_forest_pass(ctypes.byref(plan), ctypes.byref(t), meta.data_ptr(), po.data_ptr(), pl.data_ptr(), None))
    workgroups, threads = emu.emu_last_workgroups(), emu.emu_last_threads()
    tickets = int(meta[0]) * hkv
    assert tickets >= 4 * 3 * 3, tickets  # more than the waves of three workgroups: a cap of three binds
    if cap:
        assert workgroups <= cap and workgroups * threads <= cap * 256, (workgroups, threads)
    else:
        assert workgroups > 3
    out, lse = guarded(torch.zeros(n, hq, d).bfloat16()), guarded(torch.zeros(n, hq))
    _ok(emu, emu.fca_merge(ctypes.byref(plan), meta.data_ptr(), po.data_ptr(), pl.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), _lib.FCA_BF16, lse.data_ptr(), None))
    _check_attention(out, lse, w.q, w.kv_cache, scales, w.block_table, range(n), w.seq_lens.tolist(), w.scale, f"cap {cap}")
