"""Every launch is made with the device of its tensors as the current one (a stream belongs to a device, and a
launch goes to the current one).  No GPU: the library's launching functions are replaced by ones that look."""

import contextlib
import os

import pytest
import torch

from arctic_platform_amd import _lib, cache, forest, ops, reconstruct, split_attention
from arctic_platform_amd.kv_layout import block_scales_shape, kv_cache_shape


class _Library:
    """The built library, but for the functions that would launch: those note whether their device is set."""

    HOST_ONLY = ("fca_meta_describe", "fca_workspace_bytes_dtype", "fca_split_layout_ints", "fca_split_layout_build", "fca_split_workspace_bytes")

    def __init__(self, real, state):
        self.real, self.state, self.launched = real, state, []

    def __getattr__(self, name):
        real = getattr(self.real, name)
        if name in self.HOST_ONLY:
            return real

        def launch(*args):
            self.launched.append((name, self.state["device"]))
            return 0

        return launch


@pytest.fixture
def library(monkeypatch):
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build_library()
    state = {"device": None}

    @contextlib.contextmanager
    def on_device(device):
        before, state["device"] = state["device"], device
        yield
        state["device"] = before

    lib = _Library(_lib.load_library(), state)
    monkeypatch.setattr(_lib, "load_library", lambda: lib)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    for module in (cache, forest, ops, reconstruct, split_attention):
        monkeypatch.setattr(module, "_stream_ptr", lambda device: None)
        monkeypatch.setattr(module, "on_device", on_device, raising=False)
    return lib


def _take(lib, *names):
    got, lib.launched = lib.launched, []
    assert [n for n, _ in got] == list(names), got
    assert all(device == torch.device("cpu") for _, device in got), got


def test_cache_rows(library):
    rows, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    fp8 = torch.zeros(kv_cache_shape(4, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    for kw, names in ((dict(), ("fca_append_kv", "fca_gather_kv")), (dict(block_scales=torch.ones(block_scales_shape(4, 2))), ("fca_append_kv_block_scaled", "fca_gather_kv_block_scaled"))):
        cache.append_kv(rows, rows, fp8, slots, **kw)
        cache.gather_kv(fp8, slots, 64, **kw)
        _take(library, *names)


def test_metadata_attention_and_merge(library):
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([20, 30], dtype=torch.int32)
    sizes = dict(num_q_heads=4, num_kv_heads=2, head_dim=64)
    md = forest.build_forest_metadata(table, lens, **sizes)
    md = forest.build_forest_metadata(table, lens, out=md, update=True, **sizes)
    rt, rl, rg = forest.rows_from_query_runs(torch.tensor([0, 1, 3], dtype=torch.int32), lens, 3, 4)
    forest.build_forest_metadata(table, torch.full((3,), 9, dtype=torch.int32), row_table=torch.zeros(3, dtype=torch.int32), row_group=torch.zeros(3, dtype=torch.int32), **sizes)
    _take(library, "fca_build_metadata", "fca_update_metadata", "fca_rows_from_query_runs", "fca_build_metadata_rows")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    fp8 = torch.zeros(kv_cache_shape(4, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    kw = dict(block_scales=torch.ones(block_scales_shape(4, 2)))
    out = ops.forest_cascade_decode(q, fp8, md, 0.1, return_lse=False, **kw)
    ops.forest_cascade_decode_static(q, fp8, md, 0.1, out=out, **kw)
    ops.prefix_pass(q, fp8, md, 0.1, **kw)
    ops.suffix_pass(q, fp8, md, 0.1, **kw)
    ops.forest_pass(q, fp8, md, 0.1, **kw)
    ops.merge_partials(md, q)
    _take(library, "fca_decode_step", "fca_decode_step_static", "fca_prefix_pass", "fca_suffix_pass", "fca_forest_pass", "fca_merge_dtype")


def test_the_trainers_operators(library):
    layout = split_attention.SplitLayout([(3, [2, 1])], device="cpu")
    layout.dev = torch.from_numpy(layout.host)
    t = layout.num_tokens
    q, k, v = (torch.zeros(t, 4, 64, dtype=torch.bfloat16) for _ in range(3))
    out, lse = split_attention.split_attention_forward(q, k, v, layout, 0.1)
    split_attention.split_attention_backward(out, q, k, v, out, lse, layout, 0.1)
    x = torch.zeros(t, 8, requires_grad=True)
    reconstruct.reconstruct_sequences(x, layout, [[0, 1]]).sum().backward()
    names = [n for n, _ in library.launched]
    assert "fca_split_attention_forward" in names and "fca_split_attention_backward" in names and "fca_gather_rows" in names and "fca_sum_rows" in names
    assert all(device == torch.device("cpu") for _, device in library.launched), library.launched


def test_outputs_on_another_device_are_refused(library):
    """(A host tensor's address would reach the kernel.)"""
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([20, 30], dtype=torch.int32)
    md = forest.build_forest_metadata(table, lens, num_q_heads=4, num_kv_heads=2, head_dim=64)
    q, elsewhere = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="meta")
    fp8 = torch.zeros(kv_cache_shape(4, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    library.launched = []
    for kw in (dict(), dict(block_scales=torch.ones(block_scales_shape(4, 2)))):
        with pytest.raises(ValueError, match="out is on meta"):
            ops.forest_cascade_decode(q, fp8, md, 0.1, out=elsewhere, **kw)
        with pytest.raises(ValueError, match="out is on meta"):
            ops.forest_cascade_decode_static(q, fp8, md, 0.1, out=elsewhere, **kw)
        with pytest.raises(ValueError, match="lse is on meta"):
            ops.forest_cascade_decode_static(q, fp8, md, 0.1, out=torch.zeros_like(q), lse=torch.zeros(2, 4, device="meta"), **kw)
    with pytest.raises(ValueError, match="out is on meta"):
        ops.merge_partials(md, q, out=elsewhere)
    assert not library.launched
