"""Gradients of a reconstruction against sums made one copy after the other on the host, bit for bit."""

import pytest
import torch

from arctic_platform_amd.split_attention import SplitLayout


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout,ids", [([(40, [20, 33, 7]), (7, [5]), (3, [])], [[3, 0, 2], [1], []]), ([(17, [1] * 9)], [list(range(8, -1, -1))])])
def test_gradients_add_the_copies_in_the_order_of_the_rows(gpu, dtype, layout, ids):
    from arctic_platform_amd.reconstruct import reconstruct_sequences, sample_index

    layout = SplitLayout(layout)
    index = sample_index(layout, ids)
    x = torch.zeros(layout.num_tokens, 24).to(dtype).to(gpu).requires_grad_()
    full = reconstruct_sequences(x, layout, ids)
    w = torch.randn(full.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    full.backward(w.to(gpu))
    want = torch.zeros(layout.num_tokens, 24)
    for row, src in enumerate(index.full_from.tolist()):  # fp32 sums, rounded once
        want[src] += w[row].float()
    assert torch.equal(x.grad.cpu(), want.to(dtype))
