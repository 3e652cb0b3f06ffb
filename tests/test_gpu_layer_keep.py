"""The probabilities that a layer step hands out, where its memory held something before."""
import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [False, "varlen"])
def test_kept_probabilities_are_zero_behind_what_a_row_sees(form):
    from energonai_amd import layer
    B, S, H, D, lens = 3, 200, 2, 64, [200, 7, 130]
    g = torch.Generator().manual_seed(1)
    T, hid = sum(lens), H * D
    hidden = torch.zeros(B, S, hid, dtype=torch.float16)
    for b, n in enumerate(lens):
        hidden[b, :n] = torch.randn(n, hid, generator=g)
    qkv = torch.randn(1, T, H, 3 * D, generator=g).half().cuda()
    gamma, beta = torch.ones(hid, dtype=torch.float16, device="cuda"), torch.zeros(hid, dtype=torch.float16, device="cuda")
    announce("kept probabilities", form)
    args = (hidden.cuda(), qkv, torch.tensor(lens, dtype=torch.int32, device="cuda"), H, D, gamma, beta, 1e-5, D ** -0.5, True, False)
    layer.padding_removal_layer(*args, keep=True, fused_attention=form)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = [torch.full((B, H, S, S), float("nan"), dtype=torch.float16, device="cuda") for _ in range(8)]      # what the next allocations hold
    del held
    probs = layer.padding_removal_layer(*args, keep=True, fused_attention=form)["probs"]
    for b, n in enumerate(lens):
        rows = probs[b, :, :n].float()
        assert (rows.triu(1) == 0).all()
        assert float((rows.sum(-1) - 1).abs().max()) < 5e-3
