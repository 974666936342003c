"""The torch-hosted NanoGPT on batches without a token, dense and packed."""
import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd.nanogpt import NanoGPT, make_packed_batch

TINY = dict(vocab=17, max_seq_len=32, d_model=32, n_heads=4, head_dim=32, mlp_dim=64, n_layers=2)
DEVICES = [("sdpa", "cpu"), pytest.param("ctattn", "cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("attention,device", DEVICES)
@pytest.mark.parametrize("kv", [None, 2])
@pytest.mark.parametrize("shape", [(0, 5), (2, 0), (0, 0)])
def test_dense(attention, device, kv, shape):
    model = NanoGPT(**TINY, n_kv_heads=kv, attention=attention).init_weights(1).to(device)
    logits = model(torch.zeros(shape, dtype=torch.long, device=device))
    assert logits.shape == (*shape, TINY["vocab"])
    logits.sum().backward()
    assert all(p.grad is None or not bool(p.grad.any()) for p in model.parameters())


@pytest.mark.parametrize("attention,device", DEVICES)
@pytest.mark.parametrize("lens", [[], [0], [0, 0]])
def test_packed(attention, device, lens):
    model = NanoGPT(**TINY, n_kv_heads=2, attention=attention).init_weights(1).to(device)
    ids, targets = make_packed_batch(lens, TINY["vocab"], seed=1)
    assert ids.dtype == targets.dtype == torch.int64 and ids.shape == targets.shape == (0,)
    logits = model(ids.to(device), ct.packed_plan(lens, 4, 2, device=device))
    assert logits.shape == (0, TINY["vocab"])
    logits.sum().backward()
    assert all(p.grad is None or not bool(p.grad.any()) for p in model.parameters())


def test_documents_without_a_token_between_others():
    model = NanoGPT(**TINY, n_kv_heads=2, attention="sdpa").init_weights(1).double()
    ids, _ = make_packed_batch([5, 3], TINY["vocab"], seed=1)
    with torch.no_grad():
        a = model(ids, ct.packed_plan([5, 3], 4, 2, device="cpu"))
        b = model(ids, ct.packed_plan([0, 5, 0, 3, 0], 4, 2, device="cpu"))
    assert torch.equal(a, b)
