"""The token table of the torch-hosted NanoGPT is one module on every path: its hooks see each lookup."""
import copy

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd.nanogpt import NanoGPT, make_packed_batch

TINY = dict(vocab=17, max_seq_len=32, d_model=32, n_heads=2, head_dim=32, mlp_dim=64, n_layers=1)
LENS = [9, 1, 20]


def _forward(model, packed, device):
    ids, _ = make_packed_batch(LENS, TINY["vocab"], seed=1)
    ids = ids.to(device)
    return model(ids, ct.packed_plan(LENS, 2, 2, device=device)) if packed else model(ids[None])


def _count_hooks(attention, device, packed):
    model = NanoGPT(**TINY, attention=attention).init_weights(1).to(device)
    assert isinstance(model.tok, torch.nn.Embedding) and list(model.tok.state_dict()) == ["weight"]
    copy.deepcopy(model)
    plain = _forward(model, packed, device)
    seen = []
    model.tok.register_forward_hook(lambda mod, args, out: seen.append(out.shape) or 0 * out)
    hooked = _forward(model, packed, device)
    n = sum(LENS)
    assert seen == [(n, 32) if packed else (1, n, 32)]
    assert not torch.equal(plain, hooked)  # what the hook returns is what the model goes on with


@pytest.mark.parametrize("packed", [True, False])
def test_hooks_on_the_cpu(packed):
    _count_hooks("sdpa", "cpu", packed)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [True, False])
def test_hooks_on_the_kernels(packed):
    _count_hooks("ctattn", "cuda", packed)


@pytest.mark.gpu
def test_padding_ids_of_a_packed_batch():
    """An id outside the vocabulary embeds as zeros and has no gradient."""
    model = NanoGPT(**TINY, embedding_scale=3.0).init_weights(1).cuda()
    ids = torch.arange(sum(LENS)) % TINY["vocab"]
    ids[::4] = -1
    out = []
    model.tok.register_forward_hook(lambda mod, args, x: out.append(x))
    model(ids.cuda(), ct.packed_plan(LENS, 2, 2)).sum().backward()
    want = torch.where((ids >= 0)[:, None], model.tok.weight.detach().cpu()[ids] * 3.0, torch.zeros(()))
    assert torch.equal(out[0].detach().cpu(), want)
    assert model.tok.weight.grad.isfinite().all()
