"""A training step on packed documents: scaled embedding, packed attention with shared key heads, their
gradients and the Muon step, as the torch-hosted NanoGPT runs them, against the same model in 64 bits on
the CPU (attention there is torch's, document by document)."""
import copy
import math

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd.nanogpt import NanoGPT, make_packed_batch, muon_parameters, to_native, train_step

CFG = dict(vocab=65, max_seq_len=128, d_model=96, n_heads=6, n_kv_heads=2, head_dim=32, mlp_dim=192, n_layers=2,
           embedding_scale=math.sqrt(96.0))
LENS = [100, 1, 37, 64, 128, 5]


def _models(seed=3):
    ref = NanoGPT(**CFG, attention="sdpa").init_weights(seed).double()
    return ref, NanoGPT(**CFG, attention="ctattn").init_weights(seed)


def test_documents_do_not_see_each_other():
    ref, _ = _models()
    plan = ct.packed_plan(LENS, CFG["n_heads"], CFG["n_kv_heads"], device="cpu")
    ids, _ = make_packed_batch(LENS, CFG["vocab"], seed=1)
    with torch.no_grad():
        packed = ref(ids, plan)
        parts = [ref(part[None])[0] for part in ids.split(LENS)]
    assert float((packed - torch.cat(parts)).abs().max()) <= 1e-12 * float(packed.abs().max())
    with pytest.raises(ValueError):
        ref(ids[:-1], plan)
    with pytest.raises(ValueError):
        ref(torch.zeros(129, dtype=torch.long), ct.packed_plan([129], 6, 2, device="cpu"))
    with pytest.raises(ValueError):
        to_native(ref)


def test_muon_takes_matrices_only():
    ref, _ = _models()
    inside, rest = muon_parameters(ref)
    assert len(inside) == 2 * 6 and len(inside) + len(rest) == len(list(ref.parameters()))
    with pytest.raises(ValueError):
        ct.Muon(ref.parameters())


@pytest.mark.gpu
def test_step_matches_64_bits():
    ref, model = _models()
    model = model.cuda()
    ids, targets = make_packed_batch(LENS, CFG["vocab"], seed=1)
    plan = ct.packed_plan(LENS, CFG["n_heads"], CFG["n_kv_heads"])
    loss = model.loss(ids.cuda(), targets.cuda(), plan)
    loss.backward()
    want = ref.loss(ids, targets, plan)
    want.backward()
    # The bounds of the dense model's step in fp32: 1e-5 of the loss, 1e-3 of a gradient's largest element.
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for (name, p), (_, r) in zip(model.named_parameters(), ref.named_parameters()):
        scale = float(r.grad.abs().max())
        assert float((p.grad.double().cpu() - r.grad).abs().max()) <= 1e-3 * scale + 1e-9, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_with_muon_and_adam(dtype):
    _, model = _models()
    model = model.to(dtype).cuda()
    inside, rest = muon_parameters(model)
    opts = [ct.Muon(inside, lr=0.01, weight_decay=0.01), torch.optim.Adam(rest, lr=1e-3)]
    for step in range(3):
        lens = [LENS, [33, 90], [1, 1, 128, 7]][step]  # another batch, another plan
        plan = ct.packed_plan(lens, CFG["n_heads"], CFG["n_kv_heads"])
        ids, targets = make_packed_batch(lens, CFG["vocab"], seed=step)
        before = [p.detach().clone() for p in inside]
        moments = [opts[0].state[p].get("moment", torch.zeros_like(p, dtype=torch.float32)).clone() for p in inside]
        loss = train_step(model, opts, ids.cuda(), targets.cuda(), plan)
        assert torch.isfinite(loss)
        # Each matrix moved as its own step from this gradient moves it, together or by itself (up to the order
        # in which sums are split, which goes by the number of matrices).
        for p, b, m in zip(inside, before, moments):
            ct.muon_update([b], [p.grad], [m], lr=0.01, weight_decay=0.01)
            err = float((p.detach().double() - b.double()).norm())
            assert err <= (torch.finfo(dtype).eps + 1e-5) * float(b.double().norm())
            assert torch.equal(m, opts[0].state[p]["moment"])


@pytest.mark.gpu
def test_repeated_ids_and_dense_grouped_heads():
    """One token all over a batch; and the dense path with the same shared key heads."""
    ref, model = _models()
    model = model.cuda()
    plan = ct.packed_plan(LENS, CFG["n_heads"], CFG["n_kv_heads"])
    n = sum(LENS)
    ids, targets = torch.full((n,), 7), torch.arange(n) % CFG["vocab"]
    model.loss(ids.cuda(), targets.cuda(), plan).backward()
    ref.loss(ids, targets, plan).backward()
    g, r = model.tok.weight.grad.double().cpu(), ref.tok.weight.grad
    assert float((g - r).abs().max()) <= 1e-3 * float(r.abs().max())
    assert bool((g[torch.arange(CFG["vocab"]) != 7] == 0).all())
    dense = copy.deepcopy(model)
    x = torch.randint(0, CFG["vocab"], (2, 64), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        got, want = dense(x.cuda()).double().cpu(), ref(x)
    assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())
