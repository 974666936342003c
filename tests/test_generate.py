"""NanoGPT.generate: continuations of shared prompts on the paged cache against the whole sequences run at once."""
import math

import pytest
import torch

from cudatransformer_amd.nanogpt import NanoGPT

gpu = pytest.mark.gpu
SMALL = dict(vocab=65, max_seq_len=96, d_model=64, n_heads=4, head_dim=32, mlp_dim=96, n_layers=3)
PROMPTS = [[1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19], [60], [5, 4, 3]]


def model_of(dtype, seed=0, **kw):
    m = NanoGPT(**{**SMALL, **kw}).init_weights(seed)
    with torch.no_grad():  # without residuals the logits of small weights are all alike
        for n, p in m.named_parameters():
            if p.dim() == 2:
                p.mul_(6.0)
    return m.to(dtype).cuda()


def whole_logits(m, prompt, tokens):
    """Logits before each of the tokens, from the dense path in one piece."""
    ids = torch.tensor([list(prompt) + tokens[:-1]], device="cuda")
    with torch.no_grad():
        return m(ids)[0, len(prompt) - 1:].double()


@gpu
@pytest.mark.parametrize("dtype,kw", [(torch.float32, {}), (torch.float32, dict(n_kv_heads=2, embedding_scale=8.0)),
                                      (torch.bfloat16, dict(n_kv_heads=1)), (torch.float16, dict(head_dim=24))])
@pytest.mark.parametrize("page_size", [1, 16])
def test_against_whole_sequences(dtype, kw, page_size):
    m = model_of(dtype, **kw)
    n, samples = 21, 3
    u = torch.rand((n, 9), generator=torch.Generator().manual_seed(3)).cuda()
    how = dict(temperature=torch.tensor([0.0, 0.7, 1.0] * 3, device="cuda"), top_k=torch.tensor([0, 9, 0] * 3, dtype=torch.int32, device="cuda"),
               top_p=0.9)
    tokens, logprobs = m.generate(PROMPTS, n, samples=samples, u=u, page_size=page_size, **how)
    assert tokens.shape == logprobs.shape == (9, n) and int(tokens.min()) >= 0 and int(tokens.max()) < 65
    # Two ways of the same sums: rounded to the type in every layer, of logits up to a few units.
    tol = 40 * torch.finfo(dtype).eps
    for i in range(9):
        z = whole_logits(m, PROMPTS[i // samples], tokens[i].tolist())
        t = float(how["temperature"][i]) or 1.0
        scale = float(z.abs().max()) + 1
        lp = torch.log_softmax(z / t, 1).gather(1, tokens[i][:, None])[:, 0]
        assert (lp - logprobs[i].double()).abs().max() <= tol * scale / t
        if float(how["temperature"][i]) == 0:  # the largest, up to that rounding
            assert (z.gather(1, tokens[i][:, None])[:, 0] >= z.amax(1) - tol * scale).all()
        elif int(how["top_k"][i]):
            kth = z.topk(9, 1).values[:, -1]
            assert (z.gather(1, tokens[i][:, None])[:, 0] >= kth - tol * scale).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_and_eager_steps_agree(dtype):
    m = model_of(dtype, n_kv_heads=2)
    make = lambda: torch.Generator(device="cuda").manual_seed(5)  # noqa: E731
    a = m.generate(PROMPTS, 40, samples=4, generator=make(), top_k=20)
    b = m.generate(PROMPTS, 40, samples=4, generator=make(), top_k=20, graph=False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # A second run beside other work, on another stream.
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gen = make()
    with torch.cuda.stream(side):
        c = m.generate(PROMPTS, 40, samples=4, generator=gen, top_k=20)
    side.synchronize()
    assert torch.equal(a[0], c[0])


@gpu
def test_samples_of_a_prompt_do_not_meet():
    """A prompt's continuations are what each is alone, whatever runs beside it."""
    m = model_of(torch.float32)
    u = torch.rand((12, 6), generator=torch.Generator().manual_seed(1)).cuda()
    all_of = m.generate(PROMPTS[:2], 12, samples=3, u=u)[0]
    for i in (0, 2, 4):
        one = m.generate([PROMPTS[i // 3]], 12, u=u[:, i:i + 1].contiguous())[0]
        assert torch.equal(one[0], all_of[i])


@gpu
def test_one_token_and_the_last_position():
    m = model_of(torch.float32)
    assert m.generate([[3, 4]], 1)[0].shape == (1, 1)
    long = list(range(60)) + list(range(30))
    tokens, logprobs = m.generate([long], 7, samples=2, temperature=0.0)
    assert tokens.shape == (2, 7) and torch.equal(tokens[0], tokens[1]) and torch.isfinite(logprobs).all()
    assert float(logprobs.max()) <= 0.0 and not math.isnan(float(logprobs.sum()))


@gpu
def test_refusals_on_the_gpu():
    m = model_of(torch.float32)
    for call in (lambda: m.generate([], 3), lambda: m.generate([[]], 3), lambda: m.generate([[1]], 0), lambda: m.generate([[1]], 3, samples=0),
                 lambda: m.generate([[1] * 95], 3), lambda: m.generate([[[1]]], 3), lambda: m.generate([[1]], 3, u=torch.rand(3, device="cuda")),
                 lambda: m.double().generate([[1]], 3)):
        with pytest.raises(ValueError):
            call()


def test_refusals():
    for kw in (dict(attention="sdpa"), dict(causal=False), dict()):  # the last: not on a GPU
        with pytest.raises(ValueError):
            NanoGPT(**SMALL, **kw).generate([[1, 2]], 3)
