"""Many continuations of shared prompts from the torch-hosted NanoGPT, one token a step, on the paged cache.

The prompts run once, packed behind each other; their keys and values stay in pages that all samples of a prompt read
(``flash_attn_shared_prefix``).  A step reserves pages for its tokens, writes their keys and values and samples the next ones
on the device; from the second on it is one captured graph, replayed.
"""
from __future__ import annotations

import torch

from .packed import flash_attn_packed_fwd, packed_plan
from .paged import cache_write, flash_attn_shared_prefix, page_pool, page_reserve
from .sampling import sample_tokens


class PromptCache:
    """Keys and values of a model's layers for prompts and for `samples` requests of each, `new_tokens` long at most."""

    def __init__(self, lens, samples: int, new_tokens: int, layers: int, heads: int, kv_heads: int, d: int, dtype, device, page_size: int):
        b = len(lens) * samples
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        of = lambda n: -(-n // page_size)  # noqa: E731
        pages = sum(of(n) for n in lens) + b * of(new_tokens)
        self.page_size, self.rows = page_size, b
        self.k, self.v = (torch.empty((layers, pages, page_size, kv_heads, d), dtype=dtype, device=device) for _ in range(2))
        free, counters = page_pool(pages, device)
        self.prefix_table = torch.zeros((len(lens), of(max(lens))), dtype=torch.int32, device=device)
        self.plan = packed_plan(lens, heads, kv_heads, device)
        # The prompts' pages, and where their tokens go.
        out = page_reserve(ints([0] * len(lens)), ints(lens), self.prefix_table, free, counters, page_size, sum(lens))
        self.slots, self.positions, _, self.prefix_lens, counters = out
        # A step's: one token a request.
        self.free, self.counters, self.one = free, counters, ints([1] * b)
        self.offsets = self.prefix_lens.repeat_interleave(samples)
        self.table = torch.zeros((b, of(new_tokens)), dtype=torch.int32, device=device)
        self.lens = ints([0] * b)
        self.out = (torch.empty(b, dtype=torch.int64, device=device), torch.empty(b, dtype=torch.int64, device=device),
                    ints([0] * (b + 1)), ints([0] * b), torch.empty_like(counters))

    def step(self):
        """Room for one more token of every request; the prompts are done."""
        self.plan = None
        self.slots, self.positions, _, lens, counters = page_reserve(self.lens, self.one, self.table, self.free, self.counters,
                                                                     self.page_size, self.rows, self.offsets, out=self.out)
        self.lens.copy_(lens)
        self.counters.copy_(counters)

    def attend(self, layer: int, q, k, v):
        """Writes k and v [tokens, heads, d] into the layer's cache and attends from q."""
        cache_write(k, v, self.k[layer], self.v[layer], self.slots)
        if self.plan is not None:
            return flash_attn_packed_fwd(q, k, v, self.plan, True)[0]
        return flash_attn_shared_prefix(q, self.k[layer], self.v[layer], self.table, self.lens, self.prefix_table, self.prefix_lens)[0]


@torch.no_grad()
def generate(model, prompts, new_tokens: int, samples: int = 1, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=None,
             generator=None, page_size: int = 16, graph: bool = True):
    """(tokens, logprobs) [len(prompts) * samples, new_tokens]: `samples` continuations of each prompt (a list of sequences of
    token ids), a prompt's behind each other, and the log-probability of each token at its temperature (``sample_tokens``,
    whose parameters may be tensors of one number a continuation).  No token ends one: all are new_tokens long.  Random numbers
    come from `generator` of the model's device, or are u [new_tokens, continuations].  With graph=False every step runs
    eagerly."""
    c, p = model.config, next(model.parameters())
    if model.attention != "ctattn" or not c["causal"]:
        raise ValueError("generate: a causal model on the ctattn kernels is wanted")
    if p.dtype not in (torch.float32, torch.bfloat16, torch.float16) or not p.is_cuda:
        raise ValueError(f"generate: a float32, bfloat16 or float16 model on the GPU is wanted, not {p.dtype} on {p.device}")
    ids = [torch.as_tensor(x, dtype=torch.int64, device=p.device) for x in prompts]
    lens = [len(x) for x in ids if x.dim() == 1]
    if not ids or len(lens) != len(ids) or min(lens) < 1 or samples < 1 or new_tokens < 1:
        raise ValueError("generate: prompts of one token at least, a sample and a new token at least are wanted")
    if max(lens) + new_tokens - 1 > c["max_seq_len"]:
        raise ValueError(f"generate: {max(lens)} + {new_tokens} tokens, {c['max_seq_len']} positions")
    b = len(ids) * samples
    if u is None:
        u = torch.rand((new_tokens, b), generator=generator, device=p.device)
    elif u.shape != (new_tokens, b) or u.dtype is not torch.float32:
        raise ValueError(f"generate: u must be float32 {[new_tokens, b]}, got {u.dtype} {list(u.shape)}")
    kw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    with torch.cuda.device(p.device):
        cache = PromptCache(lens, samples, new_tokens, c["n_layers"], c["n_heads"], c.get("n_kv_heads", c["n_heads"]), c["head_dim"],
                            p.dtype, p.device, page_size)
        tokens = torch.empty((new_tokens, b), dtype=torch.int64, device=p.device)
        logprobs = torch.empty((new_tokens, b), device=p.device)
        last = torch.tensor(lens, device=p.device).cumsum(0) - 1
        logits = model.forward_cached(torch.cat(ids), cache, last).repeat_interleave(samples, 0)
        sample_tokens(logits, u[0].contiguous(), **kw, tokens=tokens[0], logprobs=logprobs[0])
        # What a step reads and leaves, at one place for all steps.
        now, draw, logprob = tokens[0].clone(), torch.empty(b, device=p.device), torch.empty(b, device=p.device)

        def step():
            cache.step()
            sample_tokens(model.forward_cached(now, cache), draw, **kw, tokens=now, logprobs=logprob)

        replay = step
        for t in range(1, new_tokens):
            draw.copy_(u[t])
            if graph and t == 2:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step()
                replay = g.replay
            replay()
            tokens[t], logprobs[t] = now, logprob
        if replay is not step:
            torch.cuda.current_stream().synchronize()  # the graph goes when this returns
    return tokens.t().contiguous(), logprobs.t().contiguous()


__all__ = ["PromptCache", "generate"]
