"""A run of a serving step's operators as they are used together, and
Model.score on the GPU."""

import math

import pytest
import torch

from conftest import print_case
from moe_engine import kv_ops, paged_attention, projection
from moe_engine.model import BlockAllocator, Model, ModelConfig

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("paged", [False, True])
def test_score_on_the_gpu_is_the_cpus(paged):
    print_case("score", paged)
    torch.manual_seed(0)
    model = Model(ModelConfig(max_seq_length=64, vocab_size=500, num_layers=2, hidden_dim=64, num_heads=4,
                              num_experts=4, top_k=2)).eval()
    ids = torch.randint(0, 500, (50,))
    want = model.score(ids, top=3)
    model.to(DEV)
    cache = model.new_block_allocator(num_blocks=4, block_size=16).new_cache() if paged else None
    got = model.score(ids.to(DEV), top=3, cache=cache)
    # Two float32 runs of the same small model: its logits (below 10 in size,
    # 64-term sums over 2 layers) differ by a few hundred roundings at most.
    for g, w in zip(got[:3], want[:3]):
        assert g.is_cuda and float((g.cpu() - w).abs().max()) < 500 * 10 * 2.0**-24
    assert projection.token_logprobs(torch.zeros(1, 5, device=DEV)).logprobs is None
    one = model.score(ids[:1].to(DEV), top=2)
    assert one.logprobs.shape == (0,) and one.top_tokens.shape == (0, 2)


class Layer:
    """One attention layer with rotary positions over float64 on the CPU,
    recomputed from the whole sequence."""

    def __init__(self, wq, wk, wv, freq, heads, kv_heads, dim):
        self.w, self.freq, self.heads, self.kv_heads, self.dim = (wq, wk, wv), freq, heads, kv_heads, dim

    def __call__(self, x):
        q, k, v = (x @ w for w in self.w)
        n = len(x)
        angle = torch.arange(n).double()[:, None] * self.freq
        c, s = angle.cos()[:, None], angle.sin()[:, None]

        def turn(y, heads):
            a, b = y.view(n, heads, self.dim).chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1)

        q, k, v = turn(q, self.heads), turn(k, self.kv_heads), v.view(n, self.kv_heads, self.dim)
        k, v = (y.repeat_interleave(self.heads // self.kv_heads, 1) for y in (k, v))
        score = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(self.dim)
        score = 20 * torch.tanh(score / 20)
        score = score.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
        return torch.einsum("hij,jhd->ihd", score.softmax(-1), v).reshape(n, -1)


def test_a_continuous_batch_step_by_step():
    """Requests of different lengths come, are prefilled in chunks beside
    others' decode tokens, finish and make room, over a pool that only just
    holds them: every token's attention output equals the layer over its whole
    sequence, and its log probability the head's over that."""
    print_case("continuous batch")
    g = torch.Generator().manual_seed(1)
    heads, kv_heads, dim, bs, rows, blocks, vocab = 4, 2, 64, 8, 4, 26, 1000
    hidden = 64
    w = [torch.randn(hidden, n * dim, generator=g) / 8 for n in (heads, kv_heads, kv_heads)]
    head = torch.randn(heads * dim, vocab, generator=g) / 8
    freq, _ = kv_ops.rope_frequencies(dim, device=DEV)
    oracle = Layer(*(x.double() for x in w), freq.cpu(), heads, kv_heads, dim)
    w, head_dev = [x.to(DEV) for x in w], head.to(DEV)

    allocator = BlockAllocator(ModelConfig(num_layers=1, hidden_dim=kv_heads * dim, num_heads=kv_heads), blocks, bs, DEV)
    free_ids, free_count = kv_ops.take_free_blocks(allocator)
    tables = torch.zeros(rows, 12, dtype=torch.int32, device=DEV)
    lens = torch.zeros(rows, dtype=torch.int32, device=DEV)
    waiting = [torch.randn(n, hidden, generator=g) for n in (70, 3, 33, 90, 1, 20, 64, 41, 8, 9)]
    running, done, failures, max_tokens = [None] * rows, 0, 0, 64
    while waiting or any(running):
        for r in range(rows):
            if running[r] is None and waiting:
                running[r] = [waiting.pop(0), 0]
        # A chunk of up to 25 tokens of those at their start, single tokens of the others.
        new = [0 if s is None else min(25 if s[1] < len(s[0]) // 2 else 1, len(s[0]) - s[1]) for s in running]
        step = kv_ops.reserve(free_ids, free_count, tables, lens, torch.tensor(new, dtype=torch.int32, device=DEV), bs,
                              max_tokens)
        if int(step.status):  # no room: the longest row waits a step
            failures += 1
            assert int(step.status) in (1, 3)
            new[max(range(rows), key=lambda r: new[r])] = 0
            step = kv_ops.reserve(free_ids, free_count, tables, lens, torch.tensor(new, dtype=torch.int32, device=DEV),
                                  bs, max_tokens)
            if int(step.status):  # or is put back
                r = max(range(rows), key=lambda r: 0 if running[r] is None else running[r][1])
                waiting.append(running[r][0])
                running[r] = None
                mask = torch.tensor([i == r for i in range(rows)], device=DEV)
                rel = kv_ops.release(free_ids, free_count, tables, lens, mask, bs)
                free_count, lens = rel.free_count, rel.context_lens
                continue
        free_count, lens = step.free_count, step.context_lens
        x = torch.zeros(max_tokens, hidden)
        t = 0
        for s, n in zip(running, new):
            if n:
                x[t : t + n] = s[0][s[1] : s[1] + n]
                t += n
        x = x.to(DEV)
        q, k, v = ((x @ m).view(max_tokens, -1, dim) for m in w)
        q = kv_ops.rope_append(q, k, v, allocator.k_pool, allocator.v_pool, 0, step.slots, step.positions, freq)
        out = torch.zeros(max_tokens, heads, dim, device=DEV)
        paged_attention.extend_batched(q, allocator.k_pool, allocator.v_pool, 0, tables, step.starts, lens, 25, 96,
                                       softcap=20.0, out=out)
        logits = out.flatten(1) @ head_dev
        target = torch.arange(max_tokens, device=DEV) * 7 % vocab
        r = projection.token_logprobs(logits, target, top=2)
        t, finished = 0, [False] * rows
        for i, (s, n) in enumerate(zip(running, new)):
            if n:
                want = oracle(s[0].double())[s[1] : s[1] + n]
                # float32 products of 64 terms in three projections, then attention.
                assert float((out[t : t + n].flatten(1).double().cpu() - want).abs().max()) < 1e-4
                logp = (want @ head.double()).log_softmax(-1)
                at = target[t : t + n].cpu()[:, None]
                assert float((r.logprobs[t : t + n].double().cpu() - logp.gather(1, at)[:, 0]).abs().max()) < 1e-3
                s[1] += n
                t += n
            if s is not None and s[1] == len(s[0]):
                finished[i], running[i] = True, None
                done += 1
        rel = kv_ops.release(free_ids, free_count, tables, lens, torch.tensor(finished, device=DEV), bs)
        free_count, lens = rel.free_count, rel.context_lens
    assert done == 10 and failures > 0 and int(free_count) == blocks
    assert sorted(free_ids.tolist()) == list(range(blocks))
