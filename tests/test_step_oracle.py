"""The oracle of a serving step's operators (step_oracle) against other
statements of the same operators, and planted mistakes that it must notice."""

import numpy as np
import torch
import torch.nn.functional as F

import step_oracle as ref
from moe_engine import kv_ops
from moe_engine.model import BlockAllocator, ModelConfig


def test_reserve_and_release_are_the_engines_allocator():
    """PagedKVCache._reserve and free, sequence after sequence, on the CPU."""
    rng = np.random.default_rng(0)
    allocator = BlockAllocator(ModelConfig(num_layers=1, hidden_dim=8, num_heads=1), 40, 4, "cpu")
    order = rng.permutation(40).tolist()
    allocator.free_blocks[:] = order
    stack, count = np.array(order, np.int32), 40
    caches, lens = [allocator.new_cache() for _ in range(5)], np.zeros(5, np.int64)
    tables = np.zeros((5, 10), np.int32)
    for _ in range(30):
        new = rng.integers(0, 8, 5)
        tables, starts, slots, positions, after, count, status = ref.reserve(stack, count, tables, lens, new, 4, 64)
        if status == 0:
            for cache, n in zip(caches, after):
                cache._reserve(int(n))
        lens = after
        assert allocator.free_blocks == stack[:count].tolist()
        for b, cache in enumerate(caches):
            assert tables[b, : len(cache.block_table)].tolist() == cache.block_table
        t = 0
        for b, n in enumerate(new if status == 0 else []):
            for i in range(n):
                block, place = caches[b]._block_for(int(lens[b] - n + i))
                assert slots[t] == block * 4 + place and positions[t] == lens[b] - n + i
                t += 1
        assert (slots[t:] == -1).all()
        finished = rng.random(5) < 0.3
        stack, lens, count, _ = ref.release(stack, count, tables, lens, finished, 4)
        for cache, done in zip(caches, finished):
            if done:
                cache.free()


def test_rope_is_a_complex_rotation():
    rng = np.random.default_rng(1)
    x, pos, freq = rng.standard_normal((5, 3, 12)), np.array([0, 1, 7, 1000, 10**6]), 10.0 ** -np.arange(4.0)
    turn = np.exp(1j * pos[:, None, None] * freq)
    z = (x[..., 0:8:2] + 1j * x[..., 1:8:2]) * turn * 1.5
    got = ref.rope(x, pos, freq, 1.5, True)
    assert np.allclose(got[..., 0:8:2], z.real, atol=1e-9) and np.allclose(got[..., 1:8:2], z.imag, atol=1e-9)
    z = (x[..., :4] + 1j * x[..., 4:8]) * turn
    got = ref.rope(x, pos, freq, 1.0, False)
    assert np.allclose(got[..., :4], z.real, atol=1e-9) and np.array_equal(got[..., 8:], x[..., 8:])
    # The opposite turn and the other layout are not it.
    assert not np.allclose(got, ref.rope(x, -pos, freq, 1.0, False))
    assert not np.allclose(got, ref.rope(x, pos, freq, 1.0, True))


def test_extend_is_masked_attention():
    g = torch.Generator().manual_seed(0)
    q = torch.randn(6, 4, 8, generator=g, dtype=torch.float64)
    k, v = torch.randn(2, 20, 2, 8, generator=g, dtype=torch.float64)
    p, j = torch.arange(14, 20)[:, None], torch.arange(20)[None]

    def sdpa(mask, bias=None):
        kk, vv = (x.transpose(0, 1).repeat_interleave(2, 0) for x in (k, v))
        m = torch.zeros(4, 6, 20, dtype=torch.float64) if bias is None else bias
        m = m.masked_fill(~mask, float("-inf"))
        return F.scaled_dot_product_attention(q.transpose(0, 1), kk, vv, attn_mask=m).transpose(0, 1)

    base = dict(scale=8**-0.5)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0], dtype=torch.float64)
    for kw, want in (
        ({}, sdpa(j <= p)),
        (dict(window=5), sdpa((j <= p) & (j > p - 5))),
        (dict(prefix=17), sdpa((j <= p) | (j < 17))),
        (dict(prefix=20, window=3), sdpa(j > p - 3)),
        (dict(slopes=slopes), sdpa(j <= p, -slopes[:, None, None] * (p - j).abs())),
        (dict(slopes=slopes, prefix=20), sdpa(j >= 0, -slopes[:, None, None] * (p - j).abs())),
    ):
        out, bound = ref.extend(q, k, v, 20, **base, **kw)
        assert torch.allclose(out, want, atol=1e-12, rtol=1e-12)
        # A mistake of one key, or of one head's partner, is far outside the bound.
        for wrong in (ref.extend(q, k.roll(1, 0), v, 20, **base, **kw)[0], ref.extend(q, k.flip(1), v, 20, **base, **kw)[0]):
            assert bool(((out - wrong).abs() > bound).any())
    capped, _ = ref.extend(q, k, v, 20, softcap=0.5, **base)
    kk = k.transpose(0, 1).repeat_interleave(2, 0)
    s = 0.5 * torch.tanh(q.transpose(0, 1) @ kk.transpose(1, 2) * 8**-0.5 / 0.5)
    w = s.masked_fill(j > p, float("-inf")).softmax(-1)
    assert torch.allclose(capped, (w @ v.transpose(0, 1).repeat_interleave(2, 0)).transpose(0, 1), atol=1e-12)


def test_rope_frequencies():
    freq, factor = kv_ops.rope_frequencies(8, 10000.0)
    assert factor == 1.0 and torch.allclose(freq, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert torch.equal(kv_ops.rope_frequencies(8, scaling="linear", scale=4.0)[0], freq / 4)
    ntk, _ = kv_ops.rope_frequencies(8, scaling="ntk", scale=4.0)
    assert float(ntk[0]) == 1.0 and abs(float(ntk[-1] / freq[-1]) - 0.25) < 1e-12
    yarn, factor = kv_ops.rope_frequencies(64, scaling="yarn", scale=16.0, original_length=4096)
    plain, _ = kv_ops.rope_frequencies(64)
    turns = plain * 4096 / (2 * np.pi)
    assert torch.equal(yarn[turns > 34], plain[turns > 34]) and torch.allclose(yarn[turns < 0.9], plain[turns < 0.9] / 16)
    assert bool(((yarn <= plain) & (yarn >= plain / 16 * (1 - 1e-12))).all()) and abs(factor - (0.1 * np.log(16) + 1)) < 1e-15
