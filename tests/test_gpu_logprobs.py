"""projection.token_logprobs on the GPU against log softmax in 64 bits.

Tolerance: with n = vocab / 1024 + 64 partial sums in float32, the sum of
exponentials (each within 2^-22) is off by (n 2^-24 + 2^-22) relatively, which
is its logarithm's error; x - m, the logarithm and the difference are rounded
once each.  The entropy's second sum has the same relative error per unit of
mean distance."""

import math

import pytest
import torch

from conftest import print_case
from moe_engine import projection

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def check(logits, tokens, top):
    got = projection.token_logprobs(logits, tokens, top=top)
    x = logits.double().cpu()
    vocab = x.shape[1]
    m = x.amax(-1, keepdim=True)
    logp = torch.log_softmax(x, -1)
    z = torch.log((x - m).exp().sum(-1))
    sum_err = (vocab / 1024 + 64) * 2.0**-24 + 2.0**-22

    def near(have, want, far, extra, name):
        have, far = have.double().cpu(), far.abs()
        inf = want.isinf()
        assert torch.equal(have[inf], want[inf]), name
        err = (have - want)[~inf].abs()
        bound = (sum_err + 2.0**-22 * (far + z.abs().expand_as(far) + 1) + extra)[~inf]
        assert bool((err <= bound).all()), (name, float((err / bound).max()))

    if tokens is not None:
        at = tokens.cpu()[:, None]
        near(got.logprobs, logp.gather(1, at)[:, 0], torch.nan_to_num((x - m).gather(1, at)[:, 0], neginf=0), 0, "logprobs")
    else:
        assert got.logprobs is None
    mean = -(logp.exp() * torch.nan_to_num(x - m, neginf=0)).sum(-1)
    near(got.entropy, -torch.xlogy(logp.exp(), logp.exp()).sum(-1), mean, 2 * sum_err * mean, "entropy")
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    assert torch.equal(got.top_tokens.cpu(), order.indices[:, :top])
    values = logp.gather(1, order.indices[:, :top])
    if top:
        z = z[:, None]
        near(got.top_logprobs, values, torch.nan_to_num(order.values[:, :top] - m, neginf=0), 0, "top")
    return got


@pytest.mark.parametrize("rows,vocab", [
    (1, 1), (1, 2), (3, 7), (2, 63), (5, 64), (1, 1000), (4, 1023), (4, 1024), (4, 1025), (2, 4097), (9, 50257),
    (3, 50304), (300, 5000), (1, 200001), (2, 131072), (600, 130), (3, 65536), (2, 70001),
])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_logprobs(rows, vocab, top, dtype):
    print_case("logprobs", rows, vocab, top, dtype)
    g = torch.Generator().manual_seed(vocab + top)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(DEV)
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(DEV)
    check(logits, tokens, min(top, vocab))


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "big in one place", "two zeros", "masked", "one left"])
@pytest.mark.parametrize("rows,vocab", [(1, 3000), (2, 50257), (3, 150000)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_orders_and_ties(kind, rows, vocab, dtype):
    print_case("logprobs order", kind, rows, vocab, dtype)
    g = torch.Generator().manual_seed(3)
    i = torch.arange(vocab, dtype=torch.float32)
    x = {
        "equal": torch.full((vocab,), 1.5),
        "rising": i / vocab * 20,
        "falling": -i / vocab * 20,
        "steps": torch.floor(i / 100) % 7,
        "big in one place": torch.where(i // 1024 == 1, 9.0, 0.0) + torch.randn(vocab, generator=g) * 0.01,
        "two zeros": torch.where(i % 2 == 0, -0.0, 0.0),
        "masked": torch.where(torch.rand(vocab, generator=g) < 0.99, -math.inf, torch.randn(vocab, generator=g)),
        "one left": torch.where(i == 1234, -300.0, -math.inf),
    }[kind].repeat(rows, 1).to(dtype).to(DEV)
    tokens = torch.full((rows,), 1234, device=DEV)
    check(x, tokens, 20)
    check(x, tokens, 64)


def test_large_values():
    print_case("logprobs large")
    x = torch.randn(4, 5000, device=DEV)
    x[0] += 1e30
    x[1] *= 1e37
    x[2] = torch.finfo(F32).min
    x[3] -= 60000
    check(x[2:], torch.tensor([7, 8], device=DEV), 5)
    got = projection.token_logprobs(x, torch.zeros(4, dtype=torch.long, device=DEV), top=2)
    assert bool(torch.isfinite(got.entropy).all()) and float(got.entropy[1]) == 0


@pytest.mark.parametrize("where", ["most", "front", "behind"])
@pytest.mark.parametrize("rows,vocab", [(1, 300), (3, 50257), (2, 150000), (600, 5000)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_tokens_masked_by_the_types_lowest_value(where, rows, vocab, dtype):
    print_case("logprobs lowest", where, rows, vocab, dtype)
    g = torch.Generator().manual_seed(vocab)
    i = torch.arange(vocab)
    masked = {"most": torch.rand(vocab, generator=g) < 0.99, "front": i < vocab - 20, "behind": i >= 20}[where]
    masked[123] = False
    x = torch.randn(rows, vocab, generator=g).to(dtype).masked_fill(masked, torch.finfo(dtype).min).to(DEV)
    tokens = torch.arange(rows).clamp(max=200)
    tokens[::2] = 123
    check(x, tokens.to(DEV), 20)


@pytest.mark.parametrize("vocab", [50, 3000, 50257, 150000])
def test_values_that_are_not_finite(vocab):
    print_case("logprobs nan", vocab)
    x = torch.randn(5, vocab, device=DEV)
    x[0] = -math.inf
    x[1, 17] = math.nan
    x[2, 18] = math.inf
    x[3, 0] = x[3, vocab - 1] = math.nan
    got = projection.token_logprobs(x, torch.arange(5, device=DEV), top=4)
    for r in range(4):
        assert got.logprobs[r].isnan() and got.entropy[r].isnan() and bool(got.top_logprobs[r].isnan().all()), r
    assert bool(torch.isfinite(got.logprobs[4]))
    rest = [i for i in torch.sort(x[1].nan_to_num(math.inf), descending=True, stable=True).indices.tolist()]
    assert got.top_tokens[0].tolist() == [0, 1, 2, 3]
    assert got.top_tokens[1].tolist() == rest[:4]
    assert got.top_tokens[2, 0] == 18
    assert got.top_tokens[3, :2].tolist() == [0, vocab - 1]


def test_tokens_outside_the_vocabulary_and_none():
    print_case("logprobs tokens")
    x = torch.randn(4, 1000, device=DEV)
    tokens = torch.tensor([-1, 1000, 2**40, 999], device=DEV)
    got = projection.token_logprobs(x, tokens)
    assert got.logprobs[:3].isnan().all() and got.logprobs[3].isfinite() and got.top_tokens.shape == (4, 0)
    check(x, None, 3)
    empty = projection.token_logprobs(x[:0], tokens[:0], top=3)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides_and_offsets(dtype):
    print_case("logprobs strides", dtype)
    wide = torch.randn(6, 5003, device=DEV).to(dtype)
    tokens = torch.arange(6, device=DEV)
    check(wide[:, 1:5000], tokens, 5)          # rows at every alignment
    check(wide[::2, 3:4003], tokens[::2], 5)
    check(wide[:, ::2], tokens, 5)             # copied
    check(wide[:1].expand(6, 5003), tokens, 5)
    check(wide.t().contiguous().t(), tokens, 2)


def test_captured_and_on_two_streams():
    print_case("logprobs captured")
    for rows, vocab in ((1, 150000), (40, 50257)):
        x = torch.randn(rows, vocab, device=DEV)
        tokens = torch.randint(0, vocab, (rows,), device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            projection.token_logprobs(x, tokens, top=5)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = projection.token_logprobs(x, tokens, top=5)
        for _ in range(4):
            x.copy_(torch.randn_like(x) * 4)
            torch.cuda.synchronize()
            side.wait_stream(torch.cuda.current_stream())
            graph.replay()
            with torch.cuda.stream(side):
                want = projection.token_logprobs(x, tokens, top=5)
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
