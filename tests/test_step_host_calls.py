"""The compiled host side of a serving step's operators: it takes the usual
forms of a call and leaves every other to the Python path, with the same
results and refusals."""

import pytest
import torch

from conftest import print_case
from moe_engine import _native, kv_ops, paged_attention, projection

DEV = "cuda"


def test_it_declines_what_is_not_a_rocm_tensor():
    host = _native.HOST
    assert host is not None, "moe_engine/_host_calls.so is not built"
    i32, f32 = torch.zeros(4, dtype=torch.int32), torch.zeros(1, 4, 2, 16, 64)
    assert host.reserve(i32, i32[:1], i32.view(2, 2), i32[:2], i32[:2], 16, 4, 0) is None
    assert host.release(i32, i32[:1], i32.view(2, 2), i32[:2], i32[:2].bool(), 16, 0) is None
    assert host.rope_append(f32[0, :, :, 0], f32[0, :, :, 0], f32[0, :, :, 0], f32, f32, 0, i32.long(), i32,
                            torch.zeros(32).double(), False, 1.0, 0) is None
    assert host.extend(f32[0, :, :, 0], f32, f32, 0, i32.view(2, 2), i32[:3], i32[:2], 1, 1, None, 0.0, None, 0, None, 0) is None
    assert host.logprobs(torch.zeros(2, 5), i32[:2].long(), 1, 0) is None
    for name, n in (("reserve", 8), ("release", 7), ("rope_append", 12), ("extend", 15), ("logprobs", 4)):
        for args in ((), (None,) * n, (1,) * n, ("x",) * n):
            assert getattr(host, name)(*args) is None


def both(monkeypatch, f):
    """f through the compiled call and through Python."""
    got = f()
    with monkeypatch.context() as m:
        m.setattr(_native, "HOST", None)
        want = f()
    return got, want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_results(monkeypatch, dtype):
    print_case("step host calls", dtype)
    ids, count = torch.randperm(200, device=DEV).int(), torch.tensor([200], dtype=torch.int32, device=DEV)
    tables = torch.zeros(3, 20, dtype=torch.int32, device=DEV)
    wide = torch.zeros(3, 30, dtype=torch.int32, device=DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    new = torch.tensor([40, 1, 77], dtype=torch.int32, device=DEV)
    for t in (tables, wide[:, :20]):
        got, want = both(monkeypatch, lambda: kv_ops.reserve(ids, count, t, lens, new, 8, 120))
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and type(got) is type(want)
    step = got
    done = torch.tensor([True, False, True], device=DEV)
    got, want = both(monkeypatch, lambda: kv_ops.release(ids.clone(), step.free_count, tables, step.context_lens, done, 8))
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    kp, vp = torch.randn(2, 2, 200, 2, 8, 64, device=DEV).to(dtype)
    qkv = torch.randn(120, 8, 64, device=DEV).to(dtype)
    q, k, v = qkv.split([4, 2, 2], 1)
    freq, _ = kv_ops.rope_frequencies(32, device=DEV)
    odd = torch.randn(120, 4, 128, device=DEV).to(dtype)[..., ::2]  # not unit stride
    for qq, kw in ((q, {}), (q.contiguous(), dict(interleaved=True, factor=2)), (odd, dict(factor=0.5))):
        def rope():
            pools = kp.clone(), vp.clone()
            out = kv_ops.rope_append(qq, k, v, *pools, 1, step.slots, step.positions, freq, **kw)
            return (out, *pools)
        got, want = both(monkeypatch, rope)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    slopes, prefix = torch.rand(4, device=DEV), torch.tensor([3, 0, 50], dtype=torch.int32, device=DEV)
    starts = step.starts
    rows = int(starts[-1])
    for qq in (q, q.contiguous(), odd, torch.nn.Parameter(q.contiguous(), requires_grad=False)):
        for kw in ({}, dict(scale=1, softcap=5), dict(slopes=slopes, window=9), dict(prefix_lens=prefix)):
            got, want = both(monkeypatch, lambda: paged_attention.extend_batched(
                qq, kp, vp, 1, tables, starts, step.context_lens, 77, 100, **kw))
            assert torch.equal(got[:rows], want[:rows])
    x = torch.randn(6, 5003, device=DEV).to(dtype)
    for logits in (x, x[:, 1:4000], x[:, ::2], x[:1].expand(6, 5003)):
        got, want = both(monkeypatch, lambda: projection.token_logprobs(logits, torch.arange(6, device=DEV), top=4))
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and type(got) is type(want)


@pytest.mark.gpu
def test_same_refusals(monkeypatch):
    print_case("step host refusals")
    ids, one = torch.arange(20, device=DEV).int(), torch.ones(1, dtype=torch.int32, device=DEV)
    two = torch.ones(2, dtype=torch.int32, device=DEV)
    tables = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    pool = torch.zeros(1, 20, 2, 4, 64, device=DEV)
    q, starts = torch.zeros(2, 2, 64, device=DEV), torch.arange(3, device=DEV).int()
    slots, freq = torch.arange(2, device=DEV), torch.ones(16, device=DEV).double()
    wide = torch.zeros(9000, 4, dtype=torch.int32, device=DEV)
    many = torch.zeros(9000, dtype=torch.int32, device=DEV)
    calls = [
        (lambda: kv_ops.reserve(ids, one, tables, two, two, 0, 8), ValueError),
        (lambda: kv_ops.reserve(ids, one, tables, two, two, 4, -1), ValueError),
        (lambda: kv_ops.reserve(ids, one, wide, many, many, 4, 8), RuntimeError),
        (lambda: kv_ops.release(ids, one, tables, two, two, 4), ValueError),
        (lambda: kv_ops.rope_append(q, q, q, pool, pool, 1, slots, two, freq), IndexError),
        (lambda: kv_ops.rope_append(q, q, q, pool, pool, 0, slots, two, torch.ones(33, device=DEV).double()), RuntimeError),
        (lambda: kv_ops.rope_append(q.requires_grad_(), q, q, pool, pool, 0, slots, two, freq), RuntimeError),
        (lambda: paged_attention.extend_batched(q.detach(), pool, pool, 0, tables, starts, two, 1, 4, softcap=float("inf")), ValueError),
        (lambda: paged_attention.extend_batched(q.detach(), pool, pool, 0, tables, starts, two, -1, 4), ValueError),
        (lambda: paged_attention.extend_batched(q.detach(), pool, pool, 0, tables, starts, two, 1, 4, scale=float("nan")), RuntimeError),
        (lambda: paged_attention.extend_batched(q.detach().requires_grad_(), pool, pool, 0, tables, starts, two, 1, 4), RuntimeError),
        (lambda: paged_attention.extend_batched(q.detach(), pool, pool, 0, tables.cpu(), starts, two, 1, 4), ValueError),
        (lambda: projection.token_logprobs(q.detach()[0], slots, top=65), ValueError),
        (lambda: projection.token_logprobs(q.detach()[0].requires_grad_(), slots), RuntimeError),
    ]
    for i, (call, error) in enumerate(calls):
        for host in (_native.HOST, None):
            monkeypatch.setattr(_native, "HOST", host)
            with pytest.raises(error):
                call()
    with torch.no_grad():
        projection.token_logprobs(q.detach()[0].requires_grad_(), slots)


@pytest.mark.gpu
def test_in_inference_mode_and_on_another_stream(monkeypatch):
    """A step under inference mode, each call on a stream of its own."""
    print_case("step host calls, inference mode")
    ids, count = torch.arange(50, device=DEV).int(), torch.tensor([50], dtype=torch.int32, device=DEV)
    tables, lens = torch.zeros(2, 8, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    new = torch.tensor([30, 9], dtype=torch.int32, device=DEV)
    freq, _ = kv_ops.rope_frequencies(64, device=DEV)
    pools = [torch.zeros(1, 50, 2, 8, 64, device=DEV) for _ in range(4)]
    qkv = torch.randn(40, 8, 64, device=DEV)
    q, k, v = qkv.split([4, 2, 2], 1)

    def step(kp, vp):
        r = kv_ops.reserve(ids, count, tables, lens, new, 8, 40)
        x = kv_ops.rope_append(q, k, v, kp, vp, 0, r.slots, r.positions, freq)
        y = paged_attention.extend_batched(x, kp, vp, 0, tables, r.starts, r.context_lens, 30, 30)[:39]
        p = projection.token_logprobs(y.reshape(39, 256), torch.arange(39, device=DEV), top=3)
        done = kv_ops.release(ids.clone(), r.free_count, tables, r.context_lens, new > 10, 8)
        return [*r, x, y, *p, *done]

    want = step(*pools[:2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(stream):
        got = step(*pools[2:])
        assert all(t.is_inference() for t in got if t is not None)
        got[0].add_(0)  # a piece of a shared allocation is a tensor like another
    torch.cuda.current_stream().wait_stream(stream)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
