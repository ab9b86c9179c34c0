"""kv_ops.rope_append on the GPU against the rotation in 64 bits.

Tolerance: the reduced angle is a float32 of at most half a turn (off by 2^-25
turns x 2 pi < 2^-22), sine and cosine are within 2^-22, the factor, two
products and a sum are rounded once each (4 x 2^-24), all relative to factor
(|x1| + |x2|): together below 2^-20 of it; bfloat16 adds half a step of the
result, 2^-8 of it."""

import numpy as np
import pytest
import torch

from conftest import print_case
from moe_engine import kv_ops
import step_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def inputs(tokens, heads, kv_heads, dim, block_size, dtype, seed, blocks=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g).to(dtype).to(DEV)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    blocks = blocks or -(-tokens // block_size) + 5
    pools = torch.randn(2, 2, blocks, kv_heads, block_size, dim, generator=g).to(dtype).to(DEV)
    slots = torch.randperm(blocks * block_size, generator=g)[:tokens].to(DEV)
    return q, k, v, pools[0], pools[1], slots


def check(q, k, v, k_pool, v_pool, slots, positions, freq, factor, interleaved, out=None, layer=1):
    before = k_pool.clone(), v_pool.clone()
    got = kv_ops.rope_append(q, k, v, k_pool, v_pool, layer, slots, positions, freq, interleaved=interleaved,
                             factor=factor, out=out)
    pos, f = positions.cpu().numpy(), freq.cpu().numpy()
    step = 0.0 if q.dtype == F32 else torch.finfo(q.dtype).eps / 2

    def near(have, x, name):
        x = x.double().cpu().numpy()
        want = ref.rope(x, pos, f, factor, interleaved)
        size = np.abs(x)
        r = 2 * len(f)
        head = size[..., :r].reshape(*size.shape[:-1], r // 2, 2).sum(-1).repeat(2, -1) if interleaved \
            else np.tile(size[..., : r // 2] + size[..., r // 2 : r], 2)
        size = np.concatenate([head * abs(factor), np.zeros_like(size[..., r:])], -1)
        err = np.abs(have.double().cpu().numpy() - want)
        # The half step is of the value before its rounding: want, off by the first term.
        bad = err > size * 2.0**-20 * (1 + step) + step * np.abs(want) * (len(f) > 0)
        assert not bad.any(), (name, err[bad].max())

    near(got, q, "q")
    bs = k_pool.shape[3]
    block, place = slots // bs, slots % bs
    ok = (slots >= 0) & (block < k_pool.shape[1])
    near(k_pool[layer, block[ok], :, place[ok]], k[ok], "k") if bool(ok.all()) else None
    assert torch.equal(v_pool[layer, block[ok], :, place[ok]], v[ok])
    # Nothing else is written.
    for pool, was in zip((k_pool, v_pool), before):
        pool[layer, block[ok], :, place[ok]] = was[layer, block[ok], :, place[ok]]
        assert torch.equal(pool, was)
    return got


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [
    (1, 12, 12, 64, 64), (3, 12, 4, 64, 32), (64, 8, 8, 96, 96), (5, 6, 2, 128, 128), (17, 32, 8, 128, 64),
    (2, 1, 1, 2, 2), (7, 3, 1, 10, 6), (9, 5, 5, 30, 30), (33, 4, 2, 256, 256), (4, 2, 1, 36, 8), (1000, 12, 12, 64, 64),
])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rope_append(tokens, heads, kv_heads, dim, rotary, interleaved, dtype):
    print_case("rope", tokens, heads, kv_heads, dim, rotary, interleaved, dtype)
    parts = inputs(tokens, heads, kv_heads, dim, 16, dtype, seed=tokens + dim)
    freq, factor = kv_ops.rope_frequencies(rotary, device=DEV)
    positions = torch.randint(0, 5000, (tokens,), dtype=torch.int32, device=DEV)
    check(*parts, positions, freq, factor, interleaved)


@pytest.mark.parametrize("scaling", kv_ops.ROPE_SCALINGS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_far_positions_and_scalings(scaling, dtype):
    print_case("rope far", scaling, dtype)
    parts = inputs(40, 4, 2, 64, 8, dtype, seed=9)
    freq, factor = kv_ops.rope_frequencies(64, 500000.0, scaling=scaling, scale=16.0, original_length=8192, device=DEV)
    positions = torch.cat([torch.tensor([0, 1, 2**31 - 1, 2**24 + 1, -5]), torch.randint(0, 10**7, (35,))]).int().to(DEV)
    check(*parts, positions, freq, factor, False)


def test_slots_outside_the_pool_store_nothing_and_rotate_q():
    print_case("rope bad slots")
    q, k, v, kp, vp, slots = inputs(20, 4, 2, 64, 16, BF16, seed=3)
    slots[::3] = torch.tensor([-1, kp.shape[1] * 16, -(2**40), 2**40, -16, 2**31, -1], device=DEV)
    freq, _ = kv_ops.rope_frequencies(64, device=DEV)
    check(q, k, v, kp, vp, slots, torch.arange(20, dtype=torch.int32, device=DEV), freq, 1.0, False)


@pytest.mark.parametrize("how", ["in place", "strided out", "odd offset", "head-major", "expanded v"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides_and_places(how, dtype):
    print_case("rope strides", how, dtype)
    q, k, v, kp, vp, slots = inputs(21, 6, 2, 64, 16, dtype, seed=5)
    freq, _ = kv_ops.rope_frequencies(48, device=DEV)
    positions = torch.arange(100, 121, dtype=torch.int32, device=DEV)
    out = None
    if how == "in place":
        q = q.contiguous()
        was = q.clone()
        check(was.clone(), k, v, kp, vp, slots, positions, freq, 1.0, True)
        want = kv_ops.rope_append(was, k, v, kp, vp, 1, slots, positions, freq, interleaved=True)
        got = kv_ops.rope_append(q, k, v, kp, vp, 1, slots, positions, freq, interleaved=True, out=q)
        assert got is q and torch.equal(got, want)
        return
    if how == "strided out":
        out = torch.full((21, 6, 80), 7.0, dtype=dtype, device=DEV)[..., 8:72]
    elif how == "odd offset":
        buffer = torch.zeros(21 * 6 * 64 + 1, dtype=dtype, device=DEV)
        buffer[1:] = q.reshape(-1)
        q = buffer[1:].view(21, 6, 64)
    elif how == "head-major":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    else:
        v = v[:1].expand(21, 2, 64)
    check(q, k, v, kp, vp, slots, positions, freq, 1.0, True, out=out)
    if out is not None:
        assert bool((out._base[..., :8] == 7).all() and (out._base[..., 72:] == 7).all())


def test_no_tokens():
    print_case("rope none")
    q, k, v, kp, vp, slots = inputs(1, 4, 2, 64, 16, F32, seed=3)
    freq, _ = kv_ops.rope_frequencies(64, device=DEV)
    got = kv_ops.rope_append(q[:0], k[:0], v[:0], kp, vp, 0, slots[:0], slots[:0].int(), freq)
    assert got.shape == (0, 4, 64)


def test_values_that_are_not_finite_stay_in_their_pair():
    print_case("rope nan")
    q, k, v, kp, vp, slots = inputs(2, 2, 2, 64, 16, F32, seed=3)
    q = q.contiguous()
    q[0, 0, 3], q[1, 1, 40] = float("nan"), float("inf")
    freq, _ = kv_ops.rope_frequencies(32, device=DEV)
    got = kv_ops.rope_append(q, k, v, kp, vp, 0, slots, torch.tensor([5, 6], dtype=torch.int32, device=DEV), freq)
    bad = (~torch.isfinite(got)).nonzero().tolist()
    assert bad == [[0, 0, 3], [0, 0, 19], [1, 1, 40]]


def test_on_another_stream_and_captured():
    print_case("rope captured")
    q, k, v, kp, vp, slots = inputs(64, 12, 12, 64, 16, BF16, seed=4)
    freq, _ = kv_ops.rope_frequencies(64, device=DEV)
    positions = torch.arange(64, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv_ops.rope_append(q, k, v, kp, vp, 0, slots, positions, freq)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv_ops.rope_append(q, k, v, kp, vp, 0, slots, positions, freq)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        positions += 17
        kp.zero_()
        graph.replay()
        pool = kp.clone()
        kp.zero_()
        want = kv_ops.rope_append(q, k, v, kp, vp, 0, slots, positions, freq)
        assert torch.equal(got, want) and torch.equal(pool, kp)
