"""kv_ops.reserve / release on the GPU against a host allocator, value for value."""

import numpy as np
import pytest
import torch

from conftest import print_case
from moe_engine import kv_ops
from moe_engine.model import BlockAllocator, ModelConfig
import step_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(batch, low, high, new_low, new_high, block_size, seed, spare=7, pad=0, extra_width=1):
    rng = np.random.default_rng(seed)
    lens = rng.integers(low, high + 1, batch)
    new = rng.integers(new_low, new_high + 1, batch)
    width = int((-(-(lens + new) // block_size)).max()) + extra_width
    blocks = int((-(-(lens + new) // block_size)).sum()) + spare
    ids = rng.permutation(blocks).astype(np.int32)
    tables = np.full((batch, width), -7, np.int32)  # entries nothing may read or write
    at = 0
    for b in range(batch):
        n = -(-int(lens[b]) // block_size)
        tables[b, :n] = ids[at : at + n]
        at += n
    stack = np.full(blocks, -9, np.int32)
    stack[: blocks - at] = ids[at:]
    return dict(stack=stack, count=blocks - at, tables=tables, lens=lens, new=new, block_size=block_size,
                max_tokens=int(new.sum()) + pad)


def dev(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).to(DEV)


def check_reserve(c):
    want = ref.reserve(**c)
    ids, count, tables = dev(c["stack"]), dev([c["count"]]), dev(c["tables"])
    lens, new = dev(c["lens"]), dev(c["new"])
    step = kv_ops.reserve(ids, count, tables, lens, new, c["block_size"], c["max_tokens"])
    got = (tables, step.starts, step.slots, step.positions, step.context_lens, step.free_count, step.status)
    for name, g, w in zip(("tables", "starts", "slots", "positions", "lens", "count", "status"), got, want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
    # Inputs other than the tables stay.
    assert np.array_equal(ids.cpu().numpy(), c["stack"]) and int(count) == c["count"]
    assert np.array_equal(lens.cpu().numpy(), c["lens"]) and np.array_equal(new.cpu().numpy(), c["new"])
    return step


@pytest.mark.parametrize("args", [
    (1, 0, 0, 1, 1, 16), (1, 0, 0, 0, 0, 16), (1, 15, 15, 1, 1, 16), (1, 16, 16, 1, 1, 16), (3, 0, 40, 0, 5, 16),
    (64, 0, 600, 1, 1, 16), (64, 0, 600, 0, 1, 1), (65, 0, 90, 0, 70, 7), (255, 0, 50, 0, 3, 8),
    (256, 0, 50, 0, 3, 32), (257, 0, 50, 0, 3, 16), (1000, 0, 100, 0, 40, 16), (5, 0, 9000, 0, 9000, 16),
    (2, 0, 0, 2500, 5000, 1), (8192, 0, 3, 0, 2, 2),
    (500, 0, 100, 0, 600, 16), (3, 0, 7, 20000, 30000, 16), (8192, 0, 40, 0, 30, 16), (90, 0, 0, 0, 5000, 7),
], ids=str)
@pytest.mark.parametrize("pad", [0, 300, 301])
def test_reserve_is_the_host_allocators(args, pad):
    print_case("reserve", args, pad)
    step = check_reserve(case(*args, seed=sum(args), pad=pad))
    assert int(step.status) == 0


def test_reserve_takes_the_last_block_and_refuses_one_more():
    print_case("reserve exact count")
    for spare, status in ((0, 0), (-1, 1)):
        c = case(33, 0, 60, 0, 50, 16, seed=1, spare=0)
        c["count"] += spare
        assert int(check_reserve(c).status) == status


@pytest.mark.parametrize("change,status", [
    (dict(max_tokens=-1), 3), (dict(lens=(4, -1)), 4), (dict(new=(4, -1)), 4), (dict(new=(4, 2**31 - 1)), 2),
    (dict(count=-1), 4), (dict(count=10**6), 4), (dict(lens=(4, 10**6)), 2),
    (dict(lens=(4, -1), new=(5, 2**31 - 1)), 4),
], ids=str)
def test_a_reservation_that_fails_changes_nothing(change, status):
    print_case("reserve refusal", change)
    c = case(9, 0, 40, 1, 30, 16, seed=2, pad=3)
    for key, value in change.items():
        if isinstance(value, tuple):
            c[key] = c[key].copy()
            c[key][value[0]] = value[1]
        elif key == "max_tokens":
            c[key] = int(c["new"].sum()) + value
        else:
            c[key] = value
    assert int(check_reserve(c).status) == status


def test_reserve_on_rows_of_a_wider_table():
    print_case("reserve strided table")
    c = case(6, 0, 80, 1, 40, 16, seed=3)
    wide = torch.full((6, c["tables"].shape[1] + 5), -3, dtype=torch.int32, device=DEV)
    wide[:, :-5] = dev(c["tables"])
    want = ref.reserve(**c)
    step = kv_ops.reserve(dev(c["stack"]), dev([c["count"]]), wide[:, :-5], dev(c["lens"]), dev(c["new"]), 16,
                          c["max_tokens"])
    assert np.array_equal(wide[:, :-5].cpu().numpy(), want[0]) and bool((wide[:, -5:] == -3).all())
    assert np.array_equal(step.slots.cpu().numpy(), want[2])


@pytest.mark.parametrize("args", [(1, 0, 0), (1, 16, 16), (64, 0, 300), (257, 0, 100), (1000, 0, 500), (8192, 0, 5)], ids=str)
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_release_is_the_host_allocators(args, share):
    print_case("release", args, share)
    c = case(*args, 0, 0, 16, seed=args[0])
    finished = np.random.default_rng(5).random(args[0]) < share
    want = ref.release(c["stack"], c["count"], c["tables"], c["lens"], finished, 16)
    ids, count, tables, lens = dev(c["stack"]), dev([c["count"]]), dev(c["tables"]), dev(c["lens"])
    step = kv_ops.release(ids, count, tables, lens, dev(finished, torch.bool), 16)
    got = (ids, step.context_lens, step.free_count, step.status)
    for name, g, w in zip(("stack", "lens", "count", "status"), got, want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
    assert np.array_equal(tables.cpu().numpy(), c["tables"]) and np.array_equal(lens.cpu().numpy(), c["lens"])


@pytest.mark.parametrize("change,status", [(dict(count=8), 1), (dict(count=-1), 4), (dict(long=True), 2), (dict(neg=True), 4)], ids=str)
def test_a_release_that_fails_changes_nothing(change, status):
    print_case("release refusal", change)
    c = case(9, 1, 40, 0, 0, 16, seed=2)
    if "count" in change:
        c["count"] = change["count"] if change["count"] < 0 else len(c["stack"]) - 2
    lens = c["lens"].copy()
    if "long" in change:
        lens[3] = 10**6
    if "neg" in change:
        lens[3] = -1
    ids = dev(c["stack"])
    step = kv_ops.release(ids, dev([c["count"]]), dev(c["tables"]), dev(lens), torch.ones(9, dtype=torch.bool, device=DEV), 16)
    assert int(step.status) == status and int(step.free_count) == c["count"]
    assert np.array_equal(ids.cpu().numpy(), c["stack"]) and np.array_equal(step.context_lens.cpu().numpy(), lens)


def test_many_steps_of_admitting_and_finishing_keep_every_block_once():
    """A pool run for 60 steps through reserve and release, with a host
    allocator beside it; blocks are lent by and given back to a BlockAllocator."""
    print_case("reserve/release loop")
    bs, batch, width, blocks = 4, 13, 12, 60
    allocator = BlockAllocator(ModelConfig(num_layers=1, hidden_dim=64, num_heads=2), blocks, bs, DEV)
    ids, count = kv_ops.take_free_blocks(allocator)
    assert not allocator.free_blocks and int(count) == blocks
    rng = np.random.default_rng(11)
    stack, n = ids.cpu().numpy(), blocks
    tables, lens = np.zeros((batch, width), np.int32), np.zeros(batch, np.int64)
    d_tables, d_lens = dev(tables), dev(lens)
    seen = set()
    for _ in range(60):
        new = rng.integers(0, 9, batch) * (rng.random(batch) < 0.6)
        tables, starts, slots, _, lens, n, status = ref.reserve(stack, n, tables, lens, new, bs, 120)
        step = kv_ops.reserve(ids, count, d_tables, d_lens, dev(new), bs, 120)
        seen.add(status)
        assert int(step.status) == status
        assert np.array_equal(step.slots.cpu().numpy(), slots) and np.array_equal(step.starts.cpu().numpy(), starts)
        count, d_lens = step.free_count, step.context_lens
        finished = rng.random(batch) < (0.5 if status else 0.15)
        stack, lens, n, _ = ref.release(stack, n, tables, lens, finished, bs)
        step = kv_ops.release(ids, count, d_tables, d_lens, dev(finished, torch.bool), bs)
        count, d_lens = step.free_count, step.context_lens
        held = [int(i) for b in range(batch) for i in tables[b, : -(-int(lens[b]) // bs)]]
        free = ids[: int(count)].cpu().tolist()
        assert sorted(held + free) == list(range(blocks))
        assert np.array_equal(d_tables.cpu().numpy(), tables) and int(count) == n
    assert 0 in seen and len(seen) > 1
    allocator.free(ids[: int(count)].tolist())
    assert len(allocator.free_blocks) == int(count)


def test_reserve_and_release_in_a_captured_step():
    """One captured step (release, reserve, the state carried) replayed with
    other lengths each time, eager work between."""
    print_case("captured reserve/release")
    c = case(17, 0, 60, 1, 9, 8, seed=8, spare=200, pad=40, extra_width=8)
    ids, count, tables, lens, new = (dev(c["stack"]), dev([c["count"]]), dev(c["tables"]), dev(c["lens"]), dev(c["new"]))
    finished = torch.zeros(17, dtype=torch.bool, device=DEV)

    def step():
        r = kv_ops.release(ids, count, tables, lens, finished, 8)
        s = kv_ops.reserve(ids, r.free_count, tables, r.context_lens, new, 8, c["max_tokens"])
        return s

    state = [t.clone() for t in (ids, count, tables, lens, new, finished)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, was in zip((ids, count, tables, lens, new, finished), state):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = step()
        lens.copy_(s.context_lens)
        count.copy_(s.free_count)
    for t, was in zip((ids, count, tables, lens, new, finished), state):
        t.copy_(was)
    stack, n, tab, ln = c["stack"].copy(), c["count"], c["tables"].copy(), np.array(c["lens"])
    rng = np.random.default_rng(3)
    for _ in range(6):
        now, done = rng.integers(0, 7, 17), rng.random(17) < 0.3
        new.copy_(dev(now))
        finished.copy_(dev(done, torch.bool))
        graph.replay()
        torch.cuda.synchronize()
        stack, ln, n, _ = ref.release(stack, n, tab, ln, done, 8)
        tab, starts, slots, positions, ln, n, status = ref.reserve(stack, n, tab, ln, now, 8, c["max_tokens"])
        assert int(s.status) == status == 0 and int(count) == n
        assert np.array_equal(s.slots.cpu().numpy(), slots) and np.array_equal(s.positions.cpu().numpy(), positions)
        assert np.array_equal(tables.cpu().numpy(), tab) and np.array_equal(lens.cpu().numpy(), ln)
        _ = torch.randn(1000, device=DEV).sum()
