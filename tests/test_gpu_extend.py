"""paged_attention.extend_batched on the GPU against attention in 64 bits
(step_oracle.extend, which says where its bound comes from; a bfloat16 output
adds half a step of the value, and weights kept in 16 bits of significand or in
bfloat16 their rounding)."""

import math

import pytest
import torch

from conftest import print_case
from moe_engine import paged_attention
import step_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def batch(new, old, heads, kv_heads, dim, block_size, dtype, seed, layers=2, heavy=0.05, extra=0, pad=0):
    """A step's inputs; unused places of the pools and tables hold what must not be read."""
    g = torch.Generator().manual_seed(seed)
    lens = [n + o for n, o in zip(new, old)]
    need = [-(-c // block_size) for c in lens]
    blocks = sum(need) + 3
    k = torch.randn(layers, blocks, kv_heads, block_size, dim, generator=g)
    k = (k * torch.where(torch.rand(k.shape[:-1], generator=g) < heavy, 8.0, 1.0)[..., None]).to(dtype)
    v = torch.randn(k.shape, generator=g).to(dtype)
    order = torch.randperm(blocks, generator=g).tolist()
    width = max(need + [1]) + extra
    tables = torch.full((len(new), width), 2**30, dtype=torch.int32)
    kept = torch.zeros(blocks, block_size, dtype=torch.bool)
    rows = []
    for b, n in enumerate(need):
        ids, order = order[:n], order[n:]
        tables[b, :n] = torch.tensor(ids, dtype=torch.int32)
        t = torch.arange(lens[b])
        rows.append((torch.tensor(ids, dtype=torch.long)[t // block_size], t % block_size))
        kept[rows[-1]] = True
    stale = (~kept).nonzero(as_tuple=True)
    for pool in (k, v):
        pool[:, stale[0], :, stale[1]] = float("nan")
    q = torch.randn(sum(new) + pad, heads, dim, generator=g).to(dtype)
    starts = torch.tensor([0] + new).cumsum(0).int()
    keys = [(k[1, r[0], :, r[1]].double(), v[1, r[0], :, r[1]].double()) for r in rows]
    return dict(q=q.to(DEV), k=k.to(DEV), v=v.to(DEV), tables=tables.to(DEV), starts=starts.to(DEV),
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV), keys=keys, new=new, len_list=lens)


def call(c, max_new=None, max_len=None, **kw):
    out = torch.full_like(c["q"], 123.0)
    got = paged_attention.extend_batched(
        c["q"], c["k"], c["v"], 1, c["tables"], c["starts"], c["lens"],
        max(c["new"] + [0]) if max_new is None else max_new, max(c["len_list"]) if max_len is None else max_len,
        out=out, **kw)
    assert got is out
    return out


def check(c, out, skip=(), prefix=None, slopes=None, scale=None, softcap=0.0, window=0):
    t = 0
    dim, dtype = out.shape[2], out.dtype
    scale = 1 / math.sqrt(dim) if scale is None else scale
    eps_p = 0.0 if dtype == F32 else 2.0**-8
    for b, n in enumerate(c["new"]):
        have = out[t : t + n].double().cpu()
        if b not in skip:
            want, bound = ref.extend(
                c["q"][t : t + n].double().cpu(), *c["keys"][b], c["len_list"][b], scale=scale, softcap=softcap,
                slopes=slopes, window=window, prefix=0 if prefix is None else prefix[b], eps_p=eps_p)
            if dtype == BF16:
                bound = bound + torch.finfo(BF16).eps / 2 * (want.abs() + bound)
            err = (have - want).abs()
            assert not bool((err > bound + 1e-30).any()) and not bool(have.isnan().any()), \
                (b, float(err.max()), float((err / (bound + 1e-30)).max()))
        t += n
    assert bool((out[t:] == 123.0).all()), "rows behind the last sequence"


SHAPES = [
    # new tokens, tokens before them
    ([1], [0]), ([1], [1]), ([1], [31]), ([1], [32]), ([1], [700]), ([4], [60]), ([17], [0]), ([70], [33]),
    ([1, 0, 5, 1], [40, 9, 0, 129]), ([0, 0, 3], [0, 5, 500]), ([1] * 9, [0, 1, 2, 15, 16, 17, 127, 128, 255]),
    ([130, 1, 2], [0, 300, 64]), ([33, 16, 15, 1], [1, 16, 240, 511]),
]


@pytest.mark.parametrize("new,old", SHAPES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (6, 2, 128), (3, 1, 96)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_extend(new, old, heads, kv_heads, dim, dtype):
    print_case("extend", new, old, heads, kv_heads, dim, dtype)
    c = batch(new, old, heads, kv_heads, dim, 16, dtype, seed=sum(new) + sum(old), extra=2, pad=3)
    check(c, call(c))


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 32), (8, 1, 64), (2, 2, 256), (20, 1, 32), (128, 1, 64), (34, 2, 96)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_heads(heads, kv_heads, dim, dtype):
    print_case("extend heads", heads, kv_heads, dim, dtype)
    c = batch([1, 3, 40], [100, 0, 7], heads, kv_heads, dim, 16, dtype, seed=heads + dim)
    check(c, call(c))


@pytest.mark.parametrize("block_size", [1, 3, 8, 32, 64, 100])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_block_sizes(block_size, dtype):
    print_case("extend block size", block_size, dtype)
    c = batch([1, 2, 50], [99, 130, 7], 4, 2, 64, block_size, dtype, seed=block_size)
    check(c, call(c))


OPTIONS = [
    dict(softcap=5.0), dict(softcap=30.0), dict(slopes=True), dict(slopes=True, softcap=8.0), dict(window=1),
    dict(window=5), dict(window=64), dict(window=10**6), dict(prefix=[0, 5, 200]), dict(prefix=[10**6, 0, 40]),
    dict(window=20, prefix=[30, 200, 100], slopes=True), dict(scale=0.5), dict(scale=-0.3, softcap=2.0), dict(scale=0.0),
]


@pytest.mark.parametrize("option", OPTIONS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scores_and_masks(option, dtype):
    print_case("extend option", option, dtype)
    c = batch([1, 37, 150], [400, 3, 90], 4, 2, 64, 16, dtype, seed=7)
    kw, want = dict(option), dict(option)
    if "slopes" in option:
        want["slopes"] = 2.0 ** -(torch.arange(4).double() * 1.5)
        kw["slopes"] = want["slopes"].float().to(DEV)
    if "prefix" in option:
        kw["prefix_lens"] = torch.tensor(kw.pop("prefix"), dtype=torch.int32, device=DEV)
        want["prefix"] = [min(p, n) for p, n in zip(option["prefix"], c["len_list"])]
    check(c, call(c, **kw), **want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_long_contexts_are_split_and_joined(dtype):
    print_case("extend long", dtype)
    c = batch([1, 2, 1], [20000, 7000, 5], 2, 1, 64, 16, dtype, seed=2, heavy=0.01)
    check(c, call(c))
    check(c, call(c, window=5000), window=5000)
    # A window far shorter than the bound, and bounds above the lengths.
    check(c, call(c, max_new=40, max_len=100000, window=100), window=100)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_what_a_token_does_not_see_has_no_part_in_it(dtype):
    """NaN and infinities in K and V of later tokens, of tokens before the
    window: rows that do not see them are as without; rows that do are not finite."""
    print_case("extend masked nan", dtype)
    for poison in (float("nan"), float("inf"), -float("inf")):
        for where in ("k", "v"):
            c = batch([60], [50], 2, 1, 64, 16, dtype, seed=4)
            clean = call(c, window=40)
            b, s = c["tables"][0, 90 // 16].item(), 90 % 16
            c[where][1, b, :, s, 5] = poison
            got = call(c, window=40)
            rows = torch.arange(50, 110)
            sees = ((rows >= 90) & (rows < 130)).to(DEV)
            assert torch.equal(got[~sees], clean[~sees]), (poison, where)
            if where == "v":
                assert not bool(got[sees][:, :, 5].isfinite().any())
                if poison == poison:
                    assert bool((got[sees][:, :, 5] == poison).all())
                others = torch.arange(64, device=DEV) != 5
                assert bool(got[sees][:, :, others].isfinite().all())
            elif poison != poison:
                assert bool(got[sees].isnan().all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_an_infinite_value_every_token_sees(dtype):
    print_case("extend inf seen by all", dtype)
    c = batch([70], [200], 2, 1, 64, 16, dtype, seed=4, heavy=0.0)
    c["v"][1, c["tables"][0, 1].item(), :, 3, 9] = float("inf")
    got = call(c)
    assert bool((got[:70, :, 9] == math.inf).all())
    assert bool(got[:70, :, torch.arange(64, device=DEV) != 9].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scores_of_the_lowest_value(dtype):
    """Scores at the type's lowest value are seen keys like others."""
    print_case("extend lowest", dtype)
    c = batch([3], [20], 1, 1, 64, 16, dtype, seed=4, heavy=0.0)
    c["k"][1] = 0
    c["q"][:] = 0
    c["q"][:, :, 0] = 1
    b = c["tables"][0]
    for j in range(23):
        c["k"][1, b[j // 16].item(), :, j % 16, 0] = torch.finfo(dtype).min
    c["keys"][0][0][:] = 0
    c["keys"][0][0][:, :, 0] = float(torch.finfo(dtype).min)
    got = call(c, scale=0.125)
    want = torch.stack([c["keys"][0][1][: 21 + i].mean(0) for i in range(3)])
    bound = (c["keys"][0][1].abs().mean(0) * 2.0**-7).max()
    assert float((got[:3].double().cpu() - want).abs().max()) < float(bound) + 2.0**-8


# Enough rows and keys for the tiles of 128 rows (the tests above stay below them).
MANY = dict(new=[300, 1, 70, 0, 33], old=[500, 700, 0, 60, 95], heads=32, kv_heads=4)


@pytest.mark.parametrize("dim,block_size", [(32, 16), (64, 16), (64, 7), (64, 32), (96, 16), (96, 24), (128, 16),
                                            (128, 1), (256, 16), (256, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_many_rows(dim, block_size, dtype):
    print_case("extend many rows", dim, block_size, dtype)
    scale = 64 // dim or 1
    c = batch(MANY["new"], MANY["old"], 32 * scale, 4 * scale, dim, block_size, dtype, seed=dim, extra=1, pad=2)
    check(c, call(c))


@pytest.mark.parametrize("heads,kv_heads", [(24, 24), (40, 8), (66, 2)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_many_rows_of_other_groups(heads, kv_heads, dtype):
    print_case("extend many rows", heads, kv_heads, dtype)
    c = batch(MANY["new"], MANY["old"], heads, kv_heads, 64, 16, dtype, seed=heads)
    check(c, call(c))


@pytest.mark.parametrize("option", OPTIONS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scores_and_masks_of_many_rows(option, dtype):
    print_case("extend many rows option", option, dtype)
    new, old = [290, 1, 101], [700, 400, 200]
    # A window bounds the work that is counted: more heads for it.
    heads = 32 if option.get("window", 10**6) > 500 else 256
    c = batch(new, old, heads, 4, 64, 16, dtype, seed=7)
    kw, want = dict(option), dict(option)
    if "slopes" in option:
        want["slopes"] = 2.0 ** -(torch.arange(heads).double() % 7 * 1.5)
        kw["slopes"] = want["slopes"].float().to(DEV)
    if "prefix" in option:
        kw["prefix_lens"] = torch.tensor(kw.pop("prefix"), dtype=torch.int32, device=DEV)
        want["prefix"] = [min(p, n) for p, n in zip(option["prefix"], c["len_list"])]
    check(c, call(c, **kw), **want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_a_prefix_far_past_the_window_over_a_split_context(dtype):
    """The prefix's keys count for the split, not the window's alone."""
    print_case("extend prefix past window", dtype)
    for new, old, heads in (([2, 1], [300, 9000], 2), ([150, 40], [600, 9000], 8)):
        c = batch(new, old, heads, 1, 64, 16, dtype, seed=3, heavy=0.01)
        for prefix in (list(c["len_list"]), [n // 2 for n in c["len_list"]]):
            kw = dict(window=64, prefix_lens=torch.tensor(prefix, dtype=torch.int32, device=DEV))
            check(c, call(c, max_len=9150, **kw), window=64, prefix=prefix)
    # All of a long sequence is new: its first tokens see the whole prefix, far past the window.
    c = batch([1500], [0], 2, 1, 64, 16, dtype, seed=5)
    check(c, call(c, window=16, prefix_lens=torch.tensor([1400], dtype=torch.int32, device=DEV)), window=16, prefix=[1400])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_many_rows_over_a_split_context(dtype):
    print_case("extend many rows split", dtype)
    c = batch([150, 40], [6000, 2500], 8, 1, 64, 16, dtype, seed=3, heavy=0.01)
    check(c, call(c))
    check(c, call(c, window=3000), window=3000)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 500])
def test_what_many_rows_do_not_see_has_no_part_in_them(dtype, window):
    print_case("extend many rows masked nan", dtype, window)
    for poison in (float("nan"), float("inf"), -float("inf")):
        for where in ("k", "v"):
            for block_size in (16, 5):
                c = batch([400], [500], 32, 4, 64, block_size, dtype, seed=4)
                clean = call(c, window=window)
                at = 700
                c[where][1, c["tables"][0, at // block_size].item(), :, at % block_size, 5] = poison
                got = call(c, window=window)
                rows = torch.arange(500, 900)
                sees = ((rows >= at) & (rows < at + (window or 10**6))).to(DEV)
                assert torch.equal(got[~sees], clean[~sees]), (poison, where)
                if where == "v":
                    assert not bool(got[sees][:, :, 5].isfinite().any())
                    if poison == poison:
                        assert bool((got[sees][:, :, 5] == poison).all())
                    others = torch.arange(64, device=DEV) != 5
                    assert bool(got[sees][:, :, others].isfinite().all())
                elif poison != poison:
                    assert bool(got[sees].isnan().all())


def test_many_rows_with_lengths_and_tables_out_of_bounds():
    print_case("extend many rows bad tables")
    for dtype in (F32, BF16):
        for block_size in (16, 9):
            c = batch([200, 300, 100, 40], [400, 400, 600, 0], 32, 4, 64, block_size, dtype, seed=6)
            c["tables"][1, 450 // block_size] = -1         # rows from its first token on see it
            c["tables"][2, 100 // block_size] = 2**31 - 1  # every row does
            c["lens"][3] = 10000                           # past the bound, and its table row
            got = call(c)
            check(c, got, skip=(1, 2, 3))
            first = 450 // block_size * block_size - 400
            assert bool(got[200 + first : 500].isnan().all()) and bool(got[500:640].isnan().all())
            assert bool(got[200 : 200 + first].isfinite().all())
            # A bad entry no token sees: behind the window.
            c = batch([300], [900], 128, 4, 64, block_size, dtype, seed=6)
            c["tables"][0, 2] = -1
            check(c, call(c, window=600), window=600)


def test_many_rows_with_broken_starts():
    print_case("extend many rows bad starts")
    c = batch([200, 300, 100], [400, 500, 300], 32, 4, 64, 16, BF16, seed=6)
    c["starts"][:] = torch.tensor([0, -5, 10000, 3])
    call(c, max_new=400, max_len=900)
    c["lens"][:] = torch.tensor([-4, 0, 1])
    c["starts"][:] = torch.tensor([0, 200, 500, 600])
    got = call(c, max_new=300, max_len=900)
    assert bool((got[:599] == 0).all()) and bool(got[599].isfinite().all())


def test_lengths_and_tables_out_of_bounds():
    print_case("extend bad tables")
    for dtype in (F32, BF16):
        c = batch([2, 3, 1, 4], [40, 40, 600, 0], 2, 2, 64, 16, dtype, seed=6)
        c["tables"][1, 1] = -1
        c["tables"][2, 30] = 2**31 - 1
        c["lens"][3] = 10000  # past the bound, and its table row
        got = call(c)
        check(c, got, skip=(1, 2, 3))
        assert bool(got[2:10].isnan().all())
        # A length that the table row does not hold.
        c = batch([2], [40], 2, 2, 64, 16, dtype, seed=6)
        c["lens"][0] = 60
        assert bool(call(c, max_len=100).isnan().all())
        # A bad entry no token sees: behind the window.
        c = batch([2], [400], 2, 2, 64, 16, dtype, seed=6)
        c["tables"][0, 2] = -1
        check(c, call(c, window=100), window=100)


def test_broken_starts_read_and_write_nothing_outside():
    print_case("extend bad starts")
    c = batch([2, 3, 4], [10, 20, 30], 2, 2, 64, 16, F32, seed=6)
    c["starts"][:] = torch.tensor([0, -5, 100, 3])
    call(c, max_new=50, max_len=1000)
    c["lens"][:] = torch.tensor([-4, 0, 1])  # fewer than new: rows before the sequence see nothing
    c["starts"][:] = torch.tensor([0, 2, 5, 9])
    got = call(c, max_new=50)
    assert bool((got[:8] == 0).all()) and bool(got[8].isfinite().all())


def test_tokens_past_max_new_are_left_as_they_were():
    print_case("extend max_new")
    c = batch([9, 2], [10, 20], 2, 2, 64, 16, BF16, seed=6)
    full, cut = call(c), call(c, max_new=4)
    assert torch.equal(cut[:4], full[:4]) and bool((cut[4:9] == 123).all()) and torch.equal(cut[9:], full[9:])


@pytest.mark.parametrize("how", ["q strided", "q odd", "q inner", "table wide", "out strided"])
def test_strides(how):
    print_case("extend strides", how)
    c = batch([5, 1, 40], [10, 200, 0], 4, 2, 64, 16, BF16, seed=8)
    want = call(c)
    out = None
    if how == "q strided":
        wide = torch.zeros(46, 8, 64, dtype=BF16, device=DEV)
        wide[:, 2:6] = c["q"]
        c["q"] = wide[:, 2:6]
    elif how == "q odd":
        flat = torch.zeros(c["q"].numel() + 1, dtype=BF16, device=DEV)
        flat[1:] = c["q"].reshape(-1)
        c["q"] = flat[1:].view(46, 4, 64)
    elif how == "q inner":
        c["q"] = c["q"].transpose(1, 2).contiguous().transpose(1, 2)
    elif how == "table wide":
        t = c["tables"]
        wide = torch.full((3, t.shape[1] + 9), -1, dtype=torch.int32, device=DEV)
        wide[:, : t.shape[1]] = t
        c["tables"] = wide[:, : t.shape[1]]
    else:
        out = torch.zeros(46, 6, 64, dtype=BF16, device=DEV)[:, 1:5]
    args = (c["q"], c["k"], c["v"], 1, c["tables"], c["starts"], c["lens"], 40, 201)
    got = paged_attention.extend_batched(*args, out=out)
    assert torch.equal(got, want)
    if out is not None:
        assert bool((out._base[:, 0] == 0).all() and (out._base[:, 5] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_the_largest_bounds(dtype):
    """Bounds beyond every length, in 32 bits and past them, mean no bound; a
    length below the new tokens puts the first ones before position 0."""
    print_case("extend largest bounds", dtype)
    c = batch([1, 40, 150], [400, 3, 90], 4, 2, 64, 16, dtype, seed=7)
    for window, most in ((2**30, 2**31 - 1), (2**30 + 1, 2**31), (2**31 - 1, 2**32), (2**32, 2**33)):
        check(c, call(c, max_new=most, window=window))
    check(c, call(c, max_len=2**30))
    check(c, call(c, softcap=1024.0, scale=1.0), softcap=1024.0, scale=1.0)
    # 40 new tokens of a length of 30: the first see the prefix alone.
    c["len_list"][1], c["lens"][1] = 30, 30
    c["keys"][1] = tuple(t[:30] for t in c["keys"][1])
    prefix = torch.tensor([0, 20, 0], dtype=torch.int32, device=DEV)
    for window in (0, 2**31 - 1):
        check(c, call(c, window=window, prefix_lens=prefix), prefix=[0, 20, 0])


@pytest.mark.parametrize("to_out", [False, True])
def test_one_table_row_for_every_sequence(to_out):
    """A broadcast table, and rows that overlap: the same as their copies."""
    print_case("extend shared table", to_out)
    c = batch([1], [200], 4, 2, 64, 16, BF16, seed=11)
    q = torch.randn(5, 4, 64, device=DEV).to(BF16)
    starts = torch.arange(6, dtype=torch.int32, device=DEV)
    lens = torch.tensor([201, 3, 90, 64, 17], dtype=torch.int32, device=DEV)
    line = torch.cat([c["tables"][0], c["tables"][0, :4]])
    for tables in (c["tables"].expand(5, -1), line.as_strided((5, 13), (1, 1))):
        got, want = (paged_attention.extend_batched(
            q, c["k"], c["v"], 1, t, starts, lens, 1, 201, out=torch.empty_like(q) if to_out else None)
            for t in (tables, tables.contiguous()))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and not bool(got[0].isnan().any())


def test_it_is_decode_where_each_sequence_has_one_token():
    print_case("extend vs decode")
    c = batch([1] * 5, [0, 30, 500, 1000, 2500], 4, 4, 64, 16, F32, seed=9)
    want = paged_attention.decode_batched(c["q"], c["k"], c["v"], 1, c["tables"], c["lens"], 2501)
    got = call(c)
    # Both are within the oracle's bound of the exact value.
    bounds = [ref.extend(c["q"][b : b + 1].double().cpu(), *c["keys"][b], c["len_list"][b], scale=0.125)[1][0]
              for b in range(5)]
    assert bool(((got - want).double().cpu().abs() <= 2 * torch.stack(bounds)).all())


def test_two_captured_steps_and_streams_keep_apart():
    """Two graphs and an eager call, each with its own split context, replayed
    in turn and on two streams at once."""
    print_case("extend captured")
    a = batch([1, 2], [9000, 4000], 2, 1, 64, 16, BF16, seed=10)
    b = batch([3, 1], [8000, 6000], 2, 1, 64, 16, BF16, seed=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a), call(b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for c in (a, b):
        c["out"] = torch.zeros_like(c["q"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_attention.extend_batched(c["q"], c["k"], c["v"], 1, c["tables"], c["starts"], c["lens"], 3, 9001,
                                           out=c["out"])
        graphs.append(graph)
    for i in range(5):
        for c in (a, b):
            c["q"].copy_(torch.randn_like(c["q"]))
            c["out"].zero_()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for c in (a, b):
            want = paged_attention.extend_batched(c["q"], c["k"], c["v"], 1, c["tables"], c["starts"], c["lens"], 3, 9001)
            assert torch.equal(c["out"], want)
            _ = c["q"].float().sum()


def test_the_same_call_gives_the_same_bits():
    print_case("extend twice")
    for dtype in (F32, BF16):
        c = batch([1, 300, 5], [5000, 100, 900], 6, 2, 128, 16, dtype, seed=12)
        assert torch.equal(call(c), call(c))
        c = batch([1, 3, 5], [500, 100, 900], 6, 2, 128, 16, dtype, seed=12)
        assert torch.equal(call(c), call(c))
