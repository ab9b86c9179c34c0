"""What the operators of a serving step refuse, on the CPU: the C entries
before any launch (stand-in addresses, never dereferenced), and the Python ones
on CPU tensors that are taken for a device's."""

import math

import pytest
import torch

from moe_engine import _native, kv_ops, paged_attention, projection

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
F32, BF16, F16 = 0, 1, 2
_addr = iter(range(1 << 24, 1 << 40, 1 << 20))


def ptr():
    return next(_addr)


def reserve_args(**over):
    a = dict(ids=ptr(), capacity=100, count=ptr(), tables=ptr(), stride=10, width=10, lens=ptr(), new=ptr(), batch=4,
             block_size=16, max_tokens=64, starts=ptr(), slots=ptr(), positions=ptr(), lens_out=ptr(), count_out=ptr(),
             status=ptr(), stream=None)
    return {**a, **over}


def release_args(**over):
    a = dict(ids=ptr(), capacity=100, count=ptr(), tables=ptr(), stride=10, width=10, lens=ptr(), finished=ptr(),
             batch=4, block_size=16, lens_out=ptr(), count_out=ptr(), status=ptr(), stream=None)
    return {**a, **over}


def rope_args(**over):
    a = dict(q=ptr(), q_st=256, q_sh=64, k=ptr(), v=ptr(), kv_st=128, kv_sh=64, kp=ptr(), vp=ptr(), sblk=2 * 16 * 64,
             shead=16 * 64, nb=8, slots=ptr(), positions=ptr(), freq=ptr(), rotary=64, interleaved=0, factor=1.0,
             tokens=5, heads=4, kv_heads=2, dim=64, block_size=16, out=ptr(), out_st=256, out_sh=64, dtype=F32,
             stream=None)
    return {**a, **over}


def extend_args(**over):
    a = dict(q=ptr(), q_st=256, q_sh=64, kp=ptr(), vp=ptr(), sblk=2 * 16 * 64, shead=16 * 64, nb=8, tables=ptr(),
             t_stride=10, width=10, starts=ptr(), lens=ptr(), tokens=5, batch=2, max_new=5, max_len=100, heads=4,
             kv_heads=2, dim=64, block_size=16, scale=0.125, cap=0.0, slopes=None, window=0, prefix=None, out=ptr(),
             out_st=256, out_sh=64, ws=None, ws_bytes=0, dtype=BF16, stream=None)
    return {**a, **over}


def logprobs_args(**over):
    a = dict(x=ptr(), stride=1000, rows=3, vocab=1000, tokens=ptr(), top=5, logprobs=ptr(), entropy=ptr(),
             top_logprobs=ptr(), top_tokens=ptr(), ws=ptr(), ws_bytes=1 << 30, dtype=F32, stream=None)
    return {**a, **over}


LENS = ptr()
CASES = [
    ("mie_step_reserve", reserve_args(batch=0), INVALID, b"batch 0"),
    ("mie_step_reserve", reserve_args(batch=8193), INVALID, b"batch 8193"),
    ("mie_step_reserve", reserve_args(block_size=0), INVALID, b"block_size 0"),
    ("mie_step_reserve", reserve_args(capacity=0), INVALID, b"free list of 0"),
    ("mie_step_reserve", reserve_args(stride=9), INVALID, b"table rows"),
    ("mie_step_reserve", reserve_args(width=0), INVALID, b"table rows"),
    ("mie_step_reserve", reserve_args(width=1 << 28, stride=1 << 28), INVALID, b"2^31 - 1"),
    ("mie_step_reserve", reserve_args(max_tokens=-1), INVALID, b"max_tokens -1"),
    ("mie_step_reserve", reserve_args(max_tokens=(1 << 30) + 1), INVALID, b"max_tokens"),
    ("mie_step_reserve", reserve_args(slots=None), INVALID, b"null pointer"),
    ("mie_step_reserve", reserve_args(status=None), INVALID, b"null pointer"),
    ("mie_step_reserve", reserve_args(lens=LENS, lens_out=LENS), INVALID, b"alias"),
    ("mie_step_reserve", reserve_args(count=LENS, count_out=LENS), INVALID, b"alias"),
    ("mie_step_release", release_args(batch=8193), INVALID, b"batch 8193"),
    ("mie_step_release", release_args(finished=None), INVALID, b"null pointer"),
    ("mie_step_release", release_args(lens=LENS, lens_out=LENS), INVALID, b"alias"),
    ("mie_step_release", release_args(stride=3), INVALID, b"table rows"),
    ("mie_rope_append", rope_args(dtype=F16), UNSUPPORTED, b"float32 or bfloat16"),
    ("mie_rope_append", rope_args(rotary=63), INVALID, b"rotary_dim 63"),
    ("mie_rope_append", rope_args(rotary=66), INVALID, b"rotary_dim 66"),
    ("mie_rope_append", rope_args(rotary=0), INVALID, b"rotary_dim 0"),
    ("mie_rope_append", rope_args(tokens=-1), INVALID, b"tokens=-1"),
    ("mie_rope_append", rope_args(tokens=(1 << 23) + 1), INVALID, b"bad shape"),
    ("mie_rope_append", rope_args(heads=0), INVALID, b"bad shape"),
    ("mie_rope_append", rope_args(freq=None), INVALID, b"null pointer"),
    ("mie_rope_append", rope_args(shead=16 * 63), INVALID, b"overlap"),
    ("mie_paged_extend", extend_args(dtype=F16), UNSUPPORTED, b"float32 or bfloat16"),
    ("mie_paged_extend", extend_args(dim=48), UNSUPPORTED, b"head_dim 48"),
    ("mie_paged_extend", extend_args(heads=5), INVALID, b"num_heads=5"),
    ("mie_paged_extend", extend_args(heads=258), INVALID, b"num_heads=258"),
    ("mie_paged_extend", extend_args(tokens=-1), INVALID, b"tokens=-1"),
    ("mie_paged_extend", extend_args(window=-1), INVALID, b"window=-1"),
    ("mie_paged_extend", extend_args(max_len=-1), INVALID, b"max_context_len=-1"),
    ("mie_paged_extend", extend_args(cap=-1.0), INVALID, b"softcap"),
    ("mie_paged_extend", extend_args(cap=math.inf), INVALID, b"softcap"),
    ("mie_paged_extend", extend_args(cap=1025.0), INVALID, b"softcap"),
    ("mie_paged_extend", extend_args(cap=math.nan), INVALID, b"softcap"),
    ("mie_paged_extend", extend_args(scale=math.nan), INVALID, b"scale"),
    ("mie_paged_extend", extend_args(scale=3e38), INVALID, b"scale"),
    ("mie_paged_extend", extend_args(cap=1e-40), INVALID, b"softcap"),
    ("mie_paged_extend", extend_args(t_stride=9), INVALID, b"table rows"),
    ("mie_paged_extend", extend_args(block_size=0), INVALID, b"block_size=0"),
    ("mie_paged_extend", extend_args(starts=None), INVALID, b"null pointer"),
    ("mie_paged_extend", extend_args(shead=16), INVALID, b"overlap"),
    ("mie_paged_extend", extend_args(out_sh=32), INVALID, b"overlap"),
    ("mie_paged_extend", extend_args(q=(1 << 24) + 2), INVALID, b"aligned"),
    ("mie_paged_extend", extend_args(q_st=260), INVALID, b"aligned"),
    ("mie_paged_extend", extend_args(max_len=100000), WORKSPACE, b"workspace of 0 bytes"),
    ("mie_token_logprobs", logprobs_args(dtype=F16), UNSUPPORTED, b"float32 or bfloat16"),
    ("mie_token_logprobs", logprobs_args(rows=-1), INVALID, b"rows=-1"),
    ("mie_token_logprobs", logprobs_args(vocab=0), INVALID, b"vocab=0"),
    ("mie_token_logprobs", logprobs_args(stride=999), INVALID, b"stride=999"),
    ("mie_token_logprobs", logprobs_args(top=65), INVALID, b"top 65"),
    ("mie_token_logprobs", logprobs_args(vocab=4, top=5), INVALID, b"top 5"),
    ("mie_token_logprobs", logprobs_args(top=-1), INVALID, b"top -1"),
    ("mie_token_logprobs", logprobs_args(tokens=None), INVALID, b"null pointer"),
    ("mie_token_logprobs", logprobs_args(top_tokens=None), INVALID, b"null pointer"),
]


@pytest.mark.parametrize("name,args,status,message", CASES, ids=[f"{c[0]}-{i}" for i, c in enumerate(CASES)])
def test_a_bad_argument_fails_on_the_host(name, args, status, message):
    lib = _native.lib()
    rc = getattr(lib, name)(*args.values())
    err = lib.mie_last_error()
    assert rc == status, err
    assert message in err, err


def test_nothing_to_do_launches_nothing():
    lib = _native.lib()
    assert lib.mie_rope_append(*rope_args(tokens=0).values()) == 0
    assert lib.mie_paged_extend(*extend_args(tokens=0).values()) == 0
    assert lib.mie_paged_extend(*extend_args(max_new=0).values()) == 0
    assert lib.mie_token_logprobs(*logprobs_args(rows=0).values()) == 0


def test_the_workspace_query_answers_on_the_host():
    query = _native.lib().mie_paged_extend_workspace
    assert query(1, 1, 1, 200, 0, 12, 12, 64, BF16) == 0          # one piece
    long = query(1, 1, 1, 131072, 0, 12, 12, 64, BF16)
    assert 0 < long < 1 << 26
    assert query(1, 1, 1, 131072, 100, 12, 12, 64, BF16) < long   # a window bounds the keys
    assert query(0, 1, 1, 131072, 0, 12, 12, 64, BF16) == 0
    assert query(1, 1, 1, 200, 0, 12, 5, 64, BF16) == -INVALID
    assert query(1, 1, 1, 200, 0, 12, 12, 65, BF16) == -UNSUPPORTED


# ---- Python ---------------------------------------------------------------------


@pytest.fixture
def device(monkeypatch):
    """CPU tensors pass for a device's: every check runs, and what would be
    launched is an error."""
    monkeypatch.setattr(_native, "is_rocm_device", lambda t: True)

    class NoLaunch:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(_native, "lib", lambda: NoLaunch())


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


RESERVE = dict(free_ids=i32(*range(9)), free_count=i32(9), block_tables=torch.zeros(2, 5, dtype=torch.int32),
               context_lens=i32(3, 4), new_lens=i32(1, 1), block_size=4, max_tokens=8)


@pytest.mark.parametrize("change,message", [
    (dict(free_ids=torch.arange(9)), "free_ids"), (dict(free_ids=i32(*range(18))[::2]), "free_ids"),
    (dict(free_count=i32(1, 2)), "free_count"), (dict(block_tables=i32(1, 2)), "block tables"),
    (dict(block_tables=torch.zeros(5, 2, dtype=torch.int32).t()), "block tables"),
    (dict(block_tables=torch.zeros(1, 5, dtype=torch.int32).expand(2, 5)), "block tables"),
    (dict(context_lens=i32(1)), "context_lens"), (dict(new_lens=i32(1)), "new_lens"),
    (dict(new_lens=torch.tensor([1, 1])), "new_lens"), (dict(block_size=0), "block_size"),
    (dict(max_tokens=-1), "max_tokens"),
], ids=str)
def test_reserve_refuses(device, change, message):
    with pytest.raises(ValueError, match=message):
        kv_ops.reserve(**{**RESERVE, **change})


@pytest.mark.parametrize("finished", [i32(1, 0), torch.tensor([True]), torch.ones(4, dtype=torch.bool)[::2]])
def test_release_refuses(device, finished):
    with pytest.raises(ValueError, match="finished"):
        kv_ops.release(RESERVE["free_ids"], RESERVE["free_count"], RESERVE["block_tables"], RESERVE["context_lens"],
                       finished, 4)


def test_step_operators_need_a_device():
    with pytest.raises(RuntimeError, match="ROCm"):
        kv_ops.reserve(**RESERVE)
    with pytest.raises(RuntimeError, match="ROCm"):
        kv_ops.rope_append(**ROPE)
    with pytest.raises(RuntimeError, match="ROCm"):
        paged_attention.extend_batched(**EXTEND)
    with pytest.raises(RuntimeError, match="ROCm"):
        projection.token_logprobs(torch.zeros(2, 5))


ROPE = dict(q=torch.zeros(3, 4, 8), k=torch.zeros(3, 2, 8), v=torch.zeros(3, 2, 8), k_pool=torch.zeros(1, 5, 2, 4, 8),
            v_pool=torch.zeros(1, 5, 2, 4, 8), layer_idx=0, slots=torch.arange(3), positions=i32(0, 1, 2),
            frequencies=torch.ones(4, dtype=torch.float64))


@pytest.mark.parametrize("change,error,message", [
    (dict(q=torch.zeros(3, 4, 6)), ValueError, "q must be"), (dict(q=torch.zeros(2, 4, 8)), ValueError, "q must be"),
    (dict(k=torch.zeros(3, 4, 8)), ValueError, "q must be"), (dict(v=torch.zeros(3, 2, 6)), ValueError, "q must be"),
    (dict(q=torch.zeros(3, 4, 8).bfloat16()), ValueError, "must be torch.float32"),
    (dict(slots=i32(0, 1, 2)), ValueError, "slots"), (dict(positions=torch.arange(3)), ValueError, "positions"),
    (dict(frequencies=torch.ones(4)), ValueError, "frequencies"), (dict(layer_idx=1), IndexError, "layer 1"),
    (dict(out=torch.zeros(3, 4, 6)), ValueError, "out"), (dict(out=torch.zeros(3, 1, 8).expand(3, 4, 8)), ValueError, "out"),
    (dict(q=torch.zeros(3, 4, 8, requires_grad=True)), RuntimeError, "backward"),
], ids=str)
def test_rope_append_refuses(device, change, error, message):
    with pytest.raises(error, match=message):
        kv_ops.rope_append(**{**ROPE, **change})


EXTEND = dict(q=torch.zeros(3, 4, 64), k_pool=torch.zeros(1, 5, 2, 4, 64), v_pool=torch.zeros(1, 5, 2, 4, 64), layer_idx=0,
              block_tables=torch.zeros(2, 3, dtype=torch.int32), starts=i32(0, 1, 3), context_lens=i32(5, 6),
              max_new_tokens=2, max_context_len=12)


@pytest.mark.parametrize("change,error,message", [
    (dict(q=torch.zeros(3, 64)), ValueError, "q must be"), (dict(layer_idx=-1), IndexError, "layer -1"),
    (dict(q=torch.zeros(3, 3, 64)), ValueError, "heads"), (dict(q=torch.zeros(3, 4, 32)), ValueError, "heads"),
    (dict(q=torch.zeros(3, 4, 64).bfloat16()), ValueError, "dtype"),
    (dict(block_tables=torch.zeros(2, 3)), ValueError, "block tables"), (dict(starts=i32(0, 1)), ValueError, "starts"),
    (dict(context_lens=torch.tensor([5, 6])), ValueError, "context_lens"), (dict(prefix_lens=i32(1)), ValueError, "prefix"),
    (dict(slopes=torch.zeros(2)), ValueError, "slopes"), (dict(slopes=torch.zeros(4).double()), ValueError, "slopes"),
    (dict(window=-1), ValueError, "window"), (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=math.nan), ValueError, "softcap"), (dict(out=torch.zeros(3, 4, 32)), ValueError, "out must be"),
    (dict(out=EXTEND["q"]), ValueError, "out must not be q"), (dict(softcap=1025), ValueError, "softcap"),
    (dict(max_context_len=2**32 + 5), ValueError, "max_context_len"),
    (dict(out=torch.zeros(3, 64, 4).transpose(1, 2)), ValueError, "unit inner stride"),
    (dict(block_tables=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "block tables"),
    (dict(q=torch.zeros(3, 4, 64, requires_grad=True)), RuntimeError, "backward"),
], ids=str)
def test_extend_batched_refuses(device, change, error, message):
    with pytest.raises(error, match=message):
        paged_attention.extend_batched(**{**EXTEND, **change})


def test_extend_batched_names_what_it_is_not_built_for(device):
    pool = torch.zeros(1, 5, 2, 4, 48)
    with pytest.raises(RuntimeError, match="head_dim 48"):
        paged_attention.extend_batched(**{**EXTEND, "q": torch.zeros(3, 4, 48), "k_pool": pool, "v_pool": pool})
    half = {k: EXTEND[k].half() for k in ("q", "k_pool", "v_pool")}
    with pytest.raises(RuntimeError, match="float16"):
        paged_attention.extend_batched(**{**EXTEND, **half})


@pytest.mark.parametrize("args,message", [
    ((torch.zeros(5),), "logits"), ((torch.zeros(2, 5).half(),), "logits"), ((torch.zeros(2, 0),), "logits"),
    ((torch.zeros(2, 5), torch.zeros(3, dtype=torch.long)), "tokens"), ((torch.zeros(2, 5), i32(0, 1)), "tokens"),
    ((torch.zeros(2, 5), None, 6), "top 6"), ((torch.zeros(2, 100), None, 65), "top 65"),
    ((torch.zeros(2, 5), None, -1), "top -1"),
], ids=str)
def test_token_logprobs_refuses(device, args, message):
    with pytest.raises(ValueError, match=message):
        projection.token_logprobs(*args)


def test_token_logprobs_refuses_gradients(device):
    with pytest.raises(RuntimeError, match="backward"):
        projection.token_logprobs(torch.zeros(2, 5, requires_grad=True))


@pytest.mark.parametrize("args,kw", [
    ((7,), {}), ((0,), {}), ((8,), dict(scaling="other")), ((8,), dict(scaling="linear", scale=0.5)), ((8, 1.0), {}),
    ((8,), dict(scaling="yarn", scale=2.0)), ((2,), dict(scaling="ntk", scale=2.0)),
    ((8,), dict(scaling="yarn", original_length=100, beta_fast=1.0, beta_slow=1.0)), ((8, math.inf), {}),
], ids=str)
def test_rope_frequencies_refuses(args, kw):
    with pytest.raises(ValueError):
        kv_ops.rope_frequencies(*args, **kw)


def test_free_blocks_are_handed_over_once():
    from moe_engine.model import BlockAllocator, ModelConfig

    allocator = BlockAllocator(ModelConfig(num_layers=1, hidden_dim=8, num_heads=1), 10, 4, "cpu")
    ids, count = kv_ops.take_free_blocks(allocator, 6)
    assert ids.tolist() == [4, 5, 6, 7, 8, 9] and count.tolist() == [6] and allocator.free_blocks == [0, 1, 2, 3]
    for bad in (0, 5, -1):
        with pytest.raises(ValueError, match="count"):
            kv_ops.take_free_blocks(allocator, bad)
    allocator.free(ids.tolist())
    assert sorted(allocator.free_blocks) == list(range(10))
