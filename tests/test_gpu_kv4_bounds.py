"""The paged 4-bit cache where it can go wrong: tokens of no request, block ids that name no slot,
groups of very different size, one key that outweighs a long tail, NaN values whose weight
underflows, numbers at the end of the 16-bit range, windows of the largest integer and refused
requests that are tried again.  The bounds are those of test_gpu_kv4.py, applied group by group
where the groups differ; fp16 outputs below 2^-14 add half of the subnormal step, 2^-25."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import kv4 as ref
from test_gpu_kv4 import DT, U, Batch, heads, i32
from triton_fused_rmsnorm_qkv import _lib, device_status, kv4_append, kv4_attention, kv4_cache, kv4_gather, kv4_plan

pytestmark = pytest.mark.gpu
IDS = ["bf16", "fp16"]


@pytest.fixture(autouse=True)
def clean_status():
    yield
    assert device_status() == 0


def check_groups(b, group, got=None, **kw):
    """``Batch.check`` for each group of dims by itself."""
    got = (b.call(**kw) if got is None else got).cpu().double()
    kw.pop("max_query_len", None)
    want, spread = b.reference(**kw)
    u, tiny = U[b.dtype], 2.0 ** -25 if b.dtype == torch.float16 else 1e-30
    for at in range(0, want.shape[-1], group):
        g, w, s = (x[..., at:at + group] for x in (got, want, spread))
        bound = 8 * u * torch.maximum(w.abs(), s) + tiny
        assert ((g - w).abs() <= bound).all(), (at, ((g - w).abs() / bound).max())
        assert (g - w).norm() <= 1.5 * u * w.norm() + tiny * math.sqrt(w.numel()), (at, (g - w).norm() / w.norm() / u)


# ------------------------------------------------------------------ tokens of no request
@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 0], [40, 1, 90], [0, 0, 0]])
def test_tokens_of_no_request_are_zeros(new, dtype):
    """Tokens before the first request's and past the last one's, as a plan with an upper bound of
    the tokens leaves them: zeros in both kernels, whatever `out` held, also without any query."""
    b = Batch([max(n, 1) + 60 for n in new], new, 8, 2, 128, 64, 16, dtype, seed=len(new))
    b.fill()
    before, after = 2, 301
    q = torch.cat([heads(9, before, 8, 128, dtype=dtype), b.q, heads(8, after, 8, 128, dtype=dtype)]).cuda()
    start = i32([before + s for s in b.start])
    for bound in (1, q.shape[0]):
        wide = torch.full((q.shape[0], 9, 128), math.nan, dtype=dtype, device="cuda")
        for out in (torch.full_like(q, math.nan), wide[:, :8]):
            kv4_attention(q, b.cache, i32(b.tables), i32(b.total), start, max_query_len=bound, out=out)
            assert not out[:before].any() and not out[before + b.start[-1]:].any()
            if b.start[-1]:
                b.check(out[before:before + b.start[-1]])
        assert wide[:, 8].isnan().all()


def test_no_requests_give_zeros():
    b = Batch([40], [1], 8, 2, 128, 128, 16, torch.bfloat16)
    q = heads(1, 5, 8, 128).cuda()
    out = torch.full_like(q, math.nan)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    kv4_attention(q, b.cache, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), none, i32([0]), out=out)
    assert not out.any()


def test_a_padded_step_of_a_plan():
    """A plan whose token count is an upper bound, through append and attention."""
    n_kv, D, block, T = 2, 64, 16, 24
    cache = kv4_cache(8, n_kv, D, block_size=block)
    tables = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(8, device="cuda").int()
    plan = kv4_plan(i32([0, 0]), i32([5, 9]), tables, free, i32([8]), block_size=block, n_tokens=T)
    k, v, q = (heads(s, T, h, D) for s, h in ((1, n_kv), (2, n_kv), (3, 8)))
    kv4_append(cache, k.cuda(), v.cuda(), plan.slots)
    out = torch.full((T, 8, D), math.nan, dtype=q.dtype, device="cuda")
    kv4_attention(q.cuda(), cache, tables, plan.seq_lens, plan.query_start, max_query_len=9, out=out)
    assert not out[14:].any()
    kk, vv = (ref.values(*ref.quantise(x, D)) for x in (k, v))
    for lo, hi in ((0, 5), (5, 14)):
        want, spread = ref.attention(q[lo:hi].double(), kk[lo:hi], vv[lo:hi], hi - lo)
        got = out[lo:hi].cpu().double()
        assert ((got - want).abs() <= 8 * U[q.dtype] * torch.maximum(want.abs(), spread)).all()


# ------------------------------------------------------------------ block ids that name no slot
@pytest.mark.parametrize("bad", [-1, -(2 ** 31), 1 << 27, 1 << 28, 2 ** 31 - 1])
def test_plan_reports_blocks_without_a_slot(bad):
    """A held block, and a block of the free list, whose id is negative or whose slots pass 2^31."""
    plan = kv4_plan(i32([3, 20]), i32([2, 2]), i32([[bad, -1], [5, 6]]), i32([7]), i32([1]), block_size=16, n_tokens=4)
    assert device_status() == 2
    assert plan.slots.tolist() == [-1, -1, 6 * 16 + 4, 6 * 16 + 5] and plan.positions.tolist() == [3, 4, 20, 21]
    plan = kv4_plan(i32([3, 15]), i32([2, 2]), i32([[1, -1], [5, -1]]), i32([bad]), i32([1]), block_size=16, n_tokens=4)
    assert device_status() == 2
    assert plan.slots.tolist() == [19, 20, 5 * 16 + 15, -1] and plan.seq_lens.tolist() == [5, 17]


def test_plan_takes_the_last_block_with_a_slot():
    last = (2 ** 31 - 1) // 16 - 1   # its last slot is below 2^31 - 1
    plan = kv4_plan(i32([15]), i32([1]), i32([[last]]), i32([0]), i32([0]), block_size=16, n_tokens=1)
    assert plan.slots.tolist() == [last * 16 + 15]


# ------------------------------------------------------------------ refused requests
def test_a_refused_request_keeps_its_history():
    """Request 1 needs a block while none is free: it stores nothing and keeps its tokens and blocks.
    The step after, with a block given back, continues where it was."""
    n_q, n_kv, D, block = 4, 2, 64, 16
    cache = kv4_cache(5, n_kv, D, block_size=block)
    cache.data.fill_(255)
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    free, n_free = i32([3, 0, 4, 1, 2]), i32([5])
    ctx = i32([0, 0, 0])
    past_k, past_v = [[], [], []], [[], [], []]
    #        (new tokens, refused, lengths after)
    steps = [([33, 16, 2], 0, [33, 16, 2]), ([1, 1, 1], 1, [34, 16, 3]), ([1, 1, 0], 0, [35, 17, 0])]
    for step, (new, refused, after) in enumerate(steps):
        T = sum(new)
        if step == 2:    # request 2 is finished: its block is free again
            blocks = tables.cpu()
            assert blocks[1, 0] >= 0 and blocks[1, 1] == -1
            free, n_free, ctx = tables[2, :1].clone(), i32([1]), ctx * i32([1, 1, 0])
            tables[2] = -1
        plan = kv4_plan(ctx, i32(new), tables, free, n_free, block_size=block, n_tokens=T)
        k, v, q = (heads(10 * step + s, T, h, D) for s, h in ((1, n_kv), (2, n_kv), (3, n_q)))
        kv4_append(cache, k.cuda(), v.cuda(), plan.slots)
        out = kv4_attention(q.cuda(), cache, tables, plan.seq_lens, plan.query_start, max_query_len=max(new)).cpu()
        assert plan.refused.item() == refused
        lens, at = plan.seq_lens.tolist(), 0
        for r, n in enumerate(new):
            if n and lens[r] == 0:
                assert not out[at:at + n].any()
            elif n:
                past_k[r].append(k[at:at + n])
                past_v[r].append(v[at:at + n])
                kk, vv = (ref.values(*ref.quantise(torch.cat(x[r]), D)) for x in (past_k, past_v))
                want, spread = ref.attention(q[at:at + n].double(), kk, vv, n)
                err = (out[at:at + n].double() - want).abs()
                assert (err <= 8 * U[q.dtype] * torch.maximum(want.abs(), spread)).all()
            at += n
        ctx, n_free = plan.context_after(ctx), plan.n_free
        assert ctx.tolist() == after
    held = [x for row in tables.tolist() for x in row if x >= 0]
    assert len(held) == len(set(held)) == 5


def test_context_after_in_place():
    tables = i32([[0, -1], [1, -1], [2, -1]])
    ctx = i32([5, 16, 3])
    plan = kv4_plan(ctx, i32([2, 1, 0]), tables, i32([3]), i32([0]), block_size=16, n_tokens=3)
    assert plan.seq_lens.tolist() == [7, 0, 3]
    assert plan.context_after(ctx, out=ctx) is ctx and ctx.tolist() == [7, 16, 3]


# ------------------------------------------------------------------ weights of very different size
@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("D,group", [(128, 128), (64, 64), (64, 32)])
def test_a_dominant_key_and_a_long_tail(D, group, dtype):
    """131071 keys of which one outweighs each of the others by 2^25.2: together they hold 0.34 % of
    the weight, and their values are three times as large as the one key's.  The requests share
    their blocks and are so many that a warp walks through two requests' keys."""
    T, R = 131071, 4736
    b = Batch([T], [1], 2, 1, D, group, 64, dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    b.q = torch.ones(1, 2, D).to(dtype)
    b.k = torch.zeros(T, 1, D, dtype=dtype)
    b.k[777] = 25.2 * math.log(2) / math.sqrt(D)
    b.v = (6.0 + 15 * torch.rand(T, 1, D, generator=g)).to(dtype)
    b.v[777] = (15 * torch.rand(1, D, generator=g) - 7.5).to(dtype)
    b.fill()
    out = kv4_attention(b.q.cuda().expand(R, -1, -1).contiguous(), b.cache, i32(b.tables).repeat(R, 1), i32([T] * R))
    want, spread = b.reference()
    err = (out.cpu().double() - want).abs()
    assert (err <= 8 * U[dtype] * torch.maximum(want.abs(), spread)).all()
    assert (err.flatten(1).norm(dim=1) <= 1.5 * U[dtype] * want.norm()).all(), err.norm(dim=(1, 2)).max() / want.norm()


def group_factors(D, group, ratio, dtype):
    """Per dim: one group in two `ratio` times the others, centred so that fp16 holds both."""
    f = torch.ones(D // group)
    f[1::2] = ratio
    return (f / math.sqrt(ratio) if dtype == torch.float16 else f).repeat_interleave(group)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("D,group", [(128, 64), (128, 32), (64, 32)])
@pytest.mark.parametrize("ratio", [1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("total", [[1000, 33, 1], [100000]], ids=["short", "long"])
def test_groups_of_different_size(total, ratio, D, group, dtype):
    b = Batch(total, [1] * len(total), 4, 1, D, group, 64, dtype, seed=D + group)
    b.v = (b.v.float() * group_factors(D, group, ratio, dtype)).to(dtype)
    b.fill()
    check_groups(b, group)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("growing", [True, False])
def test_groups_whose_size_changes_along_the_keys(growing, dtype):
    """Values that grow or shrink by 1e4 along the keys, in one group of two, and single tokens
    whose group is 100 times its neighbours'."""
    T, D, group = 9000, 128, 32
    b = Batch([T, 500], [1, 2], 8, 2, D, group, 32, dtype, seed=11)
    n = b.v.shape[0]
    size = torch.logspace(-2, 2, n)[:, None, None]
    f = torch.ones(n, 1, D)
    wide = (torch.arange(D) // group % 2 == 1)
    f[:, :, wide] = size if growing else size.flip(0)
    f[::1777, :, wide] *= 100
    b.v = (b.v.float() * f).clamp(-60000, 60000).to(dtype)
    b.fill()
    check_groups(b, group)


def test_parameters_of_hidden_tokens_do_not_matter():
    """Tokens past the last key, beyond a query or before a window may hold any scale."""
    D, group = 128, 32
    for dtype in DT:
        b = Batch([45, 300], [2, 1], 4, 1, D, group, 16, dtype, seed=12)
        b.fill()
        first = b.call(window=37)
        big = 6e4 if dtype == torch.float16 else 1e30
        params = b.cache.data[..., 16 * D:].view(dtype).unflatten(-1, (2, 16, D // group, 2))
        flat = [s for s in range(b.cache.n_blocks * 16)]
        held = set(b.slots)
        for s in flat:   # every slot that no request holds, and those before the second one's window
            if s not in held:
                params[s // 16, 0, 0, :, s % 16] = big
        for t in range(45, 45 + 300 - 37):
            s = b.slots[t]
            params[s // 16, 0, 0, :, s % 16] = big
        assert torch.equal(b.call(window=37), first)


# ------------------------------------------------------------------ NaN, infinities, windows
@pytest.mark.parametrize("key", [0, 100, 671, 672, 690, 699])
@pytest.mark.parametrize("bound", [1, 100])
def test_a_nan_value_of_no_weight_is_seen_wherever_a_tile_ends(key, bound):
    """A NaN value whose weight underflows to zero makes a row that sees it NaN, in whole and in
    partly hidden tiles of both kernels."""
    b = Batch([700, 40], [1, 30], 2, 1, 64, 32, 16, torch.bfloat16, seed=6)
    b.q = torch.ones_like(b.q)
    b.k[key] = -40.0                # a score of -320
    b.v[key, 0, 5] = math.nan
    b.fill()
    out = b.call(max_query_len=bound).cpu()
    assert out[0].isnan().all() and not out[1:].isnan().any()


def test_a_nan_value_outside_a_window_is_not_seen():
    b = Batch([700, 40], [3, 30], 2, 1, 64, 64, 16, torch.bfloat16, seed=6)
    b.v[600, 0, 5] = math.nan       # the last position that sees it with a window of 99 is 698
    b.fill()
    for bound in (1, 100):
        out = b.call(window=99, max_query_len=bound).cpu()
        assert out[:2].isnan().all() and not out[2:].isnan().any()


@pytest.mark.parametrize("D,group", [(128, 64), (128, 32), (64, 32)])
@pytest.mark.parametrize("ratio", [1e-4, 1e-6, 1e-8])
def test_bf16_queries_whose_groups_differ(ratio, D, group):
    """Queries that are small in the groups where the keys are large: each group's share of a score
    is as large as any other's."""
    b = Batch([1000, 33], [1, 1], 4, 1, D, group, 64, torch.bfloat16, seed=D + group)
    f = group_factors(D, group, ratio, torch.bfloat16)
    b.q = (b.q.float() * f).to(b.dtype)
    b.k = (b.k.float() / f).to(b.dtype)
    b.fill()
    b.check()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 40])
@pytest.mark.parametrize("total,new", [(3, 6), (30, 60), (1, 40)])
def test_largest_window_with_more_queries_than_tokens(total, new, window):
    """Queries before the first token give zeros; the others see all that they do without a window."""
    b = Batch([total, 50], [new, 9], 4, 1, 128, 128, 16, torch.bfloat16, seed=new)
    b.fill()
    for bound in (1, 100):
        out = b.call(window=window, max_query_len=bound)
        assert torch.equal(out, b.call(max_query_len=bound))
        b.check(out)


@pytest.mark.parametrize("D,group", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("low", [0.0, -65504.0])
@pytest.mark.parametrize("where", ["k", "v"])
def test_fp16_numbers_at_the_end_of_the_range(where, low, D, group):
    """Values of up to 65504 whose scale is rounded up, so that 15 steps would end at 65520 or more:
    rows that do not see the key are untouched and rows that see it are finite.  (Queries are small
    where the key is large, so that its error of one part in 2048 moves no score by more than u.)"""
    for total, new, bound in (([300, 50], [40, 1], None), ([300, 50], [2, 1], 1), ([290, 50], [200, 3], 500)):
        b = Batch(total, new, 4, 1, D, group, 16, torch.float16, seed=D)
        x = b.k if where == "k" else b.v
        key = 299 if total[0] == 300 else 200
        x[key, 0, ::2], x[key, 0, 1::2] = low, 65504.0
        if where == "k":
            b.q = b.q * 1e-5
        b.fill()
        b.check(max_query_len=bound)
        b.check(max_query_len=bound, window=70)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("D,group", [(128, 128), (128, 32), (64, 64)])
def test_finite_rows_are_read_back_finite(D, group, dtype):
    """Rows between a low number and the type's largest: the stored bytes are the definition's, and
    no number read back is infinite or further off than a step."""
    top = torch.finfo(dtype).max
    low = torch.linspace(-1, 1, 97) * top if dtype == torch.float16 else torch.linspace(-0.0039, 1, 97) * top
    x = torch.full((97, 1, D), top).to(dtype)
    x[:, 0, ::2] = low.to(dtype)[:, None]
    x[:, 0, 1::8] = (top * 0.9 + low * 0.1).to(dtype)[:, None]
    cache = kv4_cache(7, 1, D, block_size=16, group_size=group, dtype=dtype)
    slots = i32(list(range(97)))
    kv4_append(cache, x.cuda(), x.cuda(), slots)
    code, scale, low16 = ref.quantise(x, group)
    assert torch.isfinite(scale).all()
    want = ref.values(code, scale, low16).float().to(dtype)
    for got in kv4_gather(cache, slots):
        assert torch.isfinite(got).all() and torch.equal(got.cpu(), want)
        step = scale.double().repeat_interleave(group, -1)
        assert ((got.cpu().double() - x.double()).abs() <= step).all()


def test_bf16_numbers_at_the_end_of_the_range():
    """As above in bf16, -1.3e36 .. 3.39e38; the product with a probability stays in range."""
    top = torch.finfo(torch.bfloat16).max
    b = Batch([300], [40], 4, 1, 128, 128, 16, torch.bfloat16, seed=4)
    b.v[280, 0, ::2], b.v[280, 0, 1::2] = -1.3e36, top
    b.fill()
    out = b.call().cpu()
    want, _ = b.reference()
    assert torch.isfinite(out).all()
    assert (out[:20].double() - want[:20]).norm() <= 1.5 * U[torch.bfloat16] * want[:20].norm()


# ------------------------------------------------------------------ a wait that runs out
@pytest.mark.parametrize("D,group", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("total,new,bound", [([3000, 40], [1, 1], 1), ([900, 40], [130, 9], 130)],
                         ids=["split", "prompt"])
def test_a_withheld_arrival_times_out_and_the_next_launch_is_clean(total, new, bound, D, group):
    """One arrival on one barrier is left out (FQKV_FLAG_TEST_WITHHOLD) and the limit is 1 ms: the
    launch returns, the status reports it, rows are right or NaN, the arrival counters are zero
    and the next launch is as if nothing had been."""
    b = Batch(total, new, 8, 2, D, group, 16, torch.bfloat16, seed=13)
    b.fill()
    first = b.call(max_query_len=bound)
    b.check(first)
    q, tables, lens, start = b.q.cuda(), i32(b.tables), i32(b.total), i32(b.start)
    out = torch.zeros_like(first)
    need = _lib.load().fqkv_kv4_workspace_bytes(8, 2, D, bound)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    args = [b.cache._ptr, q.data_ptr(), q.stride(0), q.stride(0), q.stride(1), 8, start.data_ptr(), q.shape[0], 0,
            len(total), bound, tables.data_ptr(), tables.stride(0), tables.shape[1], lens.data_ptr(), 0, D ** -0.5,
            out.data_ptr(), out.stride(0), ws.data_ptr(), need]
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    _lib.set_wait_limit_ns(1_000_000)
    try:
        assert _lib.kv4["attention"](*args, _lib.FLAG_PDL | _lib.FLAG_TEST_WITHHOLD, stream) == 0, _lib.last_error()
        torch.cuda.synchronize()
        status = device_status()
    finally:
        _lib.set_wait_limit_ns(0)
    assert status == _lib.STATUS_WAIT_TIMEOUT
    missing = out.isnan()
    assert missing.any() and torch.equal(out[~missing], first[~missing])
    assert int(ws[:4096].count_nonzero()) == 0
    assert _lib.kv4["attention"](*args, _lib.FLAG_PDL, stream) == 0
    assert torch.equal(out, first)
