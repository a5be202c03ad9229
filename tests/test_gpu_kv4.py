"""The paged 4-bit key/value cache on the GPU against plain 64-bit definitions (oracle/kv4.py).

Codes, parameters, plans and gathered numbers are compared bit for bit.  Attention is held to
bounds that follow from its roundings, with u = 2^-8 (bf16) or 2^-11 (fp16) the largest
relative rounding error of the type.  The kernels round the output once, the probabilities
(times a scale) once, and the kernel for many queries also keys and values; each is an
independent relative error of at most u, about u / sqrt(3) on average, on summands whose
root-sum-square is `spread`.  A key's error moves a score by about u / sqrt(3) * |q| |k| / sqrt(D)
~ u for the inputs here, and its probability by as much.  Four such errors add to about
1.2 u in the 2-norm (bound: 1.5 u, as |out| ~ spread), and to 8 u, over six standard deviations,
for a single element."""
from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import kv4 as ref
from triton_fused_rmsnorm_qkv import (KV4Cache, device_status, kv4_append, kv4_attention, kv4_cache, kv4_gather,
                                      kv4_plan)

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LAYOUTS = [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)]
DT = [torch.bfloat16, torch.float16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def heads(seed, *shape, dtype=torch.bfloat16):
    """Activations (CPU) whose spread and offset differ from channel to channel."""
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(0.4 * torch.randn(shape[-1], generator=g))
    offset = 0.5 * torch.randn(shape[-1], generator=g)
    return (torch.randn(*shape, generator=g) * spread + offset).to(dtype)


@pytest.fixture(autouse=True)
def clean_status():
    yield
    assert device_status() == 0


# ------------------------------------------------------------------ plan
PLANS = [  # context, new, block, blocks short, surplus tokens
    ([0], [1], 16, 0, 0),
    ([5], [0], 16, 0, 0),
    ([15, 16, 17, 0], [1, 1, 1, 1], 16, 0, 2),
    ([0, 31, 32, 33, 100], [100, 2, 0, 64, 1], 32, 0, 0),
    ([10, 20, 30, 16], [40, 50, 60, 1], 16, 3, 0),
    ([16, 16, 3], [16, 1, 2], 16, 99, 0),            # nothing free: only the last fits its block
    ([4, -1, 7, 9], [3, 5, -2, 30], 16, 0, 1),       # negative lengths
]


def _plan_case(ctx, new, block, short, surplus, seed=0, width=None):
    rng = random.Random(seed)
    have = [ref.blocks_of(max(c, 0), block) for c in ctx]
    want = [ref.blocks_of(max(c, 0) + max(n, 0), block) for c, n in zip(ctx, new)]
    need = sum(w - h for w, h in zip(want, have))
    n_free = max(0, need + 2 - short) if short else need + 2
    ids = list(range(sum(have) + n_free))
    rng.shuffle(ids)
    width = max(want) + 2 if width is None else width
    tables, at = [], 0
    for h in have:
        tables.append((ids[at:at + h] + [-1] * width)[:width])
        at += h
    return tables, ids[at:] + [-7, -7], n_free, sum(max(n, 0) for n in new) + surplus


def _check_plan(ctx, new, tables, free, n_free, block, n_tokens, out=None):
    dev = i32(tables)
    got = kv4_plan(i32(ctx), i32(new), dev, i32(free), i32([n_free]), block_size=block, n_tokens=n_tokens, out=out)
    want = ref.plan(ctx, new, tables, free, n_free, block, n_tokens)
    for name in got._fields:
        assert getattr(got, name).tolist() == want[name], name
    assert dev.tolist() == tables
    return got


@pytest.mark.parametrize("ctx,new,block,short,surplus", PLANS)
def test_plan(ctx, new, block, short, surplus):
    tables, free, n_free, n_tokens = _plan_case(ctx, new, block, short, surplus)
    _check_plan(ctx, new, tables, free, n_free, block, n_tokens)


@pytest.mark.parametrize("R,hi,new,block", [(513, 300, 3, 16), (1300, 90, 1, 32), (3, 9000, 7000, 48), (600, 64, 40, 128)])
@pytest.mark.parametrize("short", [0, 17])
def test_plan_many(R, hi, new, block, short):
    rng = random.Random(R + short)
    ctx, add = [rng.randint(0, hi) for _ in range(R)], [rng.randint(0, new) for _ in range(R)]
    tables, free, n_free, n_tokens = _plan_case(ctx, add, block, short, 5, seed=R)
    _check_plan(ctx, add, tables, free, n_free, block, n_tokens)


def test_plan_narrow_table_few_tokens_and_reused_buffers():
    ctx, new = [20, 40, 3, 8], [20, 60, 2, 4]
    tables, free, n_free, _ = _plan_case(ctx, new, 16, 0, 0, width=4)   # request 1 needs 7 blocks
    plan = _check_plan(ctx, new, [list(t) for t in tables], free, n_free, 16, 86)
    assert plan.refused.item() == 1
    # the last request's tokens do not fit; the same buffers are written again
    plan = _check_plan(ctx, new, [list(t) for t in tables], free, n_free, 16, 84)
    _check_plan(ctx, new, tables, free, n_free, 16, 84, out=plan)
    assert plan.refused.item() == 2


# ------------------------------------------------------------------ append and gather
def _store_reference(data, x, slots, kind, block, group):
    """The cache bytes (CPU) after storing x (T, n_kv, D)."""
    code, scale, low = ref.quantise(x, group)
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        for h in range(x.shape[1]):
            ref.write_token(data[slot // block, h, slot % block // 16], slot % 16, kind, code[t, h], scale[t, h],
                            low[t, h])
    return code, scale, low


@pytest.mark.parametrize("dtype", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_append_bytes_and_gather(D, group, dtype):
    n_kv, block, T = 3, 32, 45
    cache = kv4_cache(5, n_kv, D, block_size=block, group_size=group, dtype=dtype)
    cache.data.random_(0, 256)
    before = cache.data.cpu()
    k, v = (heads(s, T, n_kv, D, dtype=dtype) for s in (1, 2))
    k[3, 1] = 0.25                       # a constant row: scale 0
    v[4, 0, :5] = math.inf
    k[5, 2, 7] = math.nan
    v[6] = 60000.0 if dtype == torch.float16 else 3e38
    v[6, :, ::2] *= -1                   # a range near (fp16) or past (bf16) the type's largest value
    k[7] *= 1e-6
    rng = random.Random(D + group)
    slots = rng.sample(range(5 * block), T - 20)
    slots = slots[:13] + [s for s in range(40, 60)] + [-1] * 12   # scattered, a run, padding
    slots = [s if slots.index(s) == i or s < 0 else -1 for i, s in enumerate(slots)]
    kv4_append(cache, k.cuda(), v.cuda(), i32(slots))
    parts = [_store_reference(before, x, slots, kind, block, group) for x, kind in ((k, "k"), (v, "v"))]
    # NaN parameters are compared as NaN, everything else byte by byte
    got = cache.data.cpu()
    rec = got.flatten(0, 2), before.flatten(0, 2)
    assert torch.equal(rec[0][:, :16 * D], rec[1][:, :16 * D])
    a, b = (r[:, 16 * D:].contiguous().view(dtype).float() for r in rec)
    written = torch.isfinite(b)
    assert torch.equal(a[written], b[written]) and torch.equal(torch.isnan(a), torch.isnan(b))
    for x, (code, scale, low) in zip(kv4_gather(cache, i32(slots)), parts):
        want = ref.values(code, scale, low).float().to(dtype)   # exact in 64 bits, then in 32
        want[torch.tensor(slots) < 0] = 0
        x = x.cpu()
        assert torch.equal(torch.isnan(x), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(x, 0.0), torch.nan_to_num(want, 0.0))


@pytest.mark.parametrize("B,S", [(1, 1), (3, 17), (2, 160)])
def test_append_layouts(B, S):
    """Head-major, token-major, strided and misaligned keys store the same codes."""
    n_kv, D, block = 2, 128, 16
    k, v = (heads(s, B, n_kv, S, D).cuda() for s in (3, 4))
    slots = i32(random.Random(S).sample(range(B * S + 64), B * S))
    first = None
    wide = torch.zeros(B, n_kv, S, D + 16, dtype=k.dtype, device="cuda")
    wide[..., 8:8 + D] = k
    odd = torch.zeros(B, n_kv, S, D + 3, dtype=k.dtype, device="cuda")
    odd[..., 1:1 + D] = k
    rows = k.transpose(1, 2).reshape(B * S, n_kv, D)
    vrows = v.transpose(1, 2).reshape(B * S, n_kv, D)
    for kk, vv in ((k, v), (wide[..., 8:8 + D], v), (odd[..., 1:1 + D], v), (rows, vrows),
                   (rows.transpose(0, 1).contiguous().transpose(0, 1), vrows)):
        cache = kv4_cache((B * S + 64) // block + 1, n_kv, D, block_size=block)
        kv4_append(cache, kk, vv, slots)
        first = cache.data if first is None else first
        assert torch.equal(cache.data, first)


def test_slots_past_the_cache_are_skipped():
    cache = kv4_cache(2, 1, 64, block_size=16)
    k = heads(1, 3, 1, 64).cuda()
    kv4_append(cache, k, k, i32([31, 32, 2 ** 31 - 1]))
    got, _ = kv4_gather(cache, i32([31, 32, 2 ** 31 - 1]))
    assert device_status() == 2 and got[0].abs().sum() > 0 and not got[1:].any()


# ------------------------------------------------------------------ attention
class Batch:
    """Requests of `total` tokens of which the last `new` are queries, in a shuffled paged cache
    whose unused bytes are all ones (NaN parameters)."""

    def __init__(self, total, new, n_q, n_kv, D, group, block, dtype, seed=0, spare=3):
        self.total, self.new, self.dtype = total, new, dtype
        counts = [ref.blocks_of(t, block) for t in total]
        ids = list(range(sum(counts) + spare))
        random.Random(seed).shuffle(ids)
        self.width = max(counts) + 1
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(ids[at:at + n] + [-5] * (self.width - n))
            at += n
        data = torch.full((len(ids), n_kv, block // 16, ref.record_bytes(D, group)), 255, dtype=torch.uint8,
                          device="cuda")
        self.cache = KV4Cache(data, head_dim=D, block_size=block, group_size=group, dtype=dtype)
        T = sum(total)
        self.k, self.v = (heads(seed + s, T, n_kv, D, dtype=dtype) for s in (1, 2))
        self.q = heads(seed + 3, sum(new), n_q, D, dtype=dtype)
        self.slots = [tab[t // block] * block + t % block for tab, n in zip(self.tables, total) for t in range(n)]
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)

    def fill(self):
        if self.slots:
            kv4_append(self.cache, self.k.cuda(), self.v.cuda(), i32(self.slots))

    def call(self, **kw):
        args = dict(max_query_len=max(self.new))
        args.update(kw)
        return kv4_attention(self.q.cuda(), self.cache, i32(self.tables), i32(self.total), i32(self.start), **args)

    def reference(self, **kw):
        group = self.cache.group_size
        k, v = (ref.values(*ref.quantise(x, group)) for x in (self.k, self.v))
        out, spread, at = [], [], 0
        for r, (t, n) in enumerate(zip(self.total, self.new)):
            o, s = ref.attention(self.q[self.start[r]:self.start[r + 1]].double(), k[at:at + t], v[at:at + t], n, **kw)
            out.append(o)
            spread.append(s)
            at += t
        return torch.cat(out), torch.cat(spread)

    def check(self, got=None, **kw):
        got = (self.call(**kw) if got is None else got).cpu().double()
        kw.pop("max_query_len", None)
        want, spread = self.reference(**kw)
        u = U[self.dtype]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        got, want, spread = (torch.nan_to_num(x, 0.0) for x in (got, want, spread))
        bound = 8 * u * torch.maximum(want.abs(), spread) + 1e-30
        assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()
        if want.norm() > 0:
            assert (got - want).norm() <= 1.5 * u * want.norm(), (got - want).norm() / want.norm() / u


EDGES = [1, 15, 16, 17, 31, 32, 33, 47, 64, 65, 255, 257]


@pytest.mark.parametrize("dtype", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,group", LAYOUTS)
@pytest.mark.parametrize("n_kv,G", [(2, 1), (2, 4), (1, 7), (1, 16)])
def test_decode_edges(n_kv, G, D, group, dtype):
    b = Batch(EDGES, [1] * len(EDGES), n_kv * G, n_kv, D, group, 32, dtype, seed=D + group + G)
    b.fill()
    b.check()


@pytest.mark.parametrize("block", [16, 48, 128])
@pytest.mark.parametrize("window", [None, 1, 16, 100, 5000])
def test_decode_long_and_windows(block, window):
    total = [3001, 1, 777, 4096]
    b = Batch(total, [1] * 4, 8, 2, 128, 128, block, torch.bfloat16, seed=block)
    b.fill()
    b.check(window=window)


@pytest.mark.parametrize("D,group,dtype", [(128, 128, torch.bfloat16), (128, 32, torch.float16), (64, 64, torch.bfloat16)])
@pytest.mark.parametrize("new,G", [(2, 4), (5, 8), (9, 7), (40, 3), (130, 4), (33, 1)])
@pytest.mark.parametrize("window", [None, 37])
def test_several_queries(new, G, D, group, dtype, window):
    total = [new, new + 1, 300, 64 + new, 1000]
    news = [new, 1, min(new, 300), new, 0]
    b = Batch(total, news, 2 * G, 2, D, group, 16, dtype, seed=new)
    b.fill()
    b.check(window=window)
    b.check(window=window, max_query_len=None)     # the hint does not change what is right
    b.check(window=window, max_query_len=1)


def test_empty_requests_and_queries_before_the_cache():
    """No tokens: zeros.  More queries than tokens: those before the first token give zeros."""
    b = Batch([0, 5, 0, 3], [1, 1, 0, 6], 8, 2, 128, 64, 16, torch.bfloat16)
    b.fill()
    out = b.call()
    assert not out[0].any() and not out[2:5].any()
    b.check(out)


@pytest.mark.parametrize("new", [3, 40, 300])
def test_refused_requests_give_zeros(new):
    """seq_lens 0 with queries, as the plan leaves a request that it refuses, beside others."""
    b = Batch([0, 300, 0, new], [new, 1, 7, new], 8, 2, 128, 128, 16, torch.bfloat16, seed=new)
    b.fill()
    out = b.call()
    assert not out[:new].any() and not out[new + 1:new + 8].any()
    b.check(out)


def test_negative_scale_and_many_requests():
    """More requests than threads of a block, of one to three tokens; scores times a negative number."""
    rng = random.Random(5)
    total = [rng.randint(0, 40) for _ in range(700)]
    new = [min(t, rng.randint(0, 3)) for t in total]
    b = Batch(total, new, 4, 1, 64, 64, 16, torch.float16, seed=8)
    b.fill()
    b.check(scale=-0.05)
    b.check(scale=-0.05, max_query_len=1000)


@pytest.mark.parametrize("new", [4, 40, 200])
def test_nan_and_infinity_stay_where_they_are_seen(new):
    """A NaN key, an infinite value: queries before them are exact, queries after them are NaN."""
    b = Batch([new + 20, 90], [new, 1], 8, 2, 128, 64, 16, torch.bfloat16, seed=7)
    b.k[20 + new // 2, 0, 3] = math.nan
    b.v[20 + new - 1, 1, 9] = math.inf
    b.fill()
    out = b.call().cpu()
    assert out[new // 2:new, :4].isnan().all() and not out[:new // 2].isnan().any()
    assert out[new - 1, 4:].isnan().all() and not out[:new - 1, 4:].isnan().any()
    assert not out[new:].isnan().any()
    b.check(out)


def test_large_scores_and_custom_scale():
    b = Batch([700, 33], [1, 1], 8, 2, 128, 128, 16, torch.bfloat16, seed=5)
    b.fill()
    b.check(scale=0.02)
    b.q = b.q * 40      # scores in the hundreds: one key takes nearly all the weight
    out = b.call().cpu()
    assert torch.isfinite(out).all()
    want, _ = b.reference()
    assert (out.double() - want).norm() <= 0.05 * want.norm()


def test_layouts_streams_graph_and_out():
    """Head-major and strided queries, out=, another stream and a replayed graph give equal bits."""
    B, S, n_q, n_kv, D = 3, 4, 8, 2, 128
    b = Batch([100, 400, 77], [S] * B, n_q, n_kv, D, 128, 16, torch.bfloat16, seed=9)
    b.fill()
    first = b.call()
    b.check(first)
    q4 = b.q.cuda().view(B, S, n_q, D).transpose(1, 2)
    tables, lens = i32(b.tables), i32(b.total)
    for q in (q4, q4.contiguous()):
        assert torch.equal(kv4_attention(q, b.cache, tables, lens).view(-1, n_q, D), first)
    wide = torch.zeros(B * S, n_q + 2, D + 8, dtype=q4.dtype, device="cuda")
    wide[:, 1:-1, :D] = b.q.cuda()
    out = torch.full((B * S, n_q + 1, D), 7.0, dtype=q4.dtype, device="cuda")
    start = i32(b.start)
    kv4_attention(wide[:, 1:-1, :D], b.cache, tables, lens, start, max_query_len=S, out=out[:, :n_q])
    assert torch.equal(out[:, :n_q], first) and (out[:, n_q] == 7).all()
    table_wide = torch.full((B, b.width + 5), -9, dtype=torch.int32, device="cuda")
    table_wide[:, :b.width] = tables
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kv4_attention(q4, b.cache, table_wide[:, :b.width], lens)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(again.view(-1, n_q, D), first)
    with torch.cuda.graph(graph, stream=side):
        held = kv4_attention(q4, b.cache, tables, lens)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held.view(-1, n_q, D), first)


def test_repeatable_bits():
    b = Batch([5000, 3, 1200], [1] * 3, 8, 2, 128, 128, 16, torch.bfloat16, seed=4)
    b.fill()
    first = b.call()
    assert all(torch.equal(b.call(), first) for _ in range(20))


def test_offsets_past_32_bits():
    """Blocks at the far end of a cache of over 4 GB."""
    n_kv, D, block = 8, 128, 128
    n_blocks = (5 << 30) // (n_kv * (block // 16) * ref.record_bytes(D, D))
    b = Batch([300, 200], [1, 1], 8, n_kv, D, D, block, torch.bfloat16, seed=3)
    data = torch.empty(n_blocks, *b.cache.data.shape[1:], dtype=torch.uint8, device="cuda")
    b.cache = KV4Cache(data, head_dim=D, block_size=block, dtype=torch.bfloat16)
    far = n_blocks - 10
    b.tables = [[far + x if x >= 0 else x for x in t] for t in b.tables]
    b.slots = [s + far * block for s in b.slots]
    assert data.numel() > 1 << 32
    b.fill()
    b.check()
    k, _ = kv4_gather(b.cache, i32(b.slots))
    want = ref.values(*ref.quantise(b.k, D)).float().to(torch.bfloat16)
    assert torch.equal(k.cpu(), want)


def test_bad_indices_are_reported():
    """A block id outside the cache, a length past the table, starts outside q: a status, no access."""
    b = Batch([40, 50], [1, 1], 8, 2, 128, 128, 16, torch.bfloat16)
    b.fill()
    good = b.tables[1][1]
    b.tables[1][1] = 1 << 30
    b.call()
    assert device_status() == 2
    b.tables[1][1] = good
    for total, start in (([40, 10 ** 6], [0, 1, 2]), ([40, 50], [0, 1, 900]), ([-4, 50], [0, 1, 2])):
        kv4_attention(b.q.cuda(), b.cache, i32(b.tables), i32(total), i32(start), max_query_len=1)
        assert device_status() == 2
    b.check()


def test_plan_append_attend_together():
    """Two steps of a served batch: prompts, then single tokens, every address from the plan."""
    n_q, n_kv, D, block = 8, 2, 64, 16
    cache = kv4_cache(40, n_kv, D, block_size=block, dtype=torch.float16)
    cache.data.fill_(255)
    tables = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.randperm(40, device="cuda").int(), i32([40])
    ctx = i32([0, 0, 0])
    ks, vs, past = [[], [], []], [[], [], []], [0, 0, 0]
    for new in ([33, 1, 70], [1, 1, 1], [4, 0, 1]):
        T = sum(new)
        plan = kv4_plan(ctx, i32(new), tables, free, n_free, block_size=block, n_tokens=T)
        k, v = (heads(T + s, T, n_kv, D, dtype=torch.float16) for s in (1, 2))
        q = heads(T + 3, T, n_q, D, dtype=torch.float16)
        kv4_append(cache, k.cuda(), v.cuda(), plan.slots)
        out = kv4_attention(q.cuda(), cache, tables, plan.seq_lens, plan.query_start, max_query_len=max(new)).cpu()
        at = 0
        for r, n in enumerate(new):
            ks[r].append(k[at:at + n])
            vs[r].append(v[at:at + n])
            kk, vv = (ref.values(*ref.quantise(torch.cat(x[r]), D)) for x in (ks, vs))
            want, spread = ref.attention(q[at:at + n].double(), kk, vv, n)
            assert ((out[at:at + n].double() - want).abs() <= 8 * U[torch.float16] * torch.maximum(want.abs(), spread)).all()
            at += n
        ctx, n_free = plan.seq_lens, plan.n_free
        assert plan.refused.item() == 0


# ------------------------------------------------------------------ refusals
def test_refusals():
    b = Batch([40, 50], [1, 1], 8, 2, 128, 128, 16, torch.bfloat16)
    q, c, t, n, s = b.q.cuda(), b.cache, i32(b.tables), i32(b.total), i32(b.start)
    for error, args, kw in [
        (TypeError, (q.half(), c, t, n, s), {}),
        (TypeError, (q, c, t.long(), n, s), {}),
        (TypeError, (q, c, t, n.long(), s), {}),
        (ValueError, (q[..., :64], c, t, n, s), {}),
        (ValueError, (q[:, :3], c, t, n, s), {}),
        (ValueError, (q, c, t[:1], n, s), {}),
        (ValueError, (q, c, t.t(), n, s), {}),
        (ValueError, (q, c, t, n, s[:2]), {}),
        (ValueError, (q[:1], c, t, n), {}),
        (ValueError, (q.view(1, 2, 8, 128).transpose(1, 2), c, t, n), {}),
        (ValueError, (q.view(2, 1, 8, 128).transpose(1, 2), c, t, n, s), {}),
        (ValueError, (q, c, t, n, s), dict(window=0)),
        (ValueError, (q, c, t, n, s), dict(max_query_len=-1)),
        (ValueError, (q, c, t, n, s), dict(out=q[:1])),
        (ValueError, (q, c, t, n, s), dict(out=q)),
        (ValueError, (q, c, t, n.cpu(), s), {}),
        (AssertionError, (q.cpu(), c, t, n, s), {}),
    ]:
        with pytest.raises(error):
            kv4_attention(*args, **kw)
    k = b.k.cuda()
    slots = i32(b.slots)
    for error, args in [(TypeError, (k.half(), k, slots)), (ValueError, (k[:, :1], k, slots)),
                        (ValueError, (k, k[:5], slots)), (ValueError, (k, k, slots[:5])),
                        (TypeError, (k, k, slots.long())), (ValueError, (k, k, slots.cpu()))]:
        with pytest.raises(error):
            kv4_append(c, *args)
    with pytest.raises(TypeError):
        kv4_gather(c, slots.long())
    r = i32([1, 2])
    for error, kw in [(ValueError, dict(block_size=8)), (ValueError, dict(n_tokens=-1)), (TypeError, dict(ctx=r.long())),
                      (ValueError, dict(new=r[:1])), (ValueError, dict(n_free=r)), (ValueError, dict(table=t[:1]))]:
        a = dict(ctx=r, new=r, table=t, free=slots, n_free=r[:1], block_size=16, n_tokens=3)
        a.update(kw)
        with pytest.raises(error):
            kv4_plan(a["ctx"], a["new"], a["table"], a["free"], a["n_free"], block_size=a["block_size"],
                     n_tokens=a["n_tokens"])
    data = c.data
    for error, args, kw in [(TypeError, (data.int(),), {}), (ValueError, (data[:, :, :, 16:],), {}),
                            (ValueError, (data,), dict(head_dim=96)), (ValueError, (data,), dict(block_size=24)),
                            (ValueError, (data[:0],), {}), (TypeError, (data,), dict(dtype=torch.float32)),
                            (AssertionError, (data.cpu(),), {})]:
        a = dict(head_dim=128, block_size=16, group_size=128)
        a.update(kw)
        with pytest.raises(error):
            KV4Cache(*args, **a)
