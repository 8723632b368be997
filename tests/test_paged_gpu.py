"""The paged-cache serving operators on a B200: block tables and slot maps, the
cache write through the slot map, and the attention over a shared prefix and the
requests' own blocks, against plain implementations (whole numbers exactly,
attention in float64).

Bound of the attention: with p_j the softmax weights and V bounded by vmax, the
kernel rounds each P to f16 (relative 2^-11, or 2^-25 absolute below f16's normal
range, with the row maximum's P at least 1) and the output once (2^-11 |ref|);
f32 scores and the exponential add about 1e-5. So
    |got - ref| <= 2^-11 |ref| + (2^-11 + keys * 2^-25 + 1e-5) vmax
holds for every element. On random V the roundings of P have independent signs,
so the relative L2 error stays below 2^-11 (output) + 2^-11 (P).
"""
from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def ceil(a, b):
    return -(-a // b)


class Batch:
    """A paged batch: pool, tables, lengths and the step's tokens."""

    def __init__(self, new, lens, Hq, Hkv, D, P, prefix, seed=0, pad=(0, 0), junk=float("nan"),
                 spread=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rng = random.Random(seed)
        self.new, self.lens, self.P, self.D, self.prefix = new, lens, P, D, prefix
        self.Hq, self.Hkv = Hq, Hkv
        B = len(new)
        blocks = [ceil(n, P) for n in lens]
        pb = ceil(prefix, P)
        total = pb + sum(blocks) + 3
        ids = list(range(total))
        rng.shuffle(ids)
        self.prefix_ids, at = ids[:pb], pb
        cols = max(blocks + [1]) + 1
        table = torch.full((B, cols + 3), -7, dtype=torch.int32)[:, :cols]
        self.ids = []
        for b, n in enumerate(blocks):
            self.ids.append(ids[at:at + n])
            table[b, :n] = torch.tensor(self.ids[-1], dtype=torch.int32)
            at += n
        base = torch.full((B, cols + 3), -7, **I32)
        self.table = base[:, :cols]
        self.table.copy_(table)

        def pool():
            # every row that no length covers holds junk
            x = torch.full((total, 2 if spread else 1, Hkv, P, D), junk, dtype=torch.float16, device=DEV)
            return x[:, 0]

        self.k, self.v = pool(), pool()
        for owner, n in [(self.prefix_ids, prefix)] + list(zip(self.ids, lens)):
            for i, blk in enumerate(owner):
                rows = min(P, n - i * P)
                for c in (self.k, self.v):
                    c[blk, :, :rows] = torch.randn(Hkv, rows, D, device=DEV, generator=g).half()
        T = sum(new)
        self.lo, self.T = pad[0], T
        wide = torch.randn(T + sum(pad), (Hq + 2) * D, device=DEV, generator=g).half()
        self.q = wide[:, D:(Hq + 1) * D].unflatten(1, (Hq, D))
        starts = [self.lo]
        for n in new:
            starts.append(starts[-1] + n)
        self.q_start = torch.tensor(starts, **I32)
        self.kv_lens = torch.tensor(lens, **I32)
        self.prefix_table = torch.tensor(self.prefix_ids or [0], **I32)

    def rows(self, cache, ids, n):
        if not ids:
            return torch.zeros(self.Hkv, 0, self.D, dtype=torch.float64, device=DEV)
        return torch.cat([cache[i] for i in ids], 1)[:, :n].double()

    def reference(self, scale, causal):
        out = torch.zeros(self.T, self.Hq, self.D, dtype=torch.float64, device=DEV)
        kp, vp = self.rows(self.k, self.prefix_ids, self.prefix), self.rows(self.v, self.prefix_ids, self.prefix)
        t = 0
        for b, n in enumerate(self.new):
            q = self.q[self.lo + t:self.lo + t + n].double().view(n, self.Hkv, self.Hq // self.Hkv, self.D)
            L = self.lens[b]
            k = torch.cat([kp, self.rows(self.k, self.ids[b], L)], 1)
            v = torch.cat([vp, self.rows(self.v, self.ids[b], L)], 1)
            s = torch.einsum("nhgd,hkd->nhgk", q, k) * scale
            if causal:
                i = torch.arange(n, device=DEV)[:, None]
                j = torch.arange(self.prefix + L, device=DEV)[None]
                hidden = (j >= self.prefix) & (j - self.prefix > L - n + i)
                s = s.masked_fill(hidden[:, None, None], -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[t:t + n] = torch.einsum("nhgk,hkd->nhgd", p, v).reshape(n, self.Hq, self.D)
            t += n
        return out

    def run(self, pkg, **kw):
        kw.setdefault("prefix_table", self.prefix_table)
        return pkg.attention_paged(self.q, self.k, self.v, self.q_start, self.kv_lens, self.table,
                                   prefix_len=self.prefix, **kw)

    def check(self, pkg, causal=True, scale=None, **kw):
        out = torch.full(self.q.shape, 77.0, dtype=torch.float16, device=DEV)
        self.run(pkg, causal=causal, scale=scale, out=out, **kw)
        torch.cuda.synchronize()
        assert pkg.device_status() == 0
        got = out[self.lo:self.lo + self.T].double()
        ref = self.reference(self.D ** -0.5 if scale is None else scale, causal)
        assert bool((out[:self.lo] == 77).all()) and bool((out[self.lo + self.T:] == 77).all())
        if self.T == 0:
            return
        keys = self.prefix + max(self.lens)
        vmax = torch.nan_to_num(self.v.double(), nan=0.0).abs().max()
        bound = 2 ** -11 * ref.abs() + (2 ** -11 + keys * 2 ** -25 + 1e-5) * vmax
        diff = (got - ref).abs()
        assert bool((diff <= bound).all()), f"max |d| {diff.max():.4g}"
        norm = ref.norm()
        if norm > 0:
            assert (got - ref).norm() / norm <= 2 ** -10


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("new,lens,Hq,Hkv,D,P,prefix,causal", [
    ([1], [1], 1, 1, 128, 16, 0, True),                    # one token, one key
    ([1], [0], 4, 1, 128, 16, 1, True),                    # the prefix is all there is
    ([1], [37], 9, 3, 64, 16, 200, True),                  # the small model's heads
    ([1] * 5, [1, 128, 129, 255, 300], 32, 8, 128, 16, 500, True),
    ([1] * 3, [64, 700, 5], 8, 8, 128, 64, 128, True),     # no grouping, whole prefix blocks
    ([1] * 70, [i % 90 for i in range(70)], 32, 8, 128, 32, 129, True),   # two-tile units
    ([1] * 33, [200] * 33, 28, 4, 128, 16, 777, True),     # group 7
    ([2, 8, 1, 5], [2, 300, 1, 64], 28, 4, 128, 16, 1000, True),
    ([0, 3, 0, 0, 1, 0], [7, 3, 0, 500, 0, 9], 8, 2, 64, 16, 65, True),   # requests without tokens
    ([130, 1, 77], [130, 1, 200], 32, 8, 128, 128, 300, True),            # prompt chunks
    ([300], [300], 8, 1, 128, 256, 0, True),               # plain causal prefill
    ([300], [100], 4, 2, 64, 16, 0, True),                 # more tokens than keys: empty rows
    ([20, 3], [5, 0], 4, 2, 128, 16, 0, True),
    ([40], [333], 12, 4, 64, 1024, 0, False),              # not causal, a large block
    ([9, 2], [50, 400], 9, 1, 128, 16, 31, False),         # group 9
    ([3, 40], [3, 90], 11, 1, 64, 16, 100, True),          # group 11: one box per tile
    ([2, 1], [9, 300], 16, 1, 128, 16, 2000, True),        # group 16
    ([1, 5], [200, 7], 40, 1, 128, 16, 50, True),          # group 40
    ([2, 1], [20, 260], 128, 1, 64, 16, 130, True),        # a tile per token
    ([1] * 17, [40 * i for i in range(17)], 8, 1, 128, 16, 0, True),      # no prefix, ragged
    ([1] * 600, [(i * 7) % 40 for i in range(600)], 4, 2, 64, 16, 70, True),  # many requests
    ([1] * 2, [3000, 17], 32, 8, 128, 16, 4000, True),     # cut across many CTAs
    # a prefix that many rows share beside short requests: both roles in one launch
    ([1] * 9, [40 * i for i in range(9)], 16, 1, 128, 16, 300, True),
    ([2] * 40, [2 + (i * 13) % 500 for i in range(40)], 8, 2, 128, 32, 700, True),
    ([1] * 24, [(i * 91) % 1000 for i in range(24)], 32, 8, 64, 16, 129, True),
    ([1] * 20, [0] * 20, 32, 8, 128, 16, 1000, True),
    ([1, 0, 2] * 30, [(i * 7) % 300 for i in range(90)], 12, 4, 64, 16, 90, True),
    # every request fills tiles by itself: each visits the prefix before its own keys
    ([200, 150], [200, 300], 8, 2, 128, 16, 300, True),
    ([64, 100, 0, 33], [64, 10, 9, 700], 32, 8, 128, 128, 129, True),
    ([700], [900], 16, 2, 64, 32, 1000, True),
    ([150, 140], [0, 333], 9, 3, 64, 16, 77, True),
    ([130, 257], [300, 20], 4, 4, 128, 64, 128, False),
])
def test_attention_paged_vs_float64(cuda_pkg, new, lens, Hq, Hkv, D, P, prefix, causal):
    Batch(new, lens, Hq, Hkv, D, P, prefix, seed=sum(lens) + prefix).check(
        cuda_pkg, causal=causal, max_q_len=max(new))


@pytest.mark.parametrize("hint", [0, 1, 4, 10 ** 6])
def test_attention_paged_max_q_len_is_a_hint(cuda_pkg, hint):
    Batch([1, 30, 2, 1], [50, 30, 129, 1], 8, 2, 128, 16, 140, seed=3).check(cuda_pkg, max_q_len=hint)


@pytest.mark.parametrize("new", [[1, 2], [1, 30, 2, 1]])
def test_attention_paged_hints_above_the_batch_are_all_its_tokens(cuda_pkg, new):
    """A hint of more tokens than the batch has, the largest number among them, is the
    same as all its tokens: the same kernels, so the same bits."""
    b = Batch(new, [50 + 9 * i for i in range(len(new))], 8, 2, 128, 16, 140, seed=3)
    want = b.run(cuda_pkg, max_q_len=sum(new)).clone()
    for hint in (sum(new) + 5, 2 ** 61, 2 ** 63 - 1):
        b.check(cuda_pkg, max_q_len=hint)
        assert torch.equal(b.run(cuda_pkg, max_q_len=hint), want)


def test_attention_paged_padded_rows_and_block_stride(cuda_pkg):
    """Rows around the batch's are left as they are; K and V blocks may be
    further apart than they are long."""
    Batch([3, 1, 9], [20, 300, 9], 8, 2, 128, 32, 77, pad=(5, 11), spread=1).check(cuda_pkg)
    Batch([1, 1], [20, 300], 4, 2, 64, 32, 0, pad=(1, 2), spread=1).check(cuda_pkg, max_q_len=1)


def test_paged_entries_take_any_stride_of_an_axis_of_one(cuda_pkg):
    """One head: [blocks, rows, 1, D] storage is [blocks, 1, rows, D] too, and a query
    may be columns of wider rows. One token: its pitch is no matter."""
    g = torch.Generator(device=DEV).manual_seed(7)
    P, D, n = 16, 64, 5
    src = torch.randn(n, 4 * D, device=DEV, generator=g).half()
    slots = torch.arange(n, device=DEV) + 3
    seen = []
    for odd in (False, True):
        k, v = (torch.zeros(2, P, D, dtype=torch.float16, device=DEV)
                .as_strided((2, 1, P, D), (P * D, D if odd else P * D, D, 1)) for _ in "kv")
        q = src.as_strided((n, 1, D), (4 * D, 4 * D if odd else D, 1))
        out = torch.zeros(n, 4 * D, dtype=torch.float16, device=DEV).as_strided(q.shape, q.stride())
        cuda_pkg.kv_cache_write_paged(src[1:, D:2 * D], src[1:, 2 * D:3 * D], k, v, slots[1:])
        k0, v0 = src[:1, D:2 * D], src[:1, 2 * D:3 * D]
        cuda_pkg.kv_cache_write_paged(k0, v0.clone() if odd else v0, k, v, slots)
        cuda_pkg.attention_paged(q, k, v, torch.tensor([0, n], **I32), torch.tensor([n + 3], **I32),
                                 torch.zeros(1, 1, **I32), out=out)
        seen.append((k, v, out))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(*seen))
    assert torch.equal(seen[1][0][0, 0, 3:8], src[:, D:2 * D]) and bool((seen[1][2] != 0).any())
    assert cuda_pkg.device_status() == 0


@pytest.mark.parametrize("junk", [float("inf"), -65504.0, 65504.0])
def test_attention_paged_ignores_rows_behind_the_lengths(cuda_pkg, junk):
    Batch([1, 4], [130, 7], 8, 2, 128, 64, 33, junk=junk).check(cuda_pkg)


def test_attention_paged_large_scores(cuda_pkg):
    """Growing scores move the running maximum; lowest f16 keys leave weight 0."""
    b = Batch([2, 1], [900, 500], 8, 2, 128, 16, 600, seed=5)
    n = b.prefix // b.P
    for i, blk in enumerate(b.prefix_ids):
        b.k[blk] *= 0.2 + 3.0 * i / n
    for i, blk in enumerate(b.ids[0]):
        b.k[blk] *= 0.2 + 4.0 * i / len(b.ids[0])
    b.check(cuda_pkg, scale=0.3)
    b = Batch([1, 1], [40, 20], 4, 4, 64, 16, 20, seed=6)
    b.k[b.ids[0][1]] = -65504.0
    b.check(cuda_pkg)


def test_attention_paged_nan_query_stays_in_its_row(cuda_pkg):
    b = Batch([1, 1, 1], [40, 20, 300], 8, 2, 128, 16, 200, seed=8)
    want = b.run(cuda_pkg).clone()
    b.q[1, 3] = float("nan")
    got = b.run(cuda_pkg)
    torch.cuda.synchronize()
    assert bool(torch.isnan(got[1, 3]).all())
    got[1, 3] = want[1, 3]
    assert torch.equal(got, want)


def test_attention_paged_same_result_every_time(cuda_pkg):
    b = Batch([1] * 40, [(i * 37) % 700 for i in range(40)], 32, 8, 128, 16, 3000, seed=9)
    first = b.run(cuda_pkg).clone()
    for _ in range(3):
        assert torch.equal(b.run(cuda_pkg), first)
    ws = torch.full((cuda_pkg.attention_paged_workspace_bytes(40, 32, 128, 3000),), 255,
                    dtype=torch.uint8, device=DEV)
    assert torch.equal(b.run(cuda_pkg, workspace=ws), first)


def test_paged_cache_offsets_beyond_32_bits(cuda_pkg):
    """Blocks 2^31 elements apart: the write lands in them and attention reads them."""
    Hkv, P, D, far = 2, 16, 128, (1 << 31) + 64
    block = Hkv * P * D
    store = torch.empty(2 * far + 2 * block, dtype=torch.float16, device=DEV)
    k, v = (store[i * block:].as_strided((3, Hkv, P, D), (far, P * D, D, 1)) for i in range(2))
    g = torch.Generator(device=DEV).manual_seed(1)
    T, n = 40, 3
    src = torch.randn(T, 2 * Hkv * D, device=DEV, generator=g).half()
    slots = torch.cat([torch.arange(16) + 32, torch.arange(16), torch.arange(8) + 16]).to(DEV)
    cuda_pkg.kv_cache_write_paged(src[:, :Hkv * D], src[:, Hkv * D:], k, v, slots)
    assert torch.equal(v[2, 1], src[:16, 3 * D:])
    q = torch.randn(n, 8, D, device=DEV, generator=g).half()
    for hint in (1, n):  # both kernels
        got = cuda_pkg.attention_paged(q, k, v, torch.tensor([0, n], **I32), torch.tensor([T - 16], **I32),
                                       torch.tensor([[0, 1]], **I32), max_q_len=hint,
                                       prefix_table=torch.tensor([2], **I32), prefix_len=16)
        kk, vv = src[:, :Hkv * D].double().view(T, Hkv, D), src[:, Hkv * D:].double().view(T, Hkv, D)
        s = torch.einsum("nhgd,khd->nhgk", q.double().view(n, Hkv, 4, D), kk) * D ** -0.5
        hidden = torch.arange(T, device=DEV)[None] > T - n + torch.arange(n, device=DEV)[:, None]
        p = torch.softmax(s.masked_fill(hidden[:, None, None], -math.inf), -1)
        want = torch.einsum("nhgk,khd->nhgd", p, vv).reshape(n, 8, D)
        bound = 2 ** -11 * want.abs() + (2 ** -11 + T * 2 ** -25 + 1e-5) * vv.abs().max()
        assert bool(((got.double() - want).abs() <= bound).all())
    assert cuda_pkg.device_status() == 0


def test_attention_paged_call_of_seconds(cuda_pkg):
    """A call longer than the limit of one wait of its kernels, with whole key blocks
    only. Every key set below is the 1024 rows of one cache block over and over, so
    its softmax is that of the 1024 rows."""
    n, Hq, Hkv, P, D, times = 16384, 32, 8, 1024, 128, 12000
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(1, Hkv, P, D, device=DEV, generator=g).half() for _ in range(2))
    q = torch.randn(n, Hq, D, device=DEV, generator=g).half()
    table = torch.zeros(1, times, **I32)
    start, lens = torch.tensor([0, n], **I32), torch.tensor([P * times], **I32)
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    got = cuda_pkg.attention_paged(q, k, v, start, lens, table, causal=False)
    t1.record()
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 0
    assert t0.elapsed_time(t1) > 2000
    some = torch.cat([torch.arange(0, n, 997), torch.tensor([n - 1])]).to(DEV)
    qq = q[some].double().view(-1, Hkv, Hq // Hkv, D)
    p = torch.softmax(torch.einsum("nhgd,hkd->nhgk", qq, k[0].double()) * D ** -0.5, -1)
    want = torch.einsum("nhgk,hkd->nhgd", p, v[0].double()).reshape(-1, Hq, D)
    # P in f16; the sum of a row adds 12000 * 8 blocks' sums in f32, each addition off
    # by at most 2^-24 of the sum so far, and O the 8 products of each block
    blocks = times * P // 128
    bound = 2 ** -11 * want.abs() + (2 ** -11 + (blocks + 8 * blocks) * 2 ** -24) * v.abs().max()
    assert bool(((got[some].double() - want).abs() <= bound).all())


def counting_caches(ids, Hkv, P, D):
    """K of zeros (every visible key has the same weight) and V that says where a row
    comes from: block i of head h has a one in column (8 i + row // 128 + h) % D."""
    k = torch.zeros(ids, Hkv, P, D, dtype=torch.float16, device=DEV)
    i, h, r = (torch.arange(n, device=DEV) for n in (ids, Hkv, P))
    col = (8 * i[:, None, None] + r[None, None] // 128 + h[None, :, None]) % D
    return k, torch.nn.functional.one_hot(col, D).half()


def counted(times, Hkv, D):
    """[Hkv, D] outputs for a table with times[i] entries of block i (of 1024 rows)."""
    want = torch.zeros(Hkv, D, dtype=torch.float64)
    for i, n in enumerate(times):
        for g in range(8):
            for h in range(Hkv):
                want[h, (8 * i + g + h) % D] += n
    return (want / (8 * sum(times))).to(DEV)


def test_attention_paged_call_of_seconds_counts_every_block(cuda_pkg):
    """A call of the wide kernel of some seconds: 16 cache blocks in a shuffled table, each
    so often as no other. A key block lost or taken twice changes a column by 1 / 900 of
    its value or more, above twice the bound. Weights and V are ones, their sums whole
    numbers below 2^24; what is rounded is the quotient (2^-22), the log2 of a cut unit's
    sum (below 32, 1.5 * 2^-19) and the f16 result, by 2^-11 + 2^-17 of its value at
    most."""
    n, Hq, Hkv, P, D = 16384, 32, 8, 1024, 128
    times = list(range(600, 920, 20))
    k, v = counting_caches(16, Hkv, P, D)
    g = torch.Generator(device=DEV).manual_seed(3)
    table = torch.arange(16, **I32).repeat_interleave(torch.tensor(times, device=DEV))
    table = table[torch.randperm(sum(times), device=DEV, generator=g)][None]
    q = torch.randn(n, Hq, D, device=DEV, generator=g).half()
    got = cuda_pkg.attention_paged(q, k, v, torch.tensor([0, n], **I32),
                                   torch.tensor([P * sum(times)], **I32), table, causal=False)
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 0
    want = counted(times, Hkv, D).repeat_interleave(Hq // Hkv, 0)
    assert bool(((got.double() - want).abs() <= (2 ** -11 + 2 ** -17) * want).all())


@pytest.mark.parametrize("short", [0, 5])
def test_attention_paged_long_item_of_the_narrow_kernel(cuda_pkg, short):
    """A decode request whose part of one CTA lasts longer than the limit of one wait
    (2.8 million key blocks), and 100 short items (one per KV head, with and without
    keys) behind it in the same CTA. Sums of weights and of V are whole numbers below
    2^24 or rounded by 2^-24, the log2 of a piece's sum (below 32) by 1.5 * 2^-19, so the
    f16 result is off by 2^-11 + 2^-17 of its value at most."""
    Hkv, P, D, cols = 100, 1024, 128, (1 << 20) - 1
    times = [300001, cols - 300001]
    k, v = counting_caches(2, Hkv, P, D)
    g = torch.Generator(device=DEV).manual_seed(4)
    table = torch.zeros(2, cols, **I32)
    table[0, torch.randperm(cols, device=DEV, generator=g)[:times[1]]] = 1
    q = torch.randn(2, Hkv, D, device=DEV, generator=g).half()
    got = cuda_pkg.attention_paged(q, k, v, torch.tensor([0, 1, 2], **I32),
                                   torch.tensor([cols * P, short], **I32), table, max_q_len=1).double()
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 0
    want = counted(times, Hkv, D)
    assert bool(((got[0] - want).abs() <= (2 ** -11 + 2 ** -17) * want).all())
    assert torch.equal(got[1], v[0, :, 0].double() * (short > 0))


def test_attention_paged_two_streams(cuda_pkg):
    """Calls with workspaces of their own may run at the same time."""
    batches = [Batch([1] * 20, [30 + i * s for i in range(20)], 32, 8, 128, 16, 900, seed=s)
               for s in (11, 12)]
    want = [b.run(cuda_pkg).clone() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[] for _ in batches]
    for _ in range(5):
        for i, (b, s) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.run(cuda_pkg))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_attention_paged_two_streams_with_both_kernels(cuda_pkg):
    """The same where each call has its two kernels side by side, beside other work."""
    batches = [Batch([1] * 60, [30 + i * s for i in range(60)], 32, 8, 128, 16, p, seed=s)
               for s, p in ((11, 4000), (12, 9000))] + [Batch([150, 90], [300, 90], 32, 8, 128, 16, 400)]
    want = [b.run(cuda_pkg, max_q_len=max(b.new)).clone() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[] for _ in batches]
    for _ in range(8):
        for i, (b, s) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.run(cuda_pkg, max_q_len=max(b.new)))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
    assert cuda_pkg.device_status() == 0


def test_attention_paged_graphs_on_one_workspace(cuda_pkg):
    """Graphs of both kernels and eager calls take turns on one workspace."""
    batches = [Batch([1] * 20, [30 + i * s for i in range(20)], 32, 8, 128, 16, p, seed=s)
               for s, p in ((11, 900), (12, 0))] + [Batch([200, 90], [300, 90], 32, 8, 128, 16, 400)]
    want = [b.run(cuda_pkg, max_q_len=max(b.new)).clone() for b in batches]
    nbytes = max(cuda_pkg.attention_paged_workspace_bytes(b.q.shape[0], b.Hq, b.D, b.prefix)
                 for b in batches)
    workspace = torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV)
    graphs, outs = [], []
    for b in batches:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(b.run(cuda_pkg, max_q_len=max(b.new), workspace=workspace))
    for i in (0, 1, 2, 1, 0, 2, 2, 0):
        outs[i].zero_()
        graphs[i].replay()
        j = (i + 1) % 3
        eager = batches[j].run(cuda_pkg, max_q_len=max(batches[j].new), workspace=workspace)
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i]) and torch.equal(eager, want[j])
    assert cuda_pkg.device_status() == 0


@pytest.mark.parametrize("B,D,prefix,top", [(40, 128, 4096, 300), (64, 64, 9001, 40),
                                            (200, 128, 1500, 900)])
def test_attention_paged_both_kernels_follow_inputs_in_a_graph(cuda_pkg, B, D, prefix, top):
    """A prefix and the requests' own keys side by side: lengths and queries that the
    launch just before has written, replay after replay."""
    b = Batch([1] * B, [(i * 37) % top for i in range(B)], 32, 8, D, 16, prefix, seed=3)
    full = b.kv_lens.clone()
    step, q0 = torch.zeros_like(full), b.q.clone()
    want = []
    for i in range(4):
        b.kv_lens.copy_((full - i * 16).clamp_(min=0))
        b.lens = b.kv_lens.tolist()
        b.q.copy_(q0.roll(i, 0))
        torch.cuda.synchronize()
        b.check(cuda_pkg, max_q_len=1)
        want.append(b.run(cuda_pkg, max_q_len=1).clone())
    out = torch.empty_like(want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.kv_lens.copy_(torch.clamp(full - step * 16, min=0))
        b.q.copy_(torch.index_select(q0, 0, (torch.arange(B, device=DEV) - step[0]) % B))
        b.run(cuda_pkg, max_q_len=1, out=out)
    for i in (0, 3, 1, 2, 0, 1, 3):
        step.fill_(i)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    assert cuda_pkg.device_status() == 0


def test_attention_paged_bad_indices_are_reported_not_followed(cuda_pkg):
    b = Batch([1, 1], [40, 300], 8, 2, 128, 16, 100, seed=13)
    want = b.run(cuda_pkg).clone()
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 0
    b.table[0, 1] = 1 << 20
    got = b.run(cuda_pkg)
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 2
    assert torch.equal(got[1], want[1])  # the other request is not affected
    b.table[0, 1] = -1
    b.run(cuda_pkg)
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 2
    b.table[0, 1] = b.ids[0][1]
    b.kv_lens[0] = 1 << 30  # more rows than the table has
    b.run(cuda_pkg)
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 2
    assert cuda_pkg.device_status() == 0


@pytest.mark.parametrize("keys", [1 << 30, 33 << 20])
def test_attention_paged_call_beyond_the_work_limit_is_reported(cuda_pkg, keys):
    """A prefix of one block over and over, for so many rows that the call is above
    2^30 pairs of a query tile and a key block: it returns and says so."""
    n, Hq, Hkv, P, D = 2048, 1024, 64, 1024, 64
    keys = min(keys, (1 << 30) - 1)
    k = torch.zeros(1, Hkv, P, D, dtype=torch.float16, device=DEV)
    q = torch.zeros(n, Hq, D, dtype=torch.float16, device=DEV)
    table = torch.zeros(1, (1 << 20) - 1, **I32)
    assert cuda_pkg.device_status() == 0
    cuda_pkg.attention_paged(q, k, k, torch.tensor([0, n], **I32), torch.tensor([2100], **I32), table,
                             prefix_table=torch.zeros(1 << 20, **I32), prefix_len=keys, max_q_len=1)
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 2
    Batch([1] * 20, [30 + i for i in range(20)], 32, 8, 128, 16, 900).check(cuda_pkg, max_q_len=1)


# --------------------------------------------------------------------- tables
def plain_tables(cached, new, free, cursor, table, P, max_tokens):
    """The definition, request by request."""
    starts, slots, short = [0], [], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        for col in range(ceil(c, P), ceil(c + n, P)):
            if cursor < len(free):
                table[b][col] = free[cursor]
                cursor += 1
            else:
                table[b][col] = -1
                short += 1
        for pos in range(c, c + n):
            blk = table[b][pos // P]
            slots.append(blk * P + pos % P if blk >= 0 else -1)
        starts.append(starts[-1] + n)
    slots += [-1] * (max_tokens - len(slots))
    return starts, [c + n for c, n in zip(cached, new)], slots, [cursor, short]


def tables_case(B, new_max, cached_max, P, seed, short=0, extra=3):
    rng = random.Random(seed)
    cached = [rng.randint(0, cached_max) for _ in range(B)]
    new = [rng.randint(0, new_max) for _ in range(B)]
    cols = max(ceil(c + n, P) for c, n in zip(cached, new)) + 1
    table = [[-5] * cols for _ in range(B)]
    nxt = 100000
    for b, c in enumerate(cached):
        for col in range(ceil(c, P)):
            table[b][col] = nxt
            nxt += 1
    need = sum(ceil(c + n, P) - ceil(c, P) for c, n in zip(cached, new))
    free = list(range(need + 2 - short))
    rng.shuffle(free)
    return cached, new, free, table, sum(new) + extra


@pytest.mark.parametrize("B,new_max,cached_max,P,short,extra", [
    (1, 1, 0, 16, 0, 0), (1, 300, 40, 16, 0, 5), (7, 1, 100, 16, 0, 2), (255, 1, 4000, 64, 0, 0),
    (300, 3, 50, 1, 0, 7), (1025, 5, 300, 16, 0, 0), (3000, 2, 20, 32, 0, 1000),
    (9, 2000, 3000, 128, 0, 3), (40, 90, 100, 16, 30, 9), (5, 0, 100, 16, 0, 4),
    (16384, 2, 9, 4, 0, 0),
])
def test_paged_tables_exact(cuda_pkg, B, new_max, cached_max, P, short, extra):
    cached, new, free, table, n = tables_case(B, new_max, cached_max, P, B + P, short, extra)
    t = torch.tensor(table, **I32)
    got = cuda_pkg.paged_tables(torch.tensor(cached, **I32), torch.tensor(new, **I32),
                                torch.tensor(free, **I32), torch.tensor([2], **I32), t,
                                block_rows=P, max_tokens=n)
    want = plain_tables(cached, new, free, 2, table, P, n)
    torch.cuda.synchronize()
    for g, w, name in zip(got, want, ("q_start", "kv_lens", "slots", "cursor")):
        assert g.tolist() == w, name
    assert t.tolist() == table
    assert cuda_pkg.device_status() == 0


@pytest.mark.parametrize("B,new_max", [(3, 2), (2500, 4)])
def test_paged_tables_in_place(cuda_pkg, B, new_max):
    """The lengths and the cursor advanced where they are, step after step."""
    cached, new, free, table, _ = tables_case(B, new_max, 100, 16, 1)
    free = list(range(4 * B * new_max))
    cols = max(len(r) for r in table) + ceil(3 * new_max, 16)
    table = [r + [-5] * (cols - len(r)) for r in table]
    lens, cur, t = torch.tensor(cached, **I32), torch.tensor([0, 0], **I32), torch.tensor(table, **I32)
    n = sum(new)
    cursor = 0
    for _ in range(3):
        _, _, slots, _ = cuda_pkg.paged_tables(
            lens, torch.tensor(new, **I32), torch.tensor(free, **I32), cur, t, block_rows=16,
            max_tokens=n, kv_lens=lens, cursor_out=cur)
        _, cached, want, (cursor, short) = plain_tables(cached, new, free, cursor, table, 16, n)
        assert lens.tolist() == cached and slots.tolist() == want and cur.tolist() == [cursor, short]
        assert t.tolist() == table
    assert cuda_pkg.device_status() == 0


def test_paged_tables_in_place_at_the_largest_batch(cuda_pkg):
    """Lengths and cursor over themselves for 16384 requests (a cluster whose CTAs fill
    their shared memory), the free list short of a few blocks."""
    cached, new, free, table, n = tables_case(16384, 3, 40, 8, 5, short=12)
    lens, cur, t = torch.tensor(cached, **I32), torch.tensor([2, 0], **I32), torch.tensor(table, **I32)
    q_start, kv_lens, slots, cursor = cuda_pkg.paged_tables(
        lens, torch.tensor(new, **I32), torch.tensor(free, **I32), cur, t, block_rows=8,
        max_tokens=n, kv_lens=lens, cursor_out=cur)
    want = plain_tables(cached, new, free, 2, table, 8, n)
    assert want[3][1] > 0
    got = [x.tolist() for x in (q_start, kv_lens, slots, cursor)]
    assert got == list(want) and t.tolist() == table
    assert cuda_pkg.device_status() == 0


def test_paged_tables_returns_the_slots_of_its_step_only(cuda_pkg):
    """A slot buffer kept from a longer step: the entries behind max_tokens are the old
    step's, and rows of the cache write must not reach them."""
    def step(new, **kw):
        return cuda_pkg.paged_tables(torch.zeros(1, **I32), torch.tensor([new], **I32),
                                     torch.arange(10, **I32), torch.zeros(1, **I32),
                                     torch.zeros(1, 4, **I32), block_rows=16, **kw)[2]
    buf = step(20, max_tokens=24)
    assert buf.tolist() == list(range(20)) + [-1] * 4
    got = step(3, max_tokens=5, slots=buf)
    assert got.tolist() == [0, 1, 2, -1, -1] and got.data_ptr() == buf.data_ptr()
    assert step(3, slots=buf) is buf and buf.tolist() == [0, 1, 2] + [-1] * 21
    assert step(2, max_tokens=3, slots=buf.view(4, 6)).tolist() == [0, 1, -1]
    k = torch.zeros(4, 1, 16, 64, dtype=torch.float16, device=DEV)
    rows = torch.ones(20, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="slots"):  # more rows than the step has tokens
        cuda_pkg.kv_cache_write_paged(rows, rows, k, k.clone(), got)
    assert cuda_pkg.device_status() == 0


def test_paged_tables_out_of_range_is_reported(cuda_pkg):
    def call(cached, new, cursor=0, n=8, cols=4):
        t = torch.zeros(len(cached), cols, **I32)
        out = cuda_pkg.paged_tables(torch.tensor(cached, **I32), torch.tensor(new, **I32),
                                    torch.arange(10, **I32), torch.tensor([cursor], **I32), t,
                                    block_rows=16, max_tokens=n)
        torch.cuda.synchronize()
        return cuda_pkg.device_status(), out
    assert call([3], [2])[0] == 0
    # a table of 64 rows: rows 62 and 63 are rows 14 and 15 of its last block, 0
    bits, out = call([62], [4])
    assert bits == 2 and out[2].tolist() == [14, 15, -1, -1, -1, -1, -1, -1] and out[1].tolist() == [64]
    bits, out = call([0, 0], [6, 5])        # more tokens than slots
    assert bits == 2 and out[0].tolist() == [0, 6, 8] and -1 not in out[2].tolist()
    assert call([-1], [2])[0] == 2
    assert call([1], [-2])[0] == 2
    assert call([1], [2], cursor=-3)[0] == 2
    assert call([1], [2], cursor=11)[0] == 2
    assert call([1 << 30], [1 << 30])[0] == 2


# ---------------------------------------------------------------- cache write
@pytest.mark.parametrize("T,Hkv,D,P,spread", [
    (1, 1, 8, 16, 0), (5, 3, 64, 16, 0), (8, 8, 128, 16, 1), (333, 8, 128, 64, 0),
    (1000, 2, 96, 1024, 1), (4097, 4, 128, 32, 0), (0, 2, 64, 16, 0),
])
def test_kv_cache_write_paged_exact(cuda_pkg, T, Hkv, D, P, spread):
    g = torch.Generator(device=DEV).manual_seed(T + D)
    blocks = ceil(max(T, 1), P) + 5
    k, v = (torch.randn(blocks, 1 + spread, Hkv, P, D, device=DEV, generator=g).half()[:, 0]
            for _ in range(2))
    slots = torch.randperm(blocks * P, device=DEV, generator=g)[:T + 2]
    slots[T // 2::5] = -1
    src = torch.randn(max(T, 1), 3 * Hkv * D, device=DEV, generator=g).half()[:T]
    ks, vs = src[:, Hkv * D:2 * Hkv * D], src[:, 2 * Hkv * D:]
    wk, wv = k.clone(), v.clone()
    live = slots[:T] >= 0
    s = slots[:T][live]
    wk[s // P, :, s % P] = ks[live].unflatten(1, (Hkv, D))
    wv[s // P, :, s % P] = vs[live].unflatten(1, (Hkv, D))
    cuda_pkg.kv_cache_write_paged(ks, vs, k, v, slots)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert cuda_pkg.device_status() == 0


def test_kv_cache_write_paged_skips_slots_behind_the_cache(cuda_pkg):
    k, v = torch.zeros(2, 2, 1, 16, 64, dtype=torch.float16, device=DEV)
    src = torch.ones(3, 64, dtype=torch.float16, device=DEV)
    cuda_pkg.kv_cache_write_paged(src, src, k, v, torch.tensor([3, 32, 1 << 50], device=DEV))
    torch.cuda.synchronize()
    assert cuda_pkg.device_status() == 2
    assert float(k.sum()) == 64 and float(v.sum()) == 64


# --------------------------------------------------------------- the three together
def test_paged_step_as_a_captured_graph(cuda_pkg):
    """Prefill behind a prefix, then decode steps replayed from one graph whose
    lengths, tables and cursor advance on the GPU; every step against float64."""
    Hq, Hkv, D, P, prefix, B, steps = 8, 2, 128, 16, 50, 3, 20
    g = torch.Generator(device=DEV).manual_seed(0)
    pool = 64
    k_cache, v_cache = (torch.full((pool, Hkv, P, D), float("nan"), dtype=torch.float16, device=DEV)
                        for _ in range(2))
    free = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    cursor = torch.zeros(2, **I32)
    hist = [[] for _ in range(B + 1)]  # K/V rows of every request, the prefix last

    def tokens(counts, owners):
        qkv = torch.randn(sum(counts), (Hq + 2 * Hkv) * D, device=DEV, generator=g).half()
        t = 0
        for n, o in zip(counts, owners):
            hist[o].append(qkv[t:t + n, Hq * D:].clone())
            t += n
        return qkv

    def split(qkv):
        return (qkv[:, :Hq * D].unflatten(1, (Hq, D)), qkv[:, Hq * D:(Hq + Hkv) * D],
                qkv[:, (Hq + Hkv) * D:])

    def expect(b, q):
        kv = torch.cat(hist[B] + hist[b]).double()
        k, v = kv[:, :Hkv * D].view(-1, Hkv, D), kv[:, Hkv * D:].view(-1, Hkv, D)
        n, L = q.shape[0], kv.shape[0]
        s = torch.einsum("nhgd,khd->nhgk", q.double().view(n, Hkv, Hq // Hkv, D), k) * D ** -0.5
        hidden = torch.arange(L, device=DEV)[None] > L - n + torch.arange(n, device=DEV)[:, None]
        p = torch.softmax(s.masked_fill(hidden[:, None, None], -math.inf), -1)
        return torch.einsum("nhgk,khd->nhgd", p, v).reshape(n, Hq, D)

    def near(got, want):
        assert bool(((got.double() - want).abs() <= 2 ** -11 * want.abs() + 6 * 2 ** -11).all())

    # the prefix is a request of its own: its tables, its rows
    ptable = torch.full((1, 8), -1, **I32)
    q, k, v = split(tokens([prefix], [B]))
    zero = torch.zeros(1, **I32)
    qs, kl, slots, _ = cuda_pkg.paged_tables(zero, zero + prefix, free, cursor, ptable, block_rows=P,
                                             max_tokens=prefix, cursor_out=cursor)
    cuda_pkg.kv_cache_write_paged(k, v, k_cache, v_cache, slots)
    near(cuda_pkg.attention_paged(q, k_cache, v_cache, qs, kl, ptable),
         _causal_self(q, k, v, Hkv, D))
    # prefill of three prompts of different lengths
    counts = [5, 33, 16]
    table = torch.full((B, 8), -1, **I32)
    lens = torch.zeros(B, **I32)
    q, k, v = split(tokens(counts, range(B)))
    qs, _, slots, _ = cuda_pkg.paged_tables(lens, torch.tensor(counts, **I32), free, cursor, table,
                                            block_rows=P, max_tokens=sum(counts), kv_lens=lens,
                                            cursor_out=cursor)
    cuda_pkg.kv_cache_write_paged(k, v, k_cache, v_cache, slots)
    kw = dict(prefix_table=ptable[0, :4].contiguous(), prefix_len=prefix)
    out = cuda_pkg.attention_paged(q, k_cache, v_cache, qs, lens, table, **kw)
    t = 0
    for b, n in enumerate(counts):
        near(out[t:t + n], expect(b, q[t:t + n]))
        t += n
    # decode: one graph, its inputs rewritten before every replay; the batch has
    # room for four tokens and three requests
    buf = torch.zeros(4, (Hq + 2 * Hkv) * D, dtype=torch.float16, device=DEV)
    out = torch.full((4, Hq, D), 7.0, dtype=torch.float16, device=DEV)
    new = torch.zeros(B, **I32)
    sl, qs = torch.empty(4, dtype=torch.int64, device=DEV), torch.empty(B + 1, **I32)

    def step():
        q, k, v = split(buf)
        cuda_pkg.paged_tables(lens, new, free, cursor, table, block_rows=P, q_start=qs, kv_lens=lens,
                              slots=sl, cursor_out=cursor)
        cuda_pkg.kv_cache_write_paged(k, v, k_cache, v_cache, sl)
        cuda_pkg.attention_paged(q, k_cache, v_cache, qs, lens, table, max_q_len=1, out=out, **kw)

    step()  # no new token: nothing changes
    torch.cuda.synchronize()
    assert bool((out == 7).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        active = [b for b in range(B) if (i + b) % 4]
        new.copy_(torch.tensor([int(b in active) for b in range(B)], **I32))
        buf[:len(active)] = tokens([1] * len(active), active)
        graph.replay()
        for t, b in enumerate(active):
            near(out[t:t + 1], expect(b, buf[t:t + 1, :Hq * D].unflatten(1, (Hq, D))))
        assert bool((out[3] == 7).all())
    assert cursor.tolist()[1] == 0 and cuda_pkg.device_status() == 0


def _causal_self(q, k, v, Hkv, D):
    n, Hq = q.shape[:2]
    k, v = k.double().reshape(n, Hkv, D), v.double().reshape(n, Hkv, D)
    s = torch.einsum("nhgd,khd->nhgk", q.double().reshape(n, Hkv, Hq // Hkv, D), k) * D ** -0.5
    i = torch.arange(n, device=DEV)
    s = s.masked_fill((i[None] > i[:, None])[:, None, None], -math.inf)
    return torch.einsum("nhgk,khd->nhgd", torch.softmax(s, -1), v).reshape(n, Hq, D)
