"""What is measured of the paged-cache serving operators, and their plain forms.

Three operators serve a batch of requests from one paged KV cache: the block
tables and slot maps of a step (`paged_tables`), the cache write through the
slot map (`kv_cache_write_paged`) and the grouped-query attention of the batch
over a shared prefix and its own cached keys (`attention_paged`). A case of
kind "step" is the three in turn, as a serving loop calls them.
"""
import math
import random

import torch

own = False

DEV = "cuda"


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of a few requests: one new token each, latency only
        dict(name="tables-decode-8", kind="tables", batch=8, new_min=1, new_max=1, cached_min=1,
             cached_max=2048, block_rows=16, lens=1),
        # a serving step that mixes single tokens with chunks of prompts
        dict(name="tables-mixed-1001", kind="tables", batch=1001, new_min=0, new_max=64,
             cached_min=0, cached_max=8192, block_rows=16, lens=2),
        # the cache update of a small decode step, 8 KV heads of 128
        dict(name="write-decode-8", kind="write", batch=8, new_min=1, new_max=1, cached_min=0,
             cached_max=2048, block_rows=16, q_heads=32, kv_heads=8, head_dim=128, lens=3),
        # the cache update of a prefill step
        dict(name="write-prefill-8k", kind="write", batch=5, new_min=1500, new_max=1800,
             cached_min=0, cached_max=700, block_rows=64, q_heads=32, kv_heads=8, head_dim=128,
             lens=4),
        # one request of a small model (9 query heads on 3 KV heads of 64)
        dict(name="attention-one", kind="attention", batch=1, new_min=1, new_max=1, cached_min=36,
             cached_max=36, block_rows=16, q_heads=9, kv_heads=3, head_dim=64, prefix=200, lens=5),
        # an ordinary decode step behind a system prompt
        dict(name="attention-decode-16", kind="attention", batch=16, new_min=1, new_max=1,
             cached_min=1, cached_max=600, block_rows=16, q_heads=32, kv_heads=8, head_dim=128,
             prefix=2000, lens=6),
        # many requests asking about one long document
        dict(name="attention-decode-64-long", kind="attention", batch=64, new_min=1, new_max=1,
             cached_min=0, cached_max=500, block_rows=64, q_heads=32, kv_heads=8, head_dim=128,
             prefix=31999, lens=7),
        # a full decode batch: long prompt and long answers
        dict(name="attention-decode-256", kind="attention", batch=256, new_min=1, new_max=1,
             cached_min=0, cached_max=1100, block_rows=32, q_heads=32, kv_heads=8, head_dim=128,
             prefix=4096, lens=8),
        # several drafted tokens per request, group of 7
        dict(name="attention-steps-32", kind="attention", batch=32, new_min=2, new_max=8,
             cached_min=0, cached_max=700, block_rows=16, q_heads=28, kv_heads=4, head_dim=128,
             prefix=10000, lens=9),
        # chunks of prompts behind the shared prefix (compute-bound)
        dict(name="attention-chunks-6", kind="attention", batch=6, new_min=100, new_max=512,
             cached_min=0, cached_max=1000, block_rows=128, q_heads=32, kv_heads=8, head_dim=128,
             prefix=4096, lens=10),
        # no shared prefix: requests of very different lengths, one KV head
        dict(name="attention-ragged-48", kind="attention", batch=48, new_min=1, new_max=1,
             cached_min=0, cached_max=8191, block_rows=16, q_heads=8, kv_heads=1, head_dim=128,
             prefix=0, lens=11),
        # a whole decode step: tables, cache write, attention
        dict(name="step-decode-32", kind="step", batch=32, new_min=1, new_max=1, cached_min=1,
             cached_max=900, block_rows=16, q_heads=32, kv_heads=8, head_dim=128, prefix=4096,
             lens=12),
    ]


_HEADS = [(32, 8, 128), (9, 3, 64), (28, 4, 128), (8, 1, 128), (16, 2, 128), (12, 12, 64),
          (32, 32, 128), (14, 2, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    worst = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["tables", "write", "attention", "attention", "attention", "step"])
        c = dict(kind=kind, block_rows=rng.choice([16, 32, 64, 128]), lens=rng.randrange(1 << 30))
        if kind == "tables":
            c["batch"] = _log(rng, 1, 1500)
            c["new_max"] = _log(rng, 1, 64)
            c["new_min"] = rng.choice([0, 1, c["new_max"]])
            c["cached_min"], c["cached_max"] = 0, _log(rng, 1, 8192)
            return c
        c["q_heads"], c["kv_heads"], c["head_dim"] = rng.choice(_HEADS)
        if kind == "write":
            c["batch"] = _log(rng, 1, 64)
            c["new_max"] = _log(rng, 1, max(1, 8192 // c["batch"]))
            c["new_min"] = rng.choice([0, 1, c["new_max"]])
            c["cached_min"], c["cached_max"] = 0, _log(rng, 1, 2048)
            return c
        c["prefix"] = rng.choice([0, 1, 1, 1, 1, 1]) * _log(rng, 1, 32768)
        style = rng.choice(["decode", "decode", "steps", "chunks"])
        if style == "decode":
            c["batch"], c["new_min"], c["new_max"] = _log(rng, 1, 256), 1, 1
        elif style == "steps":
            c["batch"], c["new_min"], c["new_max"] = _log(rng, 1, 64), 1, _log(rng, 2, 12)
        else:
            c["batch"], c["new_max"] = _log(rng, 1, 8), _log(rng, 16, 512)
            c["new_min"] = rng.choice([0, 1, max(1, c["new_max"] // 4)])
        c["cached_min"], c["cached_max"] = 0, _log(rng, 1, 4096 if c["batch"] < 64 else 1100)
        pairs = c["batch"] * c["new_max"] * c["q_heads"]
        own_len = c["cached_max"] + c["new_max"]
        # (the plain form's score and key tensors stay under a few GB)
        if pairs * max(c["prefix"], own_len) <= 4e8 and \
                c["batch"] * own_len * c["kv_heads"] * c["head_dim"] <= 4e8 and _cost(c) <= worst:
            return c


def _lens(case):
    """(cached, new) tokens of every request, before the seed's shuffle."""
    rng = random.Random(case["lens"])
    cached = [rng.randint(case["cached_min"], case["cached_max"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    return cached, new


def _ceil(a, b):
    return -(-a // b)


def work(case):
    cached, new = _lens(case)
    B, P, kind = case["batch"], case["block_rows"], case["kind"]
    n = sum(new)
    out = {"bytes": 0, "flops": 0}
    if kind in ("tables", "step"):
        fresh = sum(_ceil(c + t, P) - _ceil(c, P) for c, t in zip(cached, new))
        partial = sum(1 for c, t in zip(cached, new) if c % P and t)
        # lengths in, row starts and lengths out, free ids in, table entries
        # out, entries of begun blocks in, slots out
        out["bytes"] += 16 * B + 8 * fresh + 4 * partial + 8 * n
        out["flops"] += 4 * n
    if kind in ("write", "step"):
        out["bytes"] += n * (2 * 2 * case["kv_heads"] * case["head_dim"] * 2 + 8)
    if kind in ("attention", "step"):
        D, hq, hk, L = case["head_dim"], case["q_heads"], case["kv_heads"], case["prefix"]
        own_keys = sum(c + t for c, t in zip(cached, new) if t)
        out["bytes"] += 2 * n * hq * D * 2                     # Q and O
        out["bytes"] += 2 * (L + own_keys) * hk * D * 2        # keys and values, once
        out["bytes"] += 4 * (_ceil(L, P) + sum(_ceil(c + t, P) for c, t in zip(cached, new)) + 2 * B)
        pairs = sum(t * (L + c) + t * (t + 1) // 2 for c, t in zip(cached, new))
        out["flops"] += 4 * D * hq * pairs
    return out


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rng = random.Random(seed)
    cached, new = _lens(case)
    order = list(range(case["batch"]))
    rng.shuffle(order)
    cached, new = [cached[i] for i in order], [new[i] for i in order]
    B, P, kind = case["batch"], case["block_rows"], case["kind"]
    L = case.get("prefix", 0)
    n = sum(new)
    i32 = dict(dtype=torch.int32, device=DEV)
    st = dict(case, n=n, new_top=max(new) if new else 0)
    # the pool: prefix blocks, the blocks that hold the cached tokens, free ones
    before = [_ceil(c, P) for c in cached]
    after = [_ceil(c + t, P) for c, t in zip(cached, new)]
    prefix_blocks = _ceil(L, P)
    need = prefix_blocks + sum(after)
    num_blocks = need + 8
    ids = torch.randperm(num_blocks, generator=g, device=DEV).to(torch.int32)
    cols = max(after) + 2 if after else 2
    c_t, n_t = torch.tensor(cached, **i32), torch.tensor(new, **i32)
    has = before if kind in ("tables", "step") else after
    has_t = torch.tensor(has, dtype=torch.int64, device=DEV)
    first = prefix_blocks + torch.cumsum(has_t, 0) - has_t
    j = torch.arange(cols, device=DEV)
    at = (first[:, None] + j[None]).clamp(max=num_blocks - 1)
    table = torch.where(j[None] < has_t[:, None], ids[at], torch.full((1, 1), -1, **i32))
    st.update(cached=c_t, new=n_t, block_table=table.contiguous(),
              prefix_table=ids[:prefix_blocks].contiguous(),
              free_blocks=ids[prefix_blocks + sum(has):].contiguous(),
              cursor=torch.tensor([2], **i32), cursor_out=torch.empty(2, **i32),
              q_start=torch.zeros(B + 1, **i32), kv_lens=(c_t + n_t).to(torch.int32),
              slots=torch.full((max(n, 1),), -1, dtype=torch.int64, device=DEV))
    st["q_start"][1:] = torch.cumsum(n_t, 0)
    if kind == "tables":
        return st
    hq, hk, D = case["q_heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16)

    # the projection of the step's tokens: query, key and value column blocks
    qkv = normal(max(n, 1), (hq + 2 * hk) * D)[:n]
    st["query"] = qkv[:, :hq * D].unflatten(1, (hq, D))
    st["k_src"] = qkv[:, hq * D:(hq + hk) * D]
    st["v_src"] = qkv[:, (hq + hk) * D:]
    st["k_cache"] = normal(num_blocks, hk, P, D)
    st["v_cache"] = normal(num_blocks, hk, P, D)
    if kind == "write":
        slots = _token_slots(st["cached"], st["new"], st["q_start"], st["block_table"], P, n)
        st["slots"] = slots
    st["out"] = torch.empty(n, hq, D, dtype=torch.float16, device=DEV)
    return st


def _token_slots(cached, new, q_start, table, P, n):
    tok = torch.arange(n, device=DEV)
    req = torch.searchsorted(q_start[1:].long(), tok, right=True)
    pos = cached.long()[req] + tok - q_start.long()[req]
    return table.long()[req, pos // P] * P + pos % P


# -------------------------------------------------------------------- runs
def run(state):
    kind = state["kind"]
    if kind == "tables":
        return _tables_own(state) if own else _tables(state)
    if kind == "write":
        return _write_own(state) if own else _write(state, state["slots"])
    if kind == "attention":
        return _attention_own(state) if own else _attention(state, state)
    if own:
        tables = _tables_own(state)
        _write_own(state)
        return [tables, state["k_cache"], state["v_cache"], _attention_own(state)]
    tables = _tables(state)
    caches = _write(state, tables[3])
    return [tables, *caches, _attention(state, dict(
        state, block_table=tables[0], q_start=tables[1], kv_lens=tables[2]))]


def _tables_own(st):
    q_start, kv_lens, slots, cursor = _pkg().paged_tables(
        st["cached"], st["new"], st["free_blocks"], st["cursor"], st["block_table"],
        block_rows=st["block_rows"], q_start=st["q_start"], kv_lens=st["kv_lens"],
        slots=st["slots"], cursor_out=st["cursor_out"])
    return [st["block_table"], q_start, kv_lens, slots, cursor]


def _write_own(st):
    _pkg().kv_cache_write_paged(st["k_src"], st["v_src"], st["k_cache"], st["v_cache"],
                                st["slots"])
    return [st["k_cache"], st["v_cache"]]


def _attention_own(st):
    return _pkg().attention_paged(
        st["query"], st["k_cache"], st["v_cache"], st["q_start"], st["kv_lens"],
        st["block_table"], prefix_table=st["prefix_table"], prefix_len=st["prefix"],
        max_q_len=st["new_top"], causal=True, out=st["out"])


# ------------------------------------------------------------- plain forms
def _tables(st):
    P, n = st["block_rows"], st["n"]
    cached, new, table = st["cached"].long(), st["new"].long(), st["block_table"]
    total = cached + new
    before, after = (cached + P - 1) // P, (total + P - 1) // P
    fresh = after - before
    first = st["cursor"].long() + torch.cumsum(fresh, 0) - fresh
    col = torch.arange(table.shape[1], device=DEV)[None]
    source = (first[:, None] + col - before[:, None]).clamp(0, st["free_blocks"].numel() - 1)
    table = torch.where((col >= before[:, None]) & (col < after[:, None]),
                        st["free_blocks"][source], table)
    q_start = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    slots = torch.full_like(st["slots"], -1)
    slots[:n] = _token_slots(cached, new, q_start, table, P, n)
    cursor = torch.cat([st["cursor"] + fresh.sum(), torch.zeros_like(st["cursor"])])
    return [table, q_start.to(torch.int32), total.to(torch.int32), slots, cursor.to(torch.int32)]


def _write(st, slots):
    P, D = st["block_rows"], st["head_dim"]
    slots = slots[:st["n"]]
    st["k_cache"][slots // P, :, slots % P] = st["k_src"].unflatten(1, (-1, D))
    st["v_cache"][slots // P, :, slots % P] = st["v_src"].unflatten(1, (-1, D))
    return [st["k_cache"], st["v_cache"]]


def _paged_rows(cache, table):
    """[..., blocks] ids -> [..., kv_heads, blocks * rows, D] in 32 bits."""
    x = cache[table.clamp(min=0).long()].float()
    return x.movedim(-3, -4).flatten(-3, -2)


def _attention(st, tables):
    n, hk, D, L = st["n"], st["kv_heads"], st["head_dim"], st["prefix"]
    group, scale, B = st["q_heads"] // hk, D ** -0.5, st["batch"]
    q_start, kv_lens = tables["q_start"].long(), tables["kv_lens"].long()
    q = st["query"].float().unflatten(1, (hk, group))            # [n, hk, group, D]
    top = st["new_top"]
    # the request and row of every token, and the padded [B, top] token grid
    i = torch.arange(top, device=DEV)
    new = q_start[1:] - q_start[:-1]
    real = i[None] < new[:, None]
    token = (q_start[:-1, None] + i[None]).clamp(max=n - 1)
    # own keys of every request: [B, hk, keys, D]
    k = _paged_rows(st["k_cache"], tables["block_table"])
    v = _paged_rows(st["v_cache"], tables["block_table"])
    j = torch.arange(k.shape[2], device=DEV)
    qp = q[token].transpose(1, 2).flatten(2, 3)                  # [B, hk, top * group, D]
    s = (qp @ k.transpose(-1, -2)) * scale
    last = (kv_lens - new)[:, None] + i[None]                    # [B, top]
    sees = (j[None, None] <= last[..., None]) & real[..., None]
    sees = sees.repeat_interleave(group, 1)[:, None]             # [B, 1, top * group, keys]
    s = torch.where(sees, s, torch.full_like(s[:1, :1, :1, :1], -math.inf))
    # back to tokens: [n, hk, group(, D)]
    pick = real.flatten().nonzero()[:, 0]

    def rows(x):
        return x.unflatten(2, (top, group)).transpose(1, 2).flatten(0, 1)[pick]

    m = rows(s.amax(-1))
    if L:
        kp = _paged_rows(st["k_cache"], st["prefix_table"])[:, :L]
        vp = _paged_rows(st["v_cache"], st["prefix_table"])[:, :L]
        sp = (q.movedim(1, 0).flatten(1, 2) @ kp.transpose(-1, -2)) * scale
        sp = sp.unflatten(1, (n, group))                         # [hk, n, group, L]
        m = torch.maximum(m, sp.amax(-1).transpose(0, 1))
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    mp = torch.zeros_like(s[..., 0]).unflatten(2, (top, group)).transpose(1, 2).flatten(0, 1)
    mp[pick] = m
    e = torch.exp(s - mp.unflatten(0, (B, top)).transpose(1, 2).flatten(2, 3)[..., None])
    total, value = rows(e.sum(-1)), rows(e @ v)
    if L:
        e = torch.exp(sp - m.transpose(0, 1)[..., None])
        total = total + e.sum(-1).transpose(0, 1)
        value = value + (e.flatten(1, 2) @ vp).unflatten(1, (n, group)).transpose(0, 1)
    out = torch.where(total[..., None] > 0, value / total[..., None], torch.zeros_like(value))
    return out.flatten(1, 2).to(torch.float16)


# ------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The caches written token by token, and the attention outputs from the
    definition, request by request, with the visible keys of a request in one
    softmax; the tables are whole numbers and have no such value."""
    kind = case["kind"]
    if kind == "tables":
        return None
    st = prepare(case, seed)
    P, D, L, hk = case["block_rows"], case["head_dim"], case.get("prefix", 0), case["kv_heads"]
    cached, new = st["cached"].tolist(), st["new"].tolist()
    k_cache, v_cache = st["k_cache"], st["v_cache"]
    table = st["block_table"].tolist()
    if kind == "step":  # the step's own blocks
        free, at = st["free_blocks"].tolist(), int(st["cursor"])
        for b, (c, m) in enumerate(zip(cached, new)):
            for col in range(_ceil(c, P), _ceil(c + m, P)):
                table[b][col] = free[at]
                at += 1
    if kind != "attention":
        t = 0
        for b, (c, m) in enumerate(zip(cached, new)):
            for pos in range(c, c + m):
                k_cache[table[b][pos // P], :, pos % P] = st["k_src"][t].view(hk, D)
                v_cache[table[b][pos // P], :, pos % P] = st["v_src"][t].view(hk, D)
                t += 1
    if kind == "write":
        return [k_cache.double(), v_cache.double()]

    def keys(cache, ids, length):
        blocks = cache[torch.tensor(ids, dtype=torch.long, device=DEV)].double()
        return torch.cat(list(blocks), 1)[:, :length] if ids else blocks.new_zeros(hk, 0, D)

    prefix_ids = st["prefix_table"].tolist()
    kp, vp = keys(k_cache, prefix_ids, L), keys(v_cache, prefix_ids, L)
    out = torch.zeros(st["n"], case["q_heads"], D, dtype=torch.float64, device=DEV)
    t = 0
    for b, (c, m) in enumerate(zip(cached, new)):
        if not m:
            continue
        ids = table[b][:_ceil(c + m, P)]
        ks, vs = keys(k_cache, ids, c + m), keys(v_cache, ids, c + m)
        q = st["query"][t:t + m].double().view(m, hk, -1, D)
        s = torch.cat([torch.einsum("mhgd,hkd->hgmk", q, kp), torch.einsum("mhgd,hkd->hgmk", q, ks)],
                      -1) / math.sqrt(D)
        pos = torch.arange(m, device=DEV)[:, None] + c
        hidden = torch.arange(c + m, device=DEV)[None] > pos
        s[..., L:].masked_fill_(hidden, -math.inf)
        p = torch.softmax(s, -1)
        o = torch.einsum("hgmk,hkd->mhgd", p[..., :L], vp)
        o = o + torch.einsum("hgmk,hkd->mhgd", p[..., L:], vs)
        out[t:t + m] = o.reshape(m, -1, D)
        t += m
    return out if kind == "attention" else [[None] * 5, k_cache.double(), v_cache.double(), out]
