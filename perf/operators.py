"""The paged-cache serving operators: cases, plain forms and exact values.

Three operators of one serving step over a KV cache that lives in pages:

* plan       the step's token layout from the request lengths: where each request's rows
             start, every new token's position and cache slot, and the block-table entries
             of the pages that the new tokens need (taken from a list of free pages);
* rope       rotary embedding of the q and k heads of a fused projection, with the write of
             the rotated k and the v into the pages;
* attention  each request's new tokens (one in decode, a chunk in prefill) over the pages of
             its whole sequence: causal, grouped query heads, an optional sliding window with
             a few first tokens that stay visible, an optional sink logit per query head.

`own` False computes them with elementary torch operations in fp32; `own` True makes the calls
of mlx_batch_invariant_b200.  A page holds `page` consecutive tokens of one request as
(kv_heads, page, head_dim).
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _bi():
    path = os.path.join(os.getcwd(), "mlx-batch-invariant_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mlx_batch_invariant_b200
    return mlx_batch_invariant_b200


# --------------------------------------------------------------------------- the cases
def listed():
    gqa = dict(heads=32, kv_heads=8, head_dim=128)
    return [
        # one decode step's bookkeeping for a small server: a launch's latency is all there is
        dict(name="plan_decode_r64", op="plan", requests=64, chunks=0, q_lo=1, q_hi=1,
             ctx_lo=17, ctx_hi=8191, page=16, pad=0, mix=1),
        # prompts of every length arriving together, some continuing a cached prefix
        dict(name="plan_prefill_r24", op="plan", requests=24, chunks=24, q_lo=31, q_hi=2048,
             ctx_lo=0, ctx_hi=4096, page=64, pad=37, mix=2),
        # a large deployment's step: a few prompt chunks beside thousands of decoding requests,
        # padded to the size of a captured graph
        dict(name="plan_mixed_r4096", op="plan", requests=4096, chunks=96, q_lo=128, q_hi=1024,
             ctx_lo=0, ctx_hi=8192, page=16, pad=1000, mix=3),
        # the decode step of the 8B-shaped decoder at 64 requests
        dict(name="rope_decode_bf16", op="rope", dtype="bf16", requests=64, chunks=0, q_lo=1,
             q_hi=1, ctx_lo=17, ctx_hi=8191, page=16, rot=128, pad=0, mix=4, **gqa),
        # that decoder's prefill of 8 prompts
        dict(name="rope_prefill_bf16", op="rope", dtype="bf16", requests=8, chunks=8, q_lo=700,
             q_hi=1500, ctx_lo=0, ctx_hi=512, page=64, rot=128, pad=3, mix=5, **gqa),
        # full precision, a quarter of each head rotated, a page size that is no power of two
        dict(name="rope_odd_fp32", op="rope", dtype="fp32", requests=7, chunks=5, q_lo=33,
             q_hi=401, ctx_lo=0, ctx_hi=900, page=48, rot=16, pad=5, mix=6, heads=9, kv_heads=3,
             head_dim=64),
        # one user decoding at a long context: latency, one row to spread over the GPU
        dict(name="attn_decode_r1", op="attention", dtype="bf16", requests=1, chunks=0, q_lo=1,
             q_hi=1, ctx_lo=8191, ctx_hi=8191, page=16, window=0, first=0, sinks=False, mix=7,
             **gqa),
        # a full decode batch, ragged contexts: the cache is read once, HBM bound
        dict(name="attn_decode_r64", op="attention", dtype="bf16", requests=64, chunks=0, q_lo=1,
             q_hi=1, ctx_lo=3000, ctx_hi=8191, page=64, window=0, first=0, sinks=False, mix=8,
             **gqa),
        # the chunk of a long prompt that follows 6144 cached tokens: tensor-core bound
        dict(name="attn_chunk_2048", op="attention", dtype="bf16", requests=1, chunks=1,
             q_lo=2048, q_hi=2048, ctx_lo=6144, ctx_hi=6144, page=64, window=0, first=0,
             sinks=False, mix=9, **gqa),
        # prompt chunks and decoding requests in one step, odd lengths, fp16
        dict(name="attn_mixed_fp16", op="attention", dtype="fp16", requests=19, chunks=5, q_lo=37,
             q_hi=517, ctx_lo=0, ctx_hi=4001, page=16, window=0, first=0, sinks=False, mix=10,
             **gqa),
        # a sliding-window layer with four first tokens kept and learned sink logits
        dict(name="attn_window_d64", op="attention", dtype="bf16", requests=6, chunks=4,
             q_lo=500, q_hi=1100, ctx_lo=2500, ctx_hi=6000, page=32, window=1024, first=4,
             sinks=True, mix=11, heads=32, kv_heads=4, head_dim=64),
        # full precision, ragged and small: the check runs of a model's port
        dict(name="attn_ragged_fp32", op="attention", dtype="fp32", requests=5, chunks=3, q_lo=3,
             q_hi=130, ctx_lo=0, ctx_hi=1500, page=32, window=0, first=0, sinks=True, mix=12,
             heads=8, kv_heads=2, head_dim=64),
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1)))


def draw(rng):
    op = rng.choice(["plan", "rope", "attention", "attention"])
    mix = rng.randrange(1 << 20)
    if op == "plan":
        requests = _log_int(rng, 1, 4096)
        chunks = _log_int(rng, 0, min(requests, 96))
        q_hi = _log_int(rng, 2, 1024)
        return dict(op=op, requests=requests, chunks=chunks, q_lo=_log_int(rng, 1, q_hi),
                    q_hi=q_hi, ctx_lo=0, ctx_hi=_log_int(rng, 1, 8192),
                    page=rng.choice([16, 32, 48, 64, 128]), pad=rng.choice([0, 0, 5, 131]),
                    mix=mix)
    group = rng.choice([1, 2, 3, 4, 8])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rope":
        requests = _log_int(rng, 1, 64)
        q_hi = _log_int(rng, 2, 8192 // requests)
        return dict(op=op, dtype=dtype, requests=requests, chunks=rng.randint(0, requests),
                    q_lo=_log_int(rng, 1, q_hi), q_hi=q_hi, ctx_lo=0,
                    ctx_hi=_log_int(rng, 1, 1024), page=rng.choice([16, 32, 48, 64, 128]),
                    rot=rng.choice([head_dim, head_dim, head_dim // 2]),
                    pad=rng.choice([0, 0, 3]), mix=mix, heads=group * kv_heads,
                    kv_heads=kv_heads, head_dim=head_dim)
    requests = _log_int(rng, 1, 64)
    most = 1024 if dtype == "fp32" else 8192
    ctx_hi = _log_int(rng, 16, most)
    # padded rows x keys stay below the largest listed chunk's (and far below in fp32)
    pairs = ((1 << 21) if dtype == "fp32" else (1 << 24)) // requests
    q_most = max(2, min(2048, pairs // (2 * ctx_hi), math.isqrt(pairs // 2)))
    q_hi = _log_int(rng, 2, q_most)
    window = rng.choice([0, 0, _log_int(rng, 1, 2048)])
    return dict(op=op, dtype=dtype, requests=requests,
                chunks=rng.choice([0, rng.randint(0, requests)]), q_lo=_log_int(rng, 1, q_hi),
                q_hi=q_hi, ctx_lo=rng.choice([0, ctx_hi // 2]), ctx_hi=ctx_hi,
                page=rng.choice([16, 32, 64, 128]), window=window,
                first=rng.choice([0, 4, 130]) if window else 0, sinks=rng.random() < 0.3,
                mix=mix, heads=group * kv_heads, kv_heads=kv_heads, head_dim=head_dim)


def _lengths(case):
    """(new tokens, cached tokens) of every request: `chunks` of them bring a chunk of
    q_lo..q_hi tokens, the others one token.  A case's lengths are the same for every seed."""
    rng = random.Random(case["mix"])
    n, m = case["requests"], case["chunks"]
    q = [_log_int(rng, case["q_lo"], case["q_hi"]) for _ in range(m)] + [1] * (n - m)
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(n)]
    both = list(zip(q, ctx))
    rng.shuffle(both)
    return [b[0] for b in both], [b[1] for b in both]


def _pages(n, page):
    return -(-n // page)


# --------------------------------------------------------------------------- the inputs
def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _tables(counts, spare, gen):
    """Random distinct pages for every request: the (requests, width) block table with -1 after
    each request's pages, and the pages that are left."""
    n, width = sum(counts), max(1, max(counts)) + 1
    perm = torch.randperm(n + spare, generator=gen, device="cuda").to(torch.int32)
    have = torch.arange(width, device="cuda")[None, :] < _ints(counts, torch.int64)[:, None]
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[have] = perm[:n]
    return table, perm[n:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    q, ctx = _lengths(case)
    page, total = case["page"], sum(q)
    s = dict(case=case, page=page, total=total)
    if case["op"] == "plan":
        seq_pages = [_pages(a + b, page) for a, b in zip(q, ctx)]
        new = sum(seq_pages) - sum(_pages(c, page) for c in ctx)
        full, left = _tables(seq_pages, 64, gen)
        old = torch.arange(full.shape[1], device="cuda")[None, :] < _ints(
            [_pages(c, page) for c in ctx], torch.int64)[:, None]
        table = torch.where(old, full, torch.full_like(full, -1))
        taken = full[(full >= 0) & ~old]  # the pages the new tokens will need, now free
        head = 11
        free = torch.cat((torch.full((head,), -1, dtype=torch.int32, device="cuda"), taken, left))
        s.update(query_lens=_ints(q), context_lens=_ints(ctx), table=table, free=free,
                 head=_ints([head]), tokens=total + case["pad"], new=new)
        return s
    dtype = _DTYPES[case["dtype"]]
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    counts = [_pages(a + b, page) for a, b in zip(q, ctx)]
    table, left = _tables(counts, 7, gen)
    n_pages = sum(counts) + 7
    start = [0]
    for n in q:
        start.append(start[-1] + n)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    s.update(k_cache=randn(n_pages, kv, page, d), v_cache=randn(n_pages, kv, page, d))
    if case["op"] == "rope":
        tokens = total + case["pad"]
        pos = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
        slots = pos.clone()
        pos[:total] = torch.cat([torch.arange(c, c + n, device="cuda") for n, c in zip(q, ctx)])
        row = torch.repeat_interleave(torch.arange(len(q), device="cuda"), _ints(q, torch.int64))
        slots[:total] = table[row, pos[:total] // page].long() * page + pos[:total] % page
        rot = case["rot"]
        inv = 500000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        ang = torch.arange(max(a + b for a, b in zip(q, ctx)), device="cuda",
                           dtype=torch.float64)[:, None] * inv
        s.update(qkv=randn(tokens, (heads + 2 * kv) * d), positions=pos, slots=slots,
                 cos=torch.cos(ang).float(), sin=torch.sin(ang).float(),
                 out=torch.zeros((tokens, heads, d), dtype=dtype, device="cuda"))
        return s
    s.update(q=randn(total, heads, d), table=table, query_start=_ints(start),
             seq_lens=_ints([a + b for a, b in zip(q, ctx)]),
             window=case["window"] or None, first=case["first"], q_most=max(q),
             scale=1.0 / math.sqrt(d),
             sinks=randn(heads) * 2 if case["sinks"] else None)
    return s


# --------------------------------------------------------------------------- the plain forms
def _plain_plan(s):
    page, table = s["page"], s["table"]
    q, ctx = s["query_lens"].long(), s["context_lens"].long()
    start = torch.zeros(q.numel() + 1, dtype=torch.int64, device=q.device)
    start[1:] = q.cumsum(0)
    old = (ctx + page - 1) // page
    need = (ctx + q + page - 1) // page - old
    first = s["head"].long() + need.cumsum(0) - need  # place of each request's pages in `free`
    t = torch.arange(s["tokens"], device=q.device)
    there = t < start[-1]
    r = torch.searchsorted(start[1:], t, right=True).clamp(max=q.numel() - 1)
    pos = ctx[r] + t - start[r]
    col = (pos // page).clamp(0, table.shape[1] - 1)
    fresh = col >= old[r]
    taken = s["free"][(first[r] + col - old[r]).clamp(0, s["free"].numel() - 1)]
    ids = torch.where(fresh, taken, table[r, col])
    put = there & fresh
    table[r[put], col[put]] = ids[put]
    slots = torch.where(there, ids.long() * page + pos % page, -1)
    return dict(query_start=start.int(), seq_lens=(q + ctx).int(),
                positions=torch.where(there, pos, -1), slots=slots, table=table,
                next_head=(s["head"].long() + need.sum()).int())


def _plain_rope(s):
    case, total, page = s["case"], s["total"], s["page"]
    heads, kv, d, half = case["heads"], case["kv_heads"], case["head_dim"], case["rot"] // 2
    x = s["qkv"][:total].view(total, heads + 2 * kv, d)
    y = x[:, :heads + kv].float()
    c, sn = s["cos"][s["positions"][:total]][:, None], s["sin"][s["positions"][:total]][:, None]
    a, b = y[..., :half], y[..., half:2 * half]
    y = torch.cat((a * c - b * sn, b * c + a * sn, y[..., 2 * half:]), dim=-1).to(x.dtype)
    at, off = s["slots"][:total] // page, s["slots"][:total] % page
    s["k_cache"][at, :, off] = y[:, heads:]
    s["v_cache"][at, :, off] = x[:, heads + kv:]
    s["out"][:total] = y[:, :heads]
    return dict(q=s["out"], k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attention(s):
    q, table, start, seq = s["q"], s["table"], s["query_start"].long(), s["seq_lens"].long()
    heads, d = q.shape[1:]
    n_req, most, kv = seq.numel(), s["q_most"], s["k_cache"].shape[1]
    dev, group = q.device, heads // kv
    n_new = start[1:] - start[:-1]
    i = torch.arange(most, device=dev)
    rows = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)          # (requests, most)
    qp = q[rows].float() * s["scale"]
    qp = qp.view(n_req, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n_req, kv, -1, d)

    def keys(cache):  # every request's sequence out of its pages, (requests, kv, keys, d)
        g = cache[table.clamp(min=0).long()]
        return g.permute(0, 2, 1, 3, 4).reshape(n_req, kv, -1, d).float()

    x = torch.matmul(qp, keys(s["k_cache"]).transpose(2, 3))
    n_keys = x.shape[-1]
    x = x.view(n_req, kv, group, most, n_keys)
    key = torch.arange(n_keys, device=dev)
    pos = (seq - n_new)[:, None] + i                                  # (requests, most)
    seen = key <= pos[..., None]
    if s["window"]:
        seen &= (key > pos[..., None] - s["window"]) | (key < s["first"])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].float().view(1, kv, group, 1, 1)
        top = torch.maximum(top, sink)
    p = x.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    o = torch.matmul(p.view(n_req, kv, -1, n_keys), keys(s["v_cache"]))
    o = o.view(n_req, kv, group, most, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n_req, most, heads, d)
    return o[i < n_new[:, None]].to(q.dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if op == "plan":
        if not own:
            return _plain_plan(s)
        p = _bi().paged_plan(s["query_lens"], s["context_lens"], s["table"], s["page"],
                             s["tokens"], free_pages=s["free"], free_head=s["head"])
        return dict(query_start=p.query_start, seq_lens=p.seq_lens, positions=p.positions,
                    slots=p.slots, table=s["table"], next_head=p.next_head)
    if op == "rope":
        if not own:
            return _plain_rope(s)
        q = _bi().rope_kv_paged(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"],
                                s["k_cache"], s["v_cache"], out=s["out"])
        return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    if not own:
        return _plain_attention(s)
    return _bi().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["query_start"],
                                 s["seq_lens"], scale=s["scale"], window=s["window"],
                                 first_tokens=s["first"], sinks=s["sinks"])


# --------------------------------------------------------------------------- what it takes
def _visible(case, n_new, n_ctx):
    """(query, key) pairs of one request, and the keys that any of its queries sees."""
    window, first = case["window"], case["first"]
    if not window:
        return n_new * n_ctx + n_new * (n_new + 1) // 2, n_ctx + n_new
    pairs = 0
    for p in range(n_ctx, n_ctx + n_new):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + min(first, lo)
    lo = max(0, n_ctx - window + 1)
    return pairs, n_ctx + n_new - lo + min(first, lo)


def work(case):
    q, ctx = _lengths(case)
    n, total, page = len(q), sum(q), case["page"]
    touched = sum(_pages(a + b, page) - b // page for a, b in zip(q, ctx))
    if case["op"] == "plan":
        tokens = total + case["pad"]
        return {"bytes": 8 * n + 4 * (2 * n + 1) + 16 * tokens + 8 * touched + 8,
                "flops": 4 * tokens}
    size, heads, kv, d = _BYTES[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        return {"bytes": total * (2 * size * (heads + 2 * kv) * d + 4 * case["rot"] + 16),
                "flops": 3 * total * (heads + kv) * case["rot"]}
    seen = [_visible(case, a, b) for a, b in zip(q, ctx)]
    keys = sum(k for _, k in seen)
    return {"bytes": size * (2 * total * heads * d + 2 * keys * kv * d) + 4 * keys // page + 8 * n,
            "flops": 4 * d * heads * sum(p for p, _ in seen)}


# --------------------------------------------------------------------------- the exact values
def exact(case, seed):
    """In 64 bits, request by request from the definition; the plan's whole numbers have none."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    q_lens, ctx = _lengths(case)
    heads, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "rope":
        n, half = s["total"], case["rot"] // 2
        out, k, v = s["out"].double(), s["k_cache"].double(), s["v_cache"].double()
        x = s["qkv"][:n].double().view(n, heads + 2 * kv, d)
        # each pair (x_i, x_{i+half}) as a complex number, turned by its angle
        z = torch.complex(x[..., :half], x[..., half:2 * half])
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"][:n]]
        z = z * turn[:, None]
        y = x.clone()
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        out[:n] = y[:, :heads]
        for h in range(kv):
            k[s["slots"][:n] // page, h, s["slots"][:n] % page] = y[:, heads + h]
            v[s["slots"][:n] // page, h, s["slots"][:n] % page] = x[:, heads + kv + h]
        return dict(q=out, k_cache=k, v_cache=v)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group, row = heads // kv, 0
    for r, (n, c) in enumerate(zip(q_lens, ctx)):
        length = n + c
        pages = s["table"][r, :_pages(length, page)].long()
        pos = torch.arange(c, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | ((key <= pos - case["window"]) & (key >= case["first"]))
        for g in range(kv):
            k = s["k_cache"][pages, g].reshape(-1, d)[:length].double()
            v = s["v_cache"][pages, g].reshape(-1, d)[:length].double()
            for h in range(g * group, (g + 1) * group):
                a = s["q"][row:row + n, h].double() @ k.t() / math.sqrt(d)
                a[hidden] = -math.inf
                if s["sinks"] is not None:  # one more logit whose value is nothing
                    a = torch.cat((a, s["sinks"][h].double().expand(n, 1)), dim=1)
                w = torch.softmax(a, dim=1)[:, :length]
                out[row:row + n, h] = w @ v
        row += n
    return out
