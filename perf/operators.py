"""The paged key/value cache and its attention, as a serving program calls them.

Four operators: the block tables and slot maps of a step, built on the GPU from
the requests' lengths (`page_tables`); the write of the step's keys and values
into the cache (`paged_cache_update`); attention of the step's tokens, one or a
chunk per request, over the paged cache (`paged_attention`); and attention with
a sliding window and a few first tokens that stay visible over contiguous keys
(`window_attention`). Head counts, head dims and lengths are those of the
package's decoder, of its benchmark and of its tests.

With `own` false `run` computes them in elementary torch operations, in 32 bits
and rounded once; with `own` true it calls the package.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
HEADS = ((32, 8), (32, 8), (16, 8), (8, 8), (32, 4))


def _bi():
    path = os.path.abspath("mlx-batch-invariant_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mlx_batch_invariant

    return mlx_batch_invariant


# -------------------------------------------------------------------- cases
#
# Requests of a case: "reqs" requests of which "chunks" bring "chunk" new
# tokens and the others one; their cached lengths are spread over
# lo .. hi by the case's own "spread" number.


def listed():
    return [
        # One decode step of a serving batch: a token each, a new page now and then.
        dict(name="tables_decode", kind="tables", reqs=64, chunks=0, chunk=1, lo=1, hi=8000,
             page=16, width=512, pad=0, spread=1),
        # A large mixed step: chunks of prompts beside decodes, padded for a captured graph.
        dict(name="tables_mixed", kind="tables", reqs=500, chunks=30, chunk=2021, lo=0, hi=6000,
             page=16, width=512, pad=1000, spread=2),
        # Three users' next tokens into the cache: the smallest call.
        dict(name="update_decode", kind="update", reqs=3, chunks=0, chunk=1, lo=1, hi=4200,
             Hkv=8, D=128, page=16, order="phtd", pad=0, dtype="bf16", spread=3),
        # Prompt chunks into a token-major cache, keys and values being slices
        # of one projection's output, with padding rows behind the last.
        dict(name="update_chunks", kind="update", reqs=17, chunks=16, chunk=511, lo=0, hi=4000,
             Hkv=8, D=128, page=32, order="pthd", pad=15, dtype="f16", spread=4),
        # One user's next token over a long cache: one sequence, 32/8 heads.
        dict(name="paged_decode_b1", kind="paged", reqs=1, chunks=0, chunk=1, lo=8191, hi=8191,
             H=32, Hkv=8, D=128, page=16, order="phtd", window=0, first=0, sinks=False,
             dtype="bf16", spread=5),
        # A full serving batch at mixed lengths up to the same.
        dict(name="paged_decode_b64", kind="paged", reqs=64, chunks=0, chunk=1, lo=1000, hi=8191,
             H=32, Hkv=8, D=128, page=16, order="pthd", window=0, first=0, sinks=False,
             dtype="bf16", spread=6),
        # A few short requests in 32 bits, heads of 64, odd lengths, logit sinks.
        dict(name="paged_small_f32", kind="paged", reqs=5, chunks=2, chunk=7, lo=0, hi=333,
             H=8, Hkv=8, D=64, page=8, order="phtd", window=0, first=0, sinks=True,
             dtype="f32", spread=7),
        # Chunked prefill beside decodes: two chunks of 511 tokens, 30 decodes, windowed.
        dict(name="paged_mixed", kind="paged", reqs=32, chunks=2, chunk=511, lo=500, hi=4200,
             H=32, Hkv=8, D=128, page=64, order="phtd", window=2048, first=4, sinks=False,
             dtype="f16", spread=8),
        # The second half of an 8192-token prompt over the first.
        dict(name="paged_prefill", kind="paged", reqs=1, chunks=1, chunk=4096, lo=4096, hi=4096,
             H=32, Hkv=8, D=128, page=16, order="phtd", window=0, first=0, sinks=False,
             dtype="bf16", spread=9),
        # Next tokens under a window: 16 sequences of which each sees 1024 keys and 4 first ones.
        dict(name="window_decode", kind="window", B=16, H=32, Hkv=8, qL=1, N=8192, D=128,
             window=1024, first=4, sinks=False, dtype="bf16"),
        # A long prompt under the same window.
        dict(name="window_prompt", kind="window", B=1, H=32, Hkv=8, qL=8192, N=8192, D=128,
             window=1024, first=4, sinks=False, dtype="bf16"),
        # Odd sizes: three short prompts over cached keys, heads of 64, logit sinks.
        dict(name="window_odd", kind="window", B=3, H=16, Hkv=8, qL=77, N=333, D=64,
             window=100, first=3, sinks=True, dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("tables", "update", "decode", "chunk", "prefill", "window_decode",
                       "window_prompt"))
    spread = rng.randrange(1 << 20)
    page = rng.choice((8, 16, 16, 32, 64, 128, 256))
    if kind == "tables":
        reqs = _log_int(rng, 1, 500)
        chunks = rng.randint(0, min(reqs, 30))
        return dict(kind=kind, reqs=reqs, chunks=chunks, chunk=_log_int(rng, 1, 2021),
                    lo=0, hi=_log_int(rng, 1, 6000), page=page, width=-(-8192 // page),
                    pad=rng.choice((0, 0, _log_int(rng, 1, 1000))), spread=spread)
    H, Hkv = rng.choice(HEADS)
    D = rng.choice((128, 128, 128, 64, 256))
    dtype = rng.choice(("bf16", "bf16", "f16", "f16", "f32"))
    order = rng.choice(("phtd", "pthd"))
    if kind == "update":
        reqs = _log_int(rng, 1, 64)
        chunks = rng.randint(0, min(reqs, 16))
        return dict(kind=kind, reqs=reqs, chunks=chunks, chunk=_log_int(rng, 1, 511), lo=0,
                    hi=_log_int(rng, 1, 4000), Hkv=Hkv, D=D, page=page, order=order,
                    pad=rng.choice((0, 15)), dtype=dtype, spread=spread)
    window = rng.choice((0, 0, _log_int(rng, 16, 4096)))
    first = rng.choice((0, 4, rng.randint(1, 64))) if window else 0
    sinks = rng.random() < 0.2
    small = D > 128 or dtype == "f32"  # keeps the work within the listed cases'
    if kind in ("decode", "chunk"):
        reqs = _log_int(rng, 1, 16 if small else 64)
        chunks = 0 if kind == "decode" else rng.randint(1, min(reqs, 4))
        return dict(kind="paged", reqs=reqs, chunks=chunks,
                    chunk=1 if kind == "decode" else _log_int(rng, 2, 511), lo=0,
                    hi=_log_int(rng, 128, 4096 if chunks else 8191), H=H, Hkv=Hkv, D=D, page=page,
                    order=order, window=window, first=first, sinks=sinks, dtype=dtype,
                    spread=spread)
    if kind == "prefill":
        chunk = _log_int(rng, 64, 1024 if small else 4096)
        ctx = rng.choice((0, rng.randint(0, 1024 if small else 4096)))
        return dict(kind="paged", reqs=1, chunks=1, chunk=chunk, lo=ctx, hi=ctx, H=H, Hkv=Hkv,
                    D=D, page=page, order=order, window=window, first=first, sinks=sinks,
                    dtype=dtype, spread=spread)
    window = _log_int(rng, 16, 2048)
    first = rng.choice((0, 4, rng.randint(1, 64)))
    if kind == "window_decode":
        return dict(kind="window", B=_log_int(rng, 1, 16), H=H, Hkv=Hkv, qL=rng.choice((1, 1, 4)),
                    N=_log_int(rng, 64, 8192), D=D, window=window, first=first, sinks=sinks,
                    dtype=dtype)
    L = _log_int(rng, 64, 1024 if small else 8192)
    return dict(kind="window", B=_log_int(rng, 1, max(1, 2048 // L)), H=H, Hkv=Hkv, qL=L, N=L, D=D,
                window=window, first=first, sinks=sinks, dtype=dtype)


# ------------------------------------------------------------------- inputs


def _lengths(case):
    """(cached lengths, new lengths) of the case's requests, from the case alone."""
    rng = random.Random(case["spread"])
    n, cap = case["reqs"], 1 << 62
    new = [case["chunk"]] * case["chunks"] + [1] * (n - case["chunks"])
    if case["kind"] == "tables":
        cap = case["width"] * case["page"]
    ctx = [min(rng.randint(case["lo"], case["hi"]), cap - new[i]) for i in range(n)]
    order = list(range(n))
    rng.shuffle(order)
    return [ctx[i] for i in order], [new[i] for i in order]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(n, page):
    return -(-n // page)


def _cache(g, pages, Hkv, page, D, order, dtype):
    """(pages, Hkv, page, D) cache, stored head-major or token-major."""
    if order == "phtd":
        return _rn(g, (pages, Hkv, page, D), dtype)
    return _rn(g, (pages, page, Hkv, D), dtype).transpose(1, 2)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "window":
        dt = DTYPES[case["dtype"]]
        B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
        q = _rn(g, (B, case["qL"], H, D), dt).transpose(1, 2)
        k = _rn(g, (B, Hkv, case["N"], D), dt)
        v = _rn(g, (B, Hkv, case["N"], D), dt)
        return dict(case=case, q=q, k=k, v=v,
                    sinks=_rn(g, (H,), dt) if case["sinks"] else None)

    ctx, new = _lengths(case)
    page, R, T = case["page"], len(ctx), sum(new)
    qs = [0]
    for n in new:
        qs.append(qs[-1] + n)
    need = [_pages(c + n, page) for c, n in zip(ctx, new)]
    held = [_pages(c, page) for c in ctx] if case["kind"] == "tables" else need
    width = case["width"] if case["kind"] == "tables" else max(need)
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # Rows of the table: the pages a request holds, in the pool's random order.
    first, table = 0, torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    start = []
    for h in held:
        start.append(first)
        first += h
    cols = torch.arange(width, dtype=torch.int32, device="cuda")[None]
    idx = _i32(start)[:, None] + cols
    table = torch.where(cols < _i32(held)[:, None], order[idx.clamp(max=pages - 1).long()], table)
    state = dict(case=case, table=table, ctx=_i32(ctx), new=_i32(new), qs=_i32(qs), tokens=T,
                 seq=_i32([c + n for c, n in zip(ctx, new)]), host_qs=qs,
                 host_seq=[c + n for c, n in zip(ctx, new)],
                 max_query=max(new), max_seq=max(c + n for c, n in zip(ctx, new)))
    if case["kind"] == "tables":
        state["free"] = order[first:].contiguous()
        return state

    dt, Hkv, D = DTYPES[case["dtype"]], case["Hkv"], case["D"]
    state["k_cache"] = _cache(g, pages, Hkv, page, D, case["order"], dt)
    state["v_cache"] = _cache(g, pages, Hkv, page, D, case["order"], dt)
    if case["kind"] == "update":
        # The projection's output holds keys and values of a token side by side.
        kv = _rn(g, (T + case["pad"], 2, Hkv, D), dt)
        state["k"], state["v"] = kv[:, 0], kv[:, 1]
        r = torch.repeat_interleave(torch.arange(R, device="cuda"), _i32(new).long())
        pos = _i32(ctx)[r] + torch.arange(T, device="cuda", dtype=torch.int32) - _i32(qs)[r]
        slots = table[r, (pos // page).long()] * page + pos % page
        state["slots"] = torch.cat([slots, torch.full((case["pad"],), -1, dtype=torch.int32,
                                                      device="cuda")])
        return state
    state["q"] = _rn(g, (T, case["H"], D), dt)
    state["sinks"] = _rn(g, (case["H"],), dt) if case["sinks"] else None
    return state


# -------------------------------------------------------------- plain forms


def _plain_tables(s):
    c = s["case"]
    page, W = c["page"], c["width"]
    table, ctx, new, free = s["table"], s["ctx"].long(), s["new"].long(), s["free"]
    T = s["tokens"] + c["pad"]
    have = ((ctx + page - 1) // page).clamp(max=W)
    end = ((ctx + new + page - 1) // page).clamp(max=W)
    take = end - have
    first = torch.cumsum(take, 0) - take
    cols = torch.arange(W, device="cuda")[None]
    idx = first[:, None] + cols - have[:, None]
    fresh = (cols >= have[:, None]) & (cols < end[:, None])
    F = free.shape[0]
    got = torch.where(idx < F, free[idx.clamp(0, max(F - 1, 0))], -1) if F else torch.full_like(
        table, -1)
    table.copy_(torch.where(fresh, got.to(torch.int32), table))
    stop = torch.cumsum(new, 0)
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(stop, t, right=True).clamp(max=len(ctx) - 1)
    inside = t < stop[-1]
    pos = ctx[r] + t - (stop - new)[r]
    pg = torch.where(pos < W * page, table[r, (pos // page).clamp(max=W - 1)].long(), -1)
    slots = torch.where(inside & (pg >= 0), pg * page + pos % page, -1).to(torch.int32)
    positions = torch.where(inside, pos, -1).to(torch.int32)
    qs = torch.cat([torch.zeros(1, dtype=stop.dtype, device="cuda"), stop]).to(torch.int32)
    return dict(block_tables=table, slots=slots, positions=positions, query_start=qs,
                seq_lens=(ctx + new).to(torch.int32), pages_used=take.sum().to(torch.int32))


def _plain_update(s):
    page, T = s["case"]["page"], s["tokens"]
    slots = s["slots"][:T].long()  # the rows behind the last request have no slot
    s["k_cache"][slots // page, :, slots % page] = s["k"][:T]
    s["v_cache"][slots // page, :, slots % page] = s["v"][:T]
    return [s["k_cache"], s["v_cache"]]


def _plain_rows(q, k, v, pos0, window, first, scale, sinks):
    """Rows at positions pos0 ... of one sequence: q (Hkv, G, L, D), k and v
    (Hkv, N, D), all fp32; sinks (Hkv, G) or None. Returns (Hkv, G, L, D)."""
    Hkv, G, L, D = q.shape
    pos = pos0 + torch.arange(L, device=q.device)[:, None]
    key = torch.arange(k.shape[1], device=q.device)[None]
    see = key <= pos
    if window:
        see = see & ((key > pos - window) | (key < first))
    kt = k.transpose(1, 2).contiguous()
    s = torch.matmul(q.reshape(Hkv, G * L, D), kt).reshape(Hkv, G, L, -1) * scale
    s = s.masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks[:, :, None, None])
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    d = p.sum(-1, keepdim=True)
    if sinks is not None:
        d = d + torch.exp(sinks[:, :, None, None] - m)
    o = torch.matmul(p.reshape(Hkv, G * L, -1), v).reshape(Hkv, G, L, -1)
    return torch.where(d > 0, o / d, torch.zeros_like(o))


def _attend(case, q, k, v, pos0, sinks, dtype):
    """q (L, H, D), k and v (Hkv, N, D) of one sequence -> (L, H, D) in `dtype`;
    1024 rows at a time."""
    L, H, D = q.shape
    Hkv = k.shape[0]
    kf, vf = k.to(dtype), v.to(dtype)
    sk = None if sinks is None else sinks.to(dtype).reshape(Hkv, H // Hkv)
    out = []
    for a in range(0, L, 1024):
        qa = q[a:a + 1024].to(dtype)
        n = qa.shape[0]
        qa = qa.reshape(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3)
        hi = pos0 + a + n  # keys that some of these rows see
        o = _plain_rows(qa, kf[:, :hi], vf[:, :hi], pos0 + a, case["window"], case["first"],
                 1.0 / math.sqrt(D), sk)
        out.append(o.permute(2, 0, 1, 3).reshape(n, H, -1))
    return torch.cat(out)


def _sequence(s, cache, r):
    """Keys or values 0 .. n - 1 of request r, (Hkv, n, D)."""
    page, n = s["case"]["page"], s["host_seq"][r]
    pages = cache[s["table"][r, :_pages(n, page)].long()]  # (p, Hkv, page, D)
    Hkv, D = pages.shape[1], pages.shape[3]
    return pages.permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n]


def _paged(s, dtype):
    qs, out = s["host_qs"], []
    for r, n in enumerate(s["host_seq"]):
        q = s["q"][qs[r]:qs[r + 1]]
        out.append(_attend(s["case"], q, _sequence(s, s["k_cache"], r),
                           _sequence(s, s["v_cache"], r), n - q.shape[0], s["sinks"], dtype))
    return torch.cat(out)


def _window(s, dtype):
    c = s["case"]
    return torch.stack([
        _attend(c, s["q"][b].transpose(0, 1), s["k"][b], s["v"][b], c["N"] - c["qL"], s["sinks"],
                dtype).transpose(0, 1) for b in range(c["B"])])


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        if kind == "tables":
            return _plain_tables(state)
        if kind == "update":
            return _plain_update(state)
        dt = DTYPES[c["dtype"]]
        return (_paged if kind == "paged" else _window)(state, torch.float32).to(dt)
    bi = _bi()
    if kind == "tables":
        return bi.page_tables(state["table"], state["ctx"], state["new"], state["free"],
                              c["page"], state["tokens"] + c["pad"])._asdict()
    if kind == "update":
        bi.paged_cache_update(state["k"], state["v"], state["k_cache"], state["v_cache"],
                              state["slots"])
        return [state["k_cache"], state["v_cache"]]
    window = c["window"] or None
    if kind == "paged":
        return bi.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"],
                                  state["qs"], state["seq"],
                                  max_query=state["max_query"], max_seq=state["max_seq"],
                                  window=window, sink_tokens=c["first"],
                                  sinks=state["sinks"])
    return bi.window_attention(state["q"], state["k"], state["v"], window,
                               sink_tokens=c["first"], sinks=state["sinks"])


# --------------------------------------------------------------------- work


def _seen(n, L, window, first):
    """(pairs, keys) that the last L rows of a sequence of n see."""
    pairs = keys = 0
    for p in range(n - L, n):
        see = p + 1
        if window and see > window:
            see = window + min(first, see - window)
        pairs += see
    lo = n - L + 1  # keys the first row sees, and all behind them
    keys = n if not window or lo <= window else n - (lo - window) + min(first, lo - window)
    return pairs, keys


def work(case):
    if case["kind"] == "tables":
        ctx, new = _lengths(case)
        page = case["page"]
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(ctx, new))
        T = sum(new) + case["pad"]
        return dict(bytes=4 * (2 * len(ctx) + 2 * fresh + 2 * T + 2 * len(ctx) + 2), flops=4 * T)
    if case["kind"] == "update":
        T = sum(_lengths(case)[1])
        return dict(bytes=4 * T * case["Hkv"] * case["D"] * BYTES[case["dtype"]] + 4 * T, flops=0)
    E, H, Hkv, D = BYTES[case["dtype"]], case["H"], case["Hkv"], case["D"]
    if case["kind"] == "paged":
        seqs = [(c + n, n) for c, n in zip(*_lengths(case))]
    else:
        seqs = [(case["N"], case["qL"])] * case["B"]
    rows = sum(n for _, n in seqs)
    seen = [_seen(n, L, case["window"], case["first"]) for n, L in seqs]
    table = 4 * sum(_pages(k, case["page"]) for _, k in seen) if case["kind"] == "paged" else 0
    return dict(bytes=2 * rows * H * D * E + 2 * sum(k for _, k in seen) * Hkv * D * E + table,
                flops=4 * D * H * sum(p for p, _ in seen))


# -------------------------------------------------------------------- exact


def _exact_sequence(q, k, v, window, first, sinks):
    """The definition for one sequence in float64: q (L, H, D) are its last L
    tokens, k and v (N, Hkv, D) its keys and values, sinks (H,) or None."""
    L, H, D = q.shape
    N, Hkv = k.shape[:2]
    out = torch.empty((L, H, D), dtype=torch.float64, device="cuda")
    keys = torch.arange(N, device="cuda")
    step = max(1, (1 << 26) // N)
    for h in range(H):
        kh = k[:, h * Hkv // H].double().t().contiguous()
        vh = v[:, h * Hkv // H].double().contiguous()
        for a in range(0, L, step):
            at = torch.arange(N - L + a, min(N - L + a + step, N), device="cuda")[:, None]
            hidden = keys > at
            if window:
                hidden |= (keys <= at - window) & (keys >= first)
            z = torch.matmul(q[a:a + step, h].double(), kh) / math.sqrt(D)
            z[hidden] = -math.inf
            if sinks is not None:  # one more term of the denominator
                z = torch.cat([z, sinks[h].double().expand(z.shape[0], 1)], 1)
            e = torch.exp(z - z.max(1, keepdim=True).values)
            out[a:a + step, h] = torch.matmul(e[:, :N].contiguous(), vh) / e.sum(1, keepdim=True)
    return out


def exact(case, seed):
    if case["kind"] == "tables":  # whole numbers throughout
        return None
    s = prepare(case, seed)
    if case["kind"] == "window":
        return torch.stack([
            _exact_sequence(s["q"][b].transpose(0, 1), s["k"][b].transpose(0, 1),
                            s["v"][b].transpose(0, 1), case["window"], case["first"],
                            s["sinks"]).transpose(0, 1) for b in range(case["B"])])
    page, out = case["page"], []
    if case["kind"] == "update":  # row by row of the slots that there are
        at = s["slots"].long()
        at = at[at >= 0]
        for name in ("k", "v"):
            pool = s[name + "_cache"].double().transpose(1, 2).contiguous()
            pool.view(-1, *pool.shape[2:]).index_copy_(0, at, s[name][:len(at)].double())
            out.append(pool.transpose(1, 2))
        return out
    kc, vc = s["k_cache"].transpose(1, 2), s["v_cache"].transpose(1, 2)  # (p, page, Hkv, D)
    for r, n in enumerate(s["host_seq"]):
        at = torch.arange(n, device="cuda")
        p, o = s["table"][r].long()[at // page], at % page
        out.append(_exact_sequence(s["q"][s["host_qs"][r]:s["host_qs"][r + 1]], kc[p, o], vc[p, o],
                                   case["window"], case["first"], s["sinks"]))
    return torch.cat(out)
