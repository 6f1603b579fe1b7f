"""Serving over a cache of 8 bits, as a serving program calls it, from the
projections to the tokens' probabilities.

Five operators: rotary positions of queries and keys (`rotary`); the write of
the step's keys and values into pages of 8-bit codes with a scale for every
token and head (`paged_cache_update` with scales); the way back to values
(`paged_cache_read`); attention of the step's tokens, one or a chunk per
request, over such pages (`paged_attention` with scales); and what a program
asks of the logits (`token_logprobs`: log probabilities of given tokens, the
entropy, the likeliest alternatives). Head counts, head dims, lengths and the
vocabulary are those of the package's decoder, of its benchmark and of its
tests.

With `own` false `run` computes them in elementary torch operations, in 32 bits
(angles and quotients in 64) and rounded once; with `own` true it calls the
package.
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
# Requests of a case over the cache: "reqs" requests of which "chunks" bring
# "chunk" new tokens and the others one; their cached lengths are spread over
# lo .. hi by the case's own "spread" number.


def listed():
    return [
        # One decode step of a serving batch: 64 tokens at their own positions.
        dict(name="rotary_decode", kind="rotary", T=64, H=32, Hkv=8, D=128, rot=128, offset=0,
             inter=False, stretch=1.0, far=8191, run=False, dtype="bf16"),
        # A long prompt's chunk far out, with frequencies and scale for a context
        # stretched fourfold; adjacent pairs, and only half of each head.
        dict(name="rotary_prompt", kind="rotary", T=8161, H=32, Hkv=8, D=128, rot=64, offset=64,
             inter=True, stretch=4.0, far=120000, run=True, dtype="f16"),
        # Three users' next tokens into the cache, and read back: the smallest call.
        dict(name="update_decode", kind="update", reqs=3, chunks=0, chunk=1, lo=1, hi=4200,
             Hkv=8, D=128, V=128, page=16, order="phtd", pad=0, dtype="bf16", spread=3),
        # Prompt chunks into a token-major cache, keys and values being slices of
        # one projection's output, with padding rows behind the last.
        dict(name="update_chunks", kind="update", reqs=17, chunks=16, chunk=511, lo=0, hi=4000,
             Hkv=8, D=128, V=128, page=32, order="pthd", pad=15, dtype="bf16", spread=4),
        # A short request's rows, in 32 bits, to compare with: heads of 64, odd length.
        dict(name="read_short", kind="read", reqs=1, chunks=0, chunk=1, lo=332, hi=332, Hkv=8,
             D=64, V=64, page=8, order="phtd", dtype="f32", spread=5),
        # A prompt that requests share, taken out of the cache as values.
        dict(name="read_prompt", kind="read", reqs=2, chunks=0, chunk=1, lo=4000, hi=8190, Hkv=8,
             D=128, V=128, page=16, order="phtd", dtype="bf16", spread=6),
        # One user's next token over a long cache: one sequence, 32/8 heads.
        dict(name="decode_b1", kind="paged", reqs=1, chunks=0, chunk=1, lo=8191, hi=8191, H=32,
             Hkv=8, D=128, V=128, page=16, order="phtd", window=0, first=0, sinks=False,
             dtype="bf16", spread=7),
        # A full serving batch at mixed lengths up to the same.
        dict(name="decode_b64", kind="paged", reqs=64, chunks=0, chunk=1, lo=1000, hi=8191, H=32,
             Hkv=8, D=128, V=128, page=16, order="pthd", window=0, first=0, sinks=False,
             dtype="bf16", spread=8),
        # Chunked prefill beside decodes under a window with first tokens and logit
        # sinks: two chunks of 511 tokens, 14 single ones, in f16.
        dict(name="mixed_window", kind="paged", reqs=16, chunks=2, chunk=511, lo=500, hi=4200,
             H=32, Hkv=8, D=128, V=128, page=64, order="phtd", window=2048, first=4, sinks=True,
             dtype="f16", spread=9),
        # The second half of an 8192-token prompt over the first.
        dict(name="prefill", kind="paged", reqs=1, chunks=1, chunk=4096, lo=4096, hi=4096, H=32,
             Hkv=8, D=128, V=128, page=16, order="phtd", window=0, first=0, sinks=False,
             dtype="bf16", spread=10),
        # The tokens a decode step has drawn for three users, with five alternatives
        # each, where most of the vocabulary is ruled out.
        dict(name="logprobs_decode", kind="logprobs", rows=3, vocab=32000, top=5, ruled_out=0.9,
             dtype="f32"),
        # A prompt's tokens scored, with the twenty likeliest of each place.
        dict(name="logprobs_prompt", kind="logprobs", rows=2021, vocab=32000, top=20,
             ruled_out=0.0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "update", "read", "decode", "decode", "chunk", "prefill",
                       "logprobs"))
    spread = rng.randrange(1 << 20)
    H, Hkv = rng.choice(HEADS)
    D, V = rng.choice(((128, 128), (128, 128), (64, 64), (96, 96), (192, 128), (192, 192),
                       (256, 256)))
    if kind == "logprobs":
        vocab = _log_int(rng, 259, 65000)
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(2021, 32000 * 1000 // vocab))),
                    vocab=vocab, top=rng.choice((0, 1, 5, 20, rng.randint(1, 32))),
                    ruled_out=rng.choice((0.0, 0.0, round(rng.random(), 2))),
                    dtype=rng.choice(("bf16", "f16", "f32")))
    if kind == "rotary":
        rot = rng.choice((D, D, D // 2, 2 * rng.randint(1, D // 2)))
        return dict(kind=kind, T=_log_int(rng, 1, 4000), H=H, Hkv=Hkv, D=D, rot=rot,
                    offset=rng.choice((0, D - rot)), inter=rng.random() < 0.5,
                    stretch=rng.choice((1.0, 1.0, round(rng.uniform(1.0, 16.0), 2))),
                    far=_log_int(rng, 1, 1000000), run=rng.random() < 0.5,
                    dtype=rng.choice(("bf16", "f16", "f32")))
    page = rng.choice((8, 16, 16, 32, 64, 128, 256))
    order = rng.choice(("phtd", "pthd"))
    if kind in ("update", "read"):
        reqs = _log_int(rng, 1, 64 if kind == "update" else 4)
        chunks = rng.randint(0, min(reqs, 8))
        case = dict(kind=kind, reqs=reqs, chunks=chunks, chunk=_log_int(rng, 1, 511), lo=0,
                    hi=_log_int(rng, 1, 4000), Hkv=Hkv, D=D, V=V, page=page, order=order,
                    dtype=rng.choice(("bf16", "f16", "f32")), spread=spread)
        return dict(case, pad=rng.choice((0, 15))) if kind == "update" else case
    window = rng.choice((0, 0, _log_int(rng, 16, 4096)))
    first = rng.choice((0, 4, rng.randint(1, 64))) if window else 0
    case = dict(kind="paged", H=H, Hkv=Hkv, D=D, V=V, page=page, order=order, window=window,
                first=first, sinks=rng.random() < 0.2, dtype=rng.choice(("bf16", "f16")),
                spread=spread)
    small = D > 128  # keeps the work within the listed cases'
    if kind == "prefill":
        ctx = rng.choice((0, rng.randint(0, 1024 if small else 4096)))
        return dict(case, reqs=1, chunks=1, chunk=_log_int(rng, 64, 1024 if small else 4096),
                    lo=ctx, hi=ctx)
    reqs = _log_int(rng, 1, 32 if small else 64)
    chunks = 0 if kind == "decode" else rng.randint(1, min(reqs, 2))
    return dict(case, reqs=reqs, chunks=chunks,
                chunk=1 if kind == "decode" else _log_int(rng, 2, 511), lo=0,
                hi=_log_int(rng, 128, 4096 if chunks or small else 8191))


# ------------------------------------------------------------------- inputs


def _lengths(case):
    """(cached lengths, new lengths) of the case's requests, from the case alone."""
    rng = random.Random(case["spread"])
    n = case["reqs"]
    new = [case["chunk"]] * case["chunks"] + [1] * (n - case["chunks"])
    ctx = [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
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


def _frequencies(rot, stretch):
    """Radians per token of every pair, (rot / 2,) float64: base 10000; a context
    stretched beyond 2048 tokens keeps the pairs that turn more than 32 times in
    these, divides those that turn less than once, and blends between."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    if stretch == 1.0:
        return f
    keep = ((2048 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return f * (keep + (1 - keep) / stretch)


def _codes(g, rows, heads, dim, order, page):
    """A pool of codes (rows / page, heads, page, dim) and its scales, as rows of
    normal values with a few large ones leave them; head-major or token-major."""
    shape = (rows // page, heads, page, dim) if order == "phtd" else (rows // page, page, heads, dim)
    code = (torch.randn(shape, generator=g, device="cuda") * 40).clamp_(-127, 127).round_()
    code = code.to(torch.int8)
    scale = torch.exp(_rn(g, shape[:3], torch.float32, 0.3)) / 40
    if order == "phtd":
        return code, scale
    return code.transpose(1, 2), scale.transpose(1, 2)


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "logprobs":
        logits = _rn(g, (case["rows"], case["vocab"]), dt, 2.5)
        if case["ruled_out"]:
            out = torch.rand(logits.shape, generator=g, device="cuda") < case["ruled_out"]
            out[:, 0] = False
            logits = logits.masked_fill(out, float("-inf"))
        # The drawn tokens: likely ones, by the largest of noisy logits.
        noise = -torch.log(-torch.log(torch.rand(logits.shape, generator=g, device="cuda")))
        return dict(case=case, logits=logits, tokens=(logits.float() + noise).argmax(-1))
    if kind == "rotary":
        T, H, Hkv, D = case["T"], case["H"], case["Hkv"], case["D"]
        qkv = _rn(g, (T, H + 2 * Hkv, D), dt)  # one projection's output
        if case["run"]:
            at = torch.arange(T, device="cuda") + int(torch.randint(0, case["far"], (), generator=g,
                                                                    device="cuda"))
        else:
            at = torch.randint(0, case["far"] + 1, (T,), generator=g, device="cuda")
        return dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + Hkv], positions=at.to(torch.int32),
                    inv_freq=_frequencies(case["rot"], case["stretch"]),
                    scale=1.0 + 0.1 * math.log(case["stretch"]))

    ctx, new = _lengths(case)
    page, R, T = case["page"], len(ctx), sum(new)
    qs = [0]
    for n in new:
        qs.append(qs[-1] + n)
    seq = [c + n for c, n in zip(ctx, new)]
    need = [_pages(n, page) for n in seq]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # Rows of the table: the pages a request holds, in the pool's random order.
    start = torch.cumsum(_i32(need), 0) - _i32(need)
    cols = torch.arange(max(need), dtype=torch.int32, device="cuda")[None]
    table = torch.where(cols < _i32(need)[:, None],
                        order[(start[:, None] + cols).clamp(max=pages - 1)], -1).to(torch.int32)
    Hkv, D, V = case["Hkv"], case["D"], case["V"]
    kc, ks = _codes(g, pages * page, Hkv, D, case["order"], page)
    vc, vs = _codes(g, pages * page, Hkv, V, case["order"], page)
    state = dict(case=case, table=table, seq=_i32(seq), qs=_i32(qs), host_qs=qs, host_seq=seq,
                 host_new=new, max_query=max(new), max_seq=max(seq), k_cache=kc, v_cache=vc,
                 k_scales=ks, v_scales=vs)
    if kind == "paged":
        state["q"] = _rn(g, (T, case["H"], D), dt)
        state["sinks"] = _rn(g, (case["H"],), dt) if case["sinks"] else None
        return state
    # Slots of the new tokens (update) or of all rows of the requests (read).
    count, base = (_i32(new), _i32(ctx)) if kind == "update" else (_i32(seq), _i32([0] * R))
    r = torch.repeat_interleave(torch.arange(R, device="cuda"), count.long())
    before = torch.cumsum(count, 0) - count
    pos = base[r] + torch.arange(len(r), device="cuda") - before[r]
    slots = (table[r, pos // page] * page + pos % page).to(torch.int32)
    if kind == "update":
        slots = torch.cat([slots, torch.full((case["pad"],), -1, dtype=torch.int32,
                                             device="cuda")])
        # The projection's output holds keys and values of a token side by side.
        kv = _rn(g, (T + case["pad"], Hkv * (D + V)), dt)
        state["k"] = kv[:, :Hkv * D].view(-1, Hkv, D)
        state["v"] = kv[:, Hkv * D:].view(-1, Hkv, V)
    state["slots"] = slots
    return state


# -------------------------------------------------------------- plain forms


def _plain_rotary(s):
    c = s["case"]
    n, o = c["rot"] // 2, c["offset"]
    turn = s["positions"].double()[:, None] * s["inv_freq"]
    cos = (torch.cos(turn) * s["scale"]).float()[:, None]
    sin = (torch.sin(turn) * s["scale"]).float()[:, None]
    first = slice(o, o + 2 * n, 2) if c["inter"] else slice(o, o + n)
    second = slice(o + 1, o + 2 * n, 2) if c["inter"] else slice(o + n, o + 2 * n)

    def turned(x):
        y = x.float()
        a, b = y[..., first], y[..., second]
        out = y.clone()
        out[..., first] = a * cos - b * sin
        out[..., second] = a * sin + b * cos
        return out.to(x.dtype)

    return [turned(s["q"]), turned(s["k"])]


def _plain_codes(x):
    """Codes of 8 bits and the scale of every row: the scale is a number of 32
    bits, the quotient is rounded once, to the nearest whole number."""
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float()
    by = scale.double()[..., None]
    code = torch.where(by > 0, (x / by).round().clamp(-127, 127), torch.zeros_like(x))
    return code.to(torch.int8), scale


def _plain_read(s, slots, dtype):
    page = s["case"]["page"]
    p, o = torch.div(slots, page, rounding_mode="floor").clamp(min=0).long(), (slots % page).long()
    there = (slots >= 0)[:, None, None]
    k = s["k_cache"][p, :, o].float() * s["k_scales"][p, :, o][..., None]
    v = s["v_cache"][p, :, o].float() * s["v_scales"][p, :, o][..., None]
    return [torch.where(there, x, 0.0).to(dtype) for x in (k, v)]


def _plain_update(s):
    page, T = s["case"]["page"], s["host_qs"][-1]
    slots = s["slots"][:T].long()  # the rows behind the last request have no slot
    p, o = slots // page, slots % page
    s["k_cache"][p, :, o], s["k_scales"][p, :, o] = _plain_codes(s["k"][:T])
    s["v_cache"][p, :, o], s["v_scales"][p, :, o] = _plain_codes(s["v"][:T])
    return _plain_read(s, s["slots"], s["k"].dtype)


def _rows_of(s, req, n, cache, scales):
    """Rows 0 .. n - 1 of the requests `req` as values, (len(req), Hkv, n, D)."""
    page = s["case"]["page"]
    at = torch.arange(n, device="cuda")
    p = s["table"][req][:, at // page].clamp(min=0).long()
    o = (at % page)[None].expand_as(p)
    return (cache[p, :, o].float() * scales[p, :, o][..., None]).transpose(1, 2).contiguous()


def _plain_attend(c, q, k, v, pos, seq, sinks):
    """Queries (R, L, H, D) at positions pos (R, L) over rows (R, Hkv, n, D) of
    requests of seq (R,) rows, in 32 bits: (R, L, H, V)."""
    R, L, H, D = q.shape
    Hkv, n = k.shape[1:3]
    key = torch.arange(n, device="cuda")
    see = (key <= pos[..., None]) & (key < seq[:, None, None])
    if c["window"]:
        see = see & ((key > pos[..., None] - c["window"]) | (key < c["first"]))
    see = see[:, None, None].expand(R, Hkv, H // Hkv, L, n).reshape(R, Hkv, -1, n)
    qt = q.float().reshape(R, L, Hkv, H // Hkv, D).permute(0, 2, 4, 3, 1).reshape(R, Hkv, D, -1)
    z = torch.matmul(k, qt.contiguous()).transpose(2, 3) / math.sqrt(D)  # (R, Hkv, G L, n)
    z = z.masked_fill(~see, float("-inf"))
    m = z.amax(-1, keepdim=True)
    if sinks is not None:
        sk = sinks.float().reshape(Hkv, -1, 1).expand(Hkv, H // Hkv, L).reshape(1, Hkv, -1, 1)
        m = torch.maximum(m, sk)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp(z - m)
    d = e.sum(-1, keepdim=True)
    if sinks is not None:
        d = d + torch.exp(sk - m)
    o = torch.matmul(e, v)
    o = torch.where(d > 0, o / d, torch.zeros_like(o))
    return o.reshape(R, Hkv, H // Hkv, L, -1).permute(0, 3, 1, 2, 4).reshape(R, L, H, -1)


def _plain_paged(s):
    c = s["case"]
    out = torch.empty((s["q"].shape[0], c["H"], c["V"]), dtype=torch.float32, device="cuda")
    single = [r for r, n in enumerate(s["host_new"]) if n == 1]
    if single:  # all single tokens side by side
        req = torch.tensor(single, device="cuda")
        n = max(s["host_seq"][r] for r in single)
        at, seq = s["qs"][req].long(), s["seq"][req]
        out[at] = _plain_attend(c, s["q"][at][:, None],
                                _rows_of(s, req, n, s["k_cache"], s["k_scales"]),
                                _rows_of(s, req, n, s["v_cache"], s["v_scales"]),
                                seq[:, None] - 1, seq, s["sinks"])[:, 0]
    for r, L in enumerate(s["host_new"]):  # a chunk's rows, 1024 at a time
        if L == 1:
            continue
        req, n, a = torch.tensor([r], device="cuda"), s["host_seq"][r], s["host_qs"][r]
        k = _rows_of(s, req, n, s["k_cache"], s["k_scales"])
        v = _rows_of(s, req, n, s["v_cache"], s["v_scales"])
        for b in range(0, L, 1024):
            e = min(L, b + 1024)
            hi = n - L + e  # rows that some of these see
            pos = torch.arange(n - L + b, hi, device="cuda")[None]
            out[a + b:a + e] = _plain_attend(c, s["q"][None, a + b:a + e], k[:, :, :hi],
                                             v[:, :, :hi], pos, s["seq"][req], s["sinks"])[0]
    return out.to(s["q"].dtype)


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lp = x - m - torch.log(z)
    own_lp = lp.gather(-1, s["tokens"][:, None])[:, 0]
    p = e / z
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    # The largest, ties to the lowest id: by one whole number of value and id.
    bits = x.contiguous().view(torch.int32).long()
    rank = torch.where(bits < 0, -2147483648 - bits, bits)  # in the values' order
    ids = torch.arange(x.shape[-1], device="cuda")
    best = torch.topk(rank * (1 << 20) - ids, top, -1).values
    best = (-best) % (1 << 20)
    return dict(logprobs=own_lp, entropy=entropy, top_ids=best, top_logprobs=lp.gather(-1, best))


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        if kind == "rotary":
            return _plain_rotary(state)
        if kind == "update":
            return _plain_update(state) + [state["k_scales"], state["v_scales"]]
        if kind == "read":
            return _plain_read(state, state["slots"], DTYPES[c["dtype"]])
        return _plain_paged(state) if kind == "paged" else _plain_logprobs(state)
    bi = _bi()
    if kind == "rotary":
        return list(bi.rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                              interleaved=c["inter"], offset=c["offset"], scale=state["scale"]))
    if kind == "logprobs":
        return bi.token_logprobs(state["logits"], state["tokens"], top=c["top"])._asdict()
    kc, vc, ks, vs = (state[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales"))
    if kind == "paged":
        return bi.paged_attention(state["q"], kc, vc, state["table"], state["qs"], state["seq"],
                                  max_query=state["max_query"], max_seq=state["max_seq"],
                                  window=c["window"] or None, sink_tokens=c["first"],
                                  sinks=state["sinks"], k_scales=ks, v_scales=vs)
    if kind == "update":
        bi.paged_cache_update(state["k"], state["v"], kc, vc, state["slots"], k_scales=ks,
                              v_scales=vs)
    back = bi.paged_cache_read(kc, vc, state["slots"], k_scales=ks, v_scales=vs,
                               dtype=DTYPES[c["dtype"]])
    return list(back) + ([ks, vs] if kind == "update" else [])


# --------------------------------------------------------------------- work


def _seen(n, L, window, first):
    """(pairs, keys) that the last L rows of a sequence of n see."""
    pairs = 0
    for p in range(n - L, n):
        see = p + 1
        if window and see > window:
            see = window + min(first, see - window)
        pairs += see
    lo = n - L + 1  # keys the first row sees, and all behind them
    keys = n if not window or lo <= window else n - (lo - window) + min(first, lo - window)
    return pairs, keys


def work(case):
    E = BYTES[case["dtype"]]
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * E + case["rows"] * (16 + 12 * case["top"]), flops=6 * n)
    if case["kind"] == "rotary":
        n = case["T"] * (case["H"] + case["Hkv"])
        return dict(bytes=2 * n * case["D"] * E + 4 * case["T"] + 4 * case["rot"],
                    flops=3 * n * case["rot"])
    ctx, new = _lengths(case)
    Hkv, dims = case["Hkv"], case["D"] + case["V"]
    if case["kind"] == "update":  # into codes, and back
        T = sum(new)
        return dict(bytes=T * Hkv * (dims * (2 * E + 1) + 8) + 4 * T, flops=4 * T * Hkv * dims)
    if case["kind"] == "read":
        T = sum(ctx) + sum(new)
        return dict(bytes=T * Hkv * (dims * (E + 1) + 8) + 4 * T, flops=T * Hkv * dims)
    seen = [_seen(c + n, n, case["window"], case["first"]) for c, n in zip(ctx, new)]
    keys = sum(k for _, k in seen)
    table = 4 * sum(_pages(k, case["page"]) for _, k in seen)
    return dict(bytes=sum(new) * case["H"] * dims * E + keys * Hkv * (dims + 8) + table,
                flops=2 * dims * case["H"] * sum(p for p, _ in seen))


# -------------------------------------------------------------------- exact


def _exact_rotary(s):
    c, out = s["case"], []
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["inv_freq"]))[:, None]
    for x in (s["q"], s["k"]):
        y = x.double()
        part = y[..., c["offset"]:c["offset"] + c["rot"]]
        pair = part.unflatten(-1, (-1, 2)) if c["inter"] else part.unflatten(-1, (2, -1)).mT
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if c["inter"] else z.mT.flatten(-2)
        out.append(torch.cat([y[..., :c["offset"]], z, y[..., c["offset"] + c["rot"]:]], -1))
    return out


def _exact_sequence(q, k, v, window, first, sinks):
    """The definition for one sequence in float64: q (L, H, D) are its last L
    tokens, k and v (n, Hkv, ...) its keys and values, sinks (H,) or None."""
    L, H, D = q.shape
    n, Hkv, V = v.shape
    out = torch.empty((L, H, V), dtype=torch.float64, device="cuda")
    keys = torch.arange(n, device="cuda")
    step = max(1, (1 << 26) // n)
    for h in range(H):
        kh = k[:, h * Hkv // H].t().contiguous()
        vh = v[:, h * Hkv // H].contiguous()
        for a in range(0, L, step):
            at = torch.arange(n - L + a, min(n - L + a + step, n), device="cuda")[:, None]
            hidden = keys > at
            if window:
                hidden |= (keys <= at - window) & (keys >= first)
            z = torch.matmul(q[a:a + step, h].double(), kh) / math.sqrt(D)
            z[hidden] = -math.inf
            if sinks is not None:  # one more term of the denominator
                z = torch.cat([z, sinks[h].double().expand(z.shape[0], 1)], 1)
            w = torch.exp(z - z.max(1, keepdim=True).values)
            out[a:a + step, h] = torch.matmul(w[:, :n].contiguous(), vh) / w.sum(1, keepdim=True)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s)
    if case["kind"] == "logprobs":
        x = s["logits"].double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices
        ids = ids[:, :case["top"]]
        return dict(logprobs=lp[torch.arange(len(x), device="cuda"), s["tokens"]],
                    entropy=torch.special.entr(lp.exp()).sum(-1), top_ids=ids,
                    top_logprobs=torch.take_along_dim(lp, ids, -1))
    page, scales = case["page"], [s["k_scales"], s["v_scales"]]
    pool = [s[n].transpose(1, 2).flatten(0, 1).double() * sc.transpose(1, 2).flatten(0, 1)[..., None]
            for n, sc in zip(("k_cache", "v_cache"), scales)]  # (rows, Hkv, dim)
    if case["kind"] == "paged":
        out = []
        for r, n in enumerate(s["host_seq"]):
            at = torch.arange(n, device="cuda")
            rows = s["table"][r].long()[at // page] * page + at % page
            out.append(_exact_sequence(s["q"][s["host_qs"][r]:s["host_qs"][r + 1]], pool[0][rows],
                                       pool[1][rows], case["window"], case["first"], s["sinks"]))
        return torch.cat(out)
    at = s["slots"].long()
    if case["kind"] == "read":
        return [p[at] for p in pool]
    there, back, kept = at >= 0, [], []
    for x, sc in ((s["k"], scales[0]), (s["v"], scales[1])):
        x = x.double()
        # The scale as it is kept, in 32 bits.
        by = (x.abs().max(-1, keepdim=True).values / 127).to(torch.float32).double()
        back.append(torch.round(x / by) * by * there[:, None, None])
        flat = sc.transpose(1, 2).flatten(0, 1).double().contiguous()
        flat[at[there]] = by[there][..., 0]
        kept.append(flat.unflatten(0, (-1, page)).transpose(1, 2))
    return back + kept
