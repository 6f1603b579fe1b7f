"""Synthetic Llama-style decoder for end-to-end determinism checks.

A torch restatement of the reference's benchmark model (reference
bench/bench.py:108-162: RMSNorm, q/k/v/o projections, causal GQA attention,
SiLU-gated MLP, residual adds, final norm and vocabulary head) and of its
determinism check (bench/bench.py:217-246): the logits of one sequence must
have the same bits whether it runs alone or inside a larger batch.

Under ``batch_invariant_mode`` every projection runs the invariant GEMM and
attention runs the invariant kernel; RMSNorm, SiLU, the embedding and the
residual adds are stock torch, which computes them per row with a fixed
reduction (tests/test_gpu_stock_ops.py guards that). Weights are random:
there is no checkpoint. They are drawn on the device from torch's seeded
generator, so the same seed gives the same model.

:class:`PagedCache` and :func:`serve_step` run the same model over a paged cache,
request by request and chunk by chunk (bi.page_tables, bi.paged_cache_update,
bi.paged_attention); :func:`generate` decodes greedily on top of them. Under
``batch_invariant_mode`` a request's logits have the same bits whatever is
served beside it and however its prompt is cut into chunks.
"""

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F


@dataclass(frozen=True)
class DecoderConfig:
    hidden: int = 4096
    inter: int = 11008
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    layers: int = 32
    vocab: int = 32000
    eps: float = 1e-5


# random-init Llama-style decoder, 32 layers, hidden 4096,
# 32/8 heads, FFN 11008, vocabulary 32000.
LLAMA_7B_SHAPE = DecoderConfig()


class Block(torch.nn.Module):
    def __init__(self, c, device, dtype):
        super().__init__()
        kw = dict(bias=False, device=device, dtype=dtype)
        self.c = c
        self.q = torch.nn.Linear(c.hidden, c.heads * c.head_dim, **kw)
        self.k = torch.nn.Linear(c.hidden, c.kv_heads * c.head_dim, **kw)
        self.v = torch.nn.Linear(c.hidden, c.kv_heads * c.head_dim, **kw)
        self.o = torch.nn.Linear(c.heads * c.head_dim, c.hidden, **kw)
        self.gate = torch.nn.Linear(c.hidden, c.inter, **kw)
        self.up = torch.nn.Linear(c.hidden, c.inter, **kw)
        self.down = torch.nn.Linear(c.inter, c.hidden, **kw)
        self.n1 = torch.nn.RMSNorm(c.hidden, eps=c.eps, device=device, dtype=dtype)
        self.n2 = torch.nn.RMSNorm(c.hidden, eps=c.eps, device=device, dtype=dtype)

    def forward(self, x):
        c = self.c
        B, L, _ = x.shape
        y = self.n1(x)
        q = self.q(y).view(B, L, c.heads, c.head_dim).transpose(1, 2)
        k = self.k(y).view(B, L, c.kv_heads, c.head_dim).transpose(1, 2)
        v = self.v(y).view(B, L, c.kv_heads, c.head_dim).transpose(1, 2)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=L > 1,
                                           scale=1.0 / math.sqrt(c.head_dim), enable_gqa=True)
        x = x + self.o(a.transpose(1, 2).reshape(B, L, c.heads * c.head_dim))
        y = self.n2(x)
        return x + self.down(F.silu(self.gate(y)) * self.up(y))


class Decoder(torch.nn.Module):
    def __init__(self, c, device, dtype):
        super().__init__()
        self.c = c
        self.embed = torch.nn.Embedding(c.vocab, c.hidden, device=device, dtype=dtype)
        self.blocks = torch.nn.ModuleList(Block(c, device, dtype) for _ in range(c.layers))
        self.norm = torch.nn.RMSNorm(c.hidden, eps=c.eps, device=device, dtype=dtype)
        self.head = torch.nn.Linear(c.hidden, c.vocab, bias=False, device=device, dtype=dtype)

    def forward(self, ids):
        """Logits of the last position of every sequence, (B, vocab)."""
        x = self.embed(ids)
        for blk in self.blocks:
            x = blk(x)
        return self.head(self.norm(x[:, -1]))


def build(config=LLAMA_7B_SHAPE, device="cuda", dtype=torch.bfloat16, seed=0):
    """Random-init decoder: nn.Linear / nn.Embedding default initialisation
    drawn on `device` after torch.manual_seed(seed)."""
    torch.manual_seed(seed)
    with torch.no_grad():
        m = Decoder(config, torch.device(device), dtype)
    return m.eval().requires_grad_(False)


def prompts(config, batch, length, seed=0, device="cuda"):
    """Token ids (batch, length): row 0 is the probe sequence, the other rows
    are unrelated sequences, all from a CPU generator seeded `seed`."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, config.vocab, (batch, length), generator=g).to(device)


def logits_bits(model, ids, invariant):
    """Bit pattern of row 0's last-position logits, with or without
    batch_invariant_mode."""
    from . import batch_invariant_mode

    with torch.no_grad():
        if invariant:
            with batch_invariant_mode():
                y = model(ids)
        else:
            y = model(ids)
    return y[0].contiguous().view(torch.int16 if y.dtype != torch.float32 else torch.int32)


def determinism(model, length=512, batches=(2, 4, 8), seed=0, invariant=True):
    """{batch: number of logits of sequence 0 whose bits differ from batch 1}."""
    c = model.c
    device = next(model.parameters()).device
    ids = prompts(c, max(batches), length, seed=seed, device=device)
    base = logits_bits(model, ids[:1], invariant)
    return {B: int((logits_bits(model, ids[:B], invariant) != base).sum()) for B in batches}


class PagedCache:
    """Keys and values of up to `requests` requests of up to `max_len` tokens in
    pages shared by all, one pool per layer; one table for all layers. The
    lengths are kept on the host too, which sizes every step without asking the
    GPU."""

    def __init__(self, config, requests, max_len, page_size=64, num_pages=None, device="cuda",
                 dtype=torch.bfloat16):
        c = config
        width = -(-max_len // page_size)
        self.num_pages = requests * width if num_pages is None else num_pages
        self.page_size, self.max_len = page_size, max_len
        shape = (c.layers, self.num_pages, c.kv_heads, page_size, c.head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.tables = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(self.num_pages, dtype=torch.int32, device=device)
        self.used = 0
        self.lens = [0] * requests

    def begin(self, new):
        """Takes the pages of a step that brings new[r] tokens of request r;
        returns its bi.PageTables and (most new tokens, longest request)."""
        from . import page_tables

        if len(new) != len(self.lens) or min(new) < 0:
            raise ValueError("expected %d token counts, got %s" % (len(self.lens), list(new)))
        after = [a + b for a, b in zip(self.lens, new)]
        if max(after) > self.max_len:
            raise ValueError("a request of %d tokens exceeds max_len %d" % (max(after), self.max_len))
        pages = lambda n: -(-n // self.page_size)
        need = sum(pages(b) - pages(a) for a, b in zip(self.lens, after))
        if self.used + need > self.num_pages:
            raise RuntimeError("%d pages needed, %d of %d free"
                               % (need, self.num_pages - self.used, self.num_pages))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.tables.device)
        t = page_tables(self.tables, i32(self.lens), i32(new), self.free[self.used:],
                        self.page_size, sum(new))
        self.used += need
        self.lens = after
        return t, max(new), max(after)

    def release(self, request):
        """Ends a request: its pages are free again and its row, empty, is
        another's. Steps that were launched before still read what was there
        (the pages change hands in the stream's order)."""
        n = -(-self.lens[request] // self.page_size)
        self.free[self.used - n:self.used] = self.tables[request, :n]
        self.tables[request] = -1
        self.used -= n
        self.lens[request] = 0


def serve_step(model, cache, ids, new):
    """One step over `cache`: ids (sum of new,) are the new tokens, new[r] of
    request r, one request behind the other. Returns the logits of every
    request's last token, (requests, vocab); those of a request without a new
    token are its neighbour's and mean nothing."""
    from . import paged_attention, paged_cache_update

    c = model.c
    if ids.ndim != 1 or ids.shape[0] != sum(new) or not ids.shape[0]:
        raise ValueError("expected %d ids, one or more, got %s" % (sum(new), tuple(ids.shape)))
    t, most, longest = cache.begin(new)
    x = model.embed(ids)
    T = x.shape[0]
    for i, blk in enumerate(model.blocks):
        y = blk.n1(x)
        k = blk.k(y).view(T, c.kv_heads, c.head_dim)
        v = blk.v(y).view(T, c.kv_heads, c.head_dim)
        paged_cache_update(k, v, cache.k[i], cache.v[i], t.slots)
        a = paged_attention(blk.q(y).view(T, c.heads, c.head_dim), cache.k[i], cache.v[i],
                            t.block_tables, t.query_start, t.seq_lens, max_query=most,
                            max_seq=longest)
        x = x + blk.o(a.reshape(T, c.heads * c.head_dim))
        y = blk.n2(x)
        x = x + blk.down(F.silu(blk.gate(y)) * blk.up(y))
    last = (t.query_start[1:] - 1).clamp(min=0).long()
    return model.head(model.norm(x[last]))


def generate(model, prompts, steps, chunk=None, page_size=64, logits=None):
    """Greedy continuation of `prompts` (1-d id tensors of any lengths) by
    `steps` tokens each, (len(prompts), steps). Prompts enter in chunks of up to
    `chunk` tokens (all of a prompt by default), all requests in one batch. A
    list passed as `logits` receives every decoded token's (requests, vocab)."""
    if not prompts or min(p.shape[0] for p in prompts) < 1 or steps < 1:
        raise ValueError("expected prompts of one token or more and steps >= 1")
    if chunk is not None and chunk < 1:
        raise ValueError("chunk must be >= 1, got %d" % chunk)
    device = next(model.parameters()).device
    dtype = model.head.weight.dtype
    left = [p.to(device) for p in prompts]
    cache = PagedCache(model.c, len(left), max(p.shape[0] for p in left) + steps, page_size,
                       device=device, dtype=dtype)
    first = [None] * len(left)
    with torch.no_grad():
        while any(p.shape[0] for p in left):
            part = [p if chunk is None else p[:chunk] for p in left]
            y = serve_step(model, cache, torch.cat(part), [p.shape[0] for p in part])
            for r, p in enumerate(part):
                left[r] = left[r][p.shape[0]:]
                if p.shape[0] and not left[r].shape[0]:
                    first[r] = y[r]
        y, out = torch.stack(first), []
        for s in range(steps):
            if logits is not None:
                logits.append(y)
            out.append(y.argmax(-1))
            if s + 1 < steps:
                y = serve_step(model, cache, out[-1], [1] * len(left))
    return torch.stack(out, 1)
