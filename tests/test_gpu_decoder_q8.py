"""The new operators together, as a decoder serves with them: positions, an 8-bit
cache, log probabilities."""

import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import decoder

import helpers

pytestmark = pytest.mark.gpu


def same(a, b):
    if not a.is_floating_point():
        return bool((a == b).all())
    return a.shape == b.shape and bool((helpers.bits(a) == helpers.bits(b)).all())


def model(cuda, dtype=torch.bfloat16, **kw):
    c = decoder.DecoderConfig(hidden=256, inter=384, heads=4, kv_heads=2, head_dim=64, layers=2, vocab=517,
                              **kw)
    return decoder.build(c, device=cuda, dtype=dtype, seed=3)


ROPE = dict(rope_base=10000.0)


def texts(cuda, *lens):
    g = torch.Generator().manual_seed(4)
    return [torch.randint(0, 517, (n,), generator=g).to(cuda) for n in lens]


@pytest.mark.parametrize("dtype, kw", [(torch.bfloat16, ROPE), (torch.float16, dict(ROPE, rope_interleaved=True)),
                                       (torch.bfloat16, dict(ROPE, rope_dim=32)), (torch.float16, {})])
@pytest.mark.parametrize("cache_dtype", [None, torch.int8])
def test_scoring_gives_the_bits_of_generating(cuda, dtype, kw, cache_dtype):
    """Log probabilities of generated tokens, with alternatives: the same bits from
    the decoding steps, from scoring the whole texts at once and in chunks, and for
    a text alone."""
    m = model(cuda, dtype, **kw)
    prompts = texts(cuda, 3, 70, 41)
    steps = 12
    with torch.no_grad(), bi.batch_invariant_mode():
        kept = []
        ids = decoder.generate(m, prompts, steps, page_size=16, cache_dtype=cache_dtype, logprobs=kept, top=4)
        whole = [torch.cat([p, i]) for p, i in zip(prompts, ids)]
        for how in (dict(), dict(chunk=7), dict(chunk=33, page_size=8)):
            got = decoder.score(m, whole, top=4, cache_dtype=cache_dtype, **how)
            for r, p in enumerate(prompts):
                assert got[r].logprobs.shape == (p.shape[0] + steps - 1,)
                for name in got[r]._fields:
                    want = torch.stack([getattr(k, name)[r] for k in kept])
                    assert same(getattr(got[r], name)[-steps:], want), (how, r, name)
        alone = decoder.score(m, whole[1:2], top=4, cache_dtype=cache_dtype)[0]
        got = decoder.score(m, whole, top=4, cache_dtype=cache_dtype)[1]
        assert all(same(a, b) for a, b in zip(alone, got))
    # Greedy decoding takes the likeliest token.
    assert all(bool((k.top_ids[:, 0] == i).all()) for k, i in zip(kept, ids.T))
    assert all(same(k.top_logprobs[:, 0].contiguous(), k.logprobs) for k in kept)


@pytest.mark.parametrize("kw", [{}, ROPE])
def test_the_cache_holds_what_the_step_wrote(cuda, kw):
    """An 8-bit cache reads back within half a step of the same steps' cache in the
    model's type, wherever pages lie and however the prompt was cut; the first layer
    exactly as bi.paged_cache_update codes its rows."""
    m = model(cuda, **kw)
    (ids,) = texts(cuda, 90)
    with torch.no_grad(), bi.batch_invariant_mode():
        full, q8, cut = (decoder.PagedCache(m.c, 1, 100, page_size=16, device=cuda, dtype=d)
                         for d in (torch.bfloat16, torch.int8, torch.int8))
        a = decoder.serve_step(m, full, ids, [90])
        b = decoder.serve_step(m, q8, ids, [90])
        for n in range(0, 90, 18):
            c = decoder.serve_step(m, cut, ids[n:n + 18], [18])
    assert same(b, c)
    for layer in (0, 1):
        for x, y in zip(q8.read(0, layer), cut.read(0, layer)):
            assert same(x, y)
    for x, y in zip(full.read(0, 0), q8.read(0, 0)):
        x = x.float()
        step = x.abs().amax(-1, keepdim=True) / 127
        assert bool(((x - y).abs() <= step * (0.5 + 1e-4)).all())
    # The logits differ by the codes' rounding only: small beside their own size.
    assert (a.float() - b.float()).abs().max() < 0.25 * a.float().abs().max()


def test_positions_matter_and_batches_agree(cuda):
    """The dense forward and the served one turn by the same positions: equal first
    tokens are told apart, and a sequence's logits do not depend on its batch."""
    m, plain = model(cuda, **ROPE), model(cuda)
    ids = texts(cuda, 40, 40)
    batch = torch.stack(ids)
    with torch.no_grad(), bi.batch_invariant_mode():
        dense = m(batch)
        assert same(dense[0], m(batch[:1])[0])
        served = decoder.serve_step(m, decoder.PagedCache(m.c, 2, 64, device=cuda), torch.cat(ids), [40, 40])
        # The same model but for the attention kernels' arithmetic (bf16 throughout:
        # a few roundings of 2^-8 a layer).
        assert (dense.float() - served.float()).abs().max() < 0.1 * dense.float().abs().max()
        swapped = torch.stack([torch.cat([i[20:39], i[:20], i[39:]]) for i in ids])
        assert not same(m(swapped)[0], dense[0])
        assert not same(plain(batch)[0], dense[0])


def test_a_captured_step(cuda):
    """Positions, write, attention and log probabilities of a decoding step in one
    graph, replayed as the requests grow."""
    m = model(cuda, **ROPE)
    prompts = texts(cuda, 30, 55)
    c = m.c
    with torch.no_grad(), bi.batch_invariant_mode():
        want = []
        ids = decoder.generate(m, prompts, 6, page_size=16, cache_dtype=torch.int8, logprobs=want, top=3)
        cache = decoder.PagedCache(c, 2, 80, page_size=16, device=cuda, dtype=torch.int8)
        y = decoder.serve_step(m, cache, torch.cat(prompts), [30, 55])
        tables, free = cache.tables, cache.free[cache.used:].clone()
        lens = torch.tensor(cache.lens, dtype=torch.int32, device=cuda)
        one = torch.ones_like(lens)
        token = y.argmax(-1)

        def step():
            t = bi.page_tables(tables, lens, one, free, 16, 2)
            x, turn = m.embed(token), m.turn(t.positions)
            for i, blk in enumerate(m.blocks):
                h = blk.n1(x)
                q, k = turn(blk.q(h).view(2, c.heads, 64), blk.k(h).view(2, c.kv_heads, 64))
                bi.paged_cache_update(k, blk.v(h).view(2, c.kv_heads, 64), cache.k[i], cache.v[i], t.slots,
                                      **cache.scales(i))
                a = bi.paged_attention(q, cache.k[i], cache.v[i], t.block_tables, t.query_start, t.seq_lens,
                                       max_query=1, max_seq=80, **cache.scales(i))
                x = x + blk.o(a.reshape(2, -1))
                h = blk.n2(x)
                x = x + blk.down(torch.nn.functional.silu(blk.gate(h)) * blk.up(h))
            z = m.head(m.norm(x))
            best = z.argmax(-1)
            return best, bi.token_logprobs(z, best, top=3), t.pages_used

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        start = lens.clone()
        with torch.cuda.stream(stream):
            step()  # (writes the first step's rows, as the first replay does again)
        torch.cuda.synchronize()
        lens.copy_(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            best, lp, taken = step()
        for s in range(1, 6):
            graph.replay()
            torch.cuda.synchronize()
            assert bool((best == ids[:, s]).all())
            assert all(same(getattr(lp, f), getattr(want[s], f)) for f in lp._fields)
            token.copy_(best)
            lens.add_(1)
            free.copy_(free.roll(-int(taken)))


def test_texts_of_one_token(cuda):
    m = model(cuda, **ROPE)
    one, more = texts(cuda, 1, 9)
    got = decoder.score(m, [one, more], top=2, cache_dtype=torch.int8)
    assert [g.logprobs.shape[0] for g in got] == [0, 8] and got[0].top_ids.shape == (0, 2)
    assert bool(got[1].logprobs.isfinite().all())
