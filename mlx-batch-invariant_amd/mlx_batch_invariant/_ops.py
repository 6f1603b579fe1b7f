"""torch.library custom ops over the kernel launches, for torch.compile.

The reference's kernels are opaque to ``mx.compile``, which may reorder and
fuse the graph around them but never inside (reference
tests/test_invariance.py:595-640). The same holds here: while torch.compile
traces, ``bi.*`` calls become the ops ``mlx_bi::gemm``, ``mlx_bi::qgemm`` and
``mlx_bi::sdpa`` (and, for the paged cache, ``mlx_bi::page_tables``,
``mlx_bi::paged_cache_update`` (``_q8`` and ``_kept`` with scales),
``mlx_bi::paged_cache_read``, ``mlx_bi::paged_attention`` (``_q8``) and
``mlx_bi::window_attention``; ``mlx_bi::rotary`` and ``mlx_bi::token_logprobs``), which
the compiler treats as opaque nodes (their
fake implementations give only output shapes) and which run the HIP kernels
unchanged. Eager calls skip the dispatcher and launch directly.
"""

from typing import List, Optional, Tuple

import torch


@torch.library.custom_op("mlx_bi::gemm", mutates_args=())
def gemm(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor], trans_b: bool,
         alpha: float, beta: float) -> torch.Tensor:
    from . import _gemm

    return _gemm._gemm_eager(a, b, bias, trans_b, alpha, beta, None)


@gemm.register_fake
def _gemm_fake(a, b, bias, trans_b, alpha, beta):
    n = b.shape[0] if trans_b else b.shape[1]
    return a.new_empty((*a.shape[:-1], n))


@torch.library.custom_op("mlx_bi::sdpa", mutates_args=())
def sdpa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, mask_mode: int,
         mask: Optional[torch.Tensor], mstrides: List[int], causal_offset: int,
         sinks: Optional[torch.Tensor]) -> torch.Tensor:
    from . import _attention

    return _attention._sdpa_eager(q, k, v, scale, mask_mode, mask, mstrides, causal_offset,
                                  sinks)


@sdpa.register_fake
def _sdpa_fake(q, k, v, scale, mask_mode, mask, mstrides, causal_offset, sinks):
    return q.new_empty((q.shape[0], q.shape[1], q.shape[2], v.shape[-1]))


@torch.library.custom_op("mlx_bi::qgemm", mutates_args=())
def qgemm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
          group_size: int, bits: int) -> torch.Tensor:
    from . import _quant

    return _quant._quantized_linear_eager(x, w, scales, biases, group_size, bits)


@qgemm.register_fake
def _qgemm_fake(x, w, scales, biases, group_size, bits):
    return x.new_empty((*x.shape[:-1], w.shape[0]))


@torch.library.custom_op("mlx_bi::page_tables", mutates_args=("block_tables",))
def page_tables(block_tables: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                free_pages: torch.Tensor, page_size: int, num_tokens: int
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import _paged

    # Outputs of a custom op may not share storage.
    return tuple(t.clone() for t in _paged._page_tables_eager(
        block_tables, context_lens, new_lens, free_pages, page_size, num_tokens))


@page_tables.register_fake
def _page_tables_fake(block_tables, context_lens, new_lens, free_pages, page_size, num_tokens):
    n = context_lens.shape[0]
    return tuple(context_lens.new_empty(s) for s in ((num_tokens,), (num_tokens,), (n + 1,), (n,),
                                                     ()))


@torch.library.custom_op("mlx_bi::paged_cache_update", mutates_args=("k_cache", "v_cache"))
def paged_cache_update(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    from . import _paged

    _paged._update_eager(k, v, k_cache, v_cache, slots)


@paged_cache_update.register_fake
def _paged_cache_update_fake(k, v, k_cache, v_cache, slots):
    return None


@torch.library.custom_op("mlx_bi::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, query_start: torch.Tensor, seq_lens: torch.Tensor,
                    max_query: int, max_seq: int, scale: float, window: int, sink_tokens: int,
                    sinks: Optional[torch.Tensor]) -> torch.Tensor:
    from . import _paged

    return _paged._paged_eager(q, k_cache, v_cache, block_tables, query_start, seq_lens,
                               max_query, max_seq, scale, window, sink_tokens, sinks)


@paged_attention.register_fake
def _paged_attention_fake(q, k_cache, v_cache, block_tables, query_start, seq_lens, max_query,
                          max_seq, scale, window, sink_tokens, sinks):
    return q.new_empty((q.shape[0], q.shape[1], v_cache.shape[3]))


@torch.library.custom_op("mlx_bi::window_attention", mutates_args=())
def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, window: int,
                     sink_tokens: int, sinks: Optional[torch.Tensor]) -> torch.Tensor:
    from . import _paged

    return _paged._window_eager(q, k, v, scale, window, sink_tokens, sinks)


@window_attention.register_fake
def _window_attention_fake(q, k, v, scale, window, sink_tokens, sinks):
    return q.new_empty((q.shape[0], q.shape[1], q.shape[2], v.shape[-1]))


@torch.library.custom_op("mlx_bi::paged_cache_update_q8",
                         mutates_args=("k_cache", "v_cache", "k_scales", "v_scales"))
def paged_cache_update_q8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, slots: torch.Tensor, k_scales: torch.Tensor,
                          v_scales: torch.Tensor) -> None:
    from . import _paged

    _paged._update_q8_eager(k, v, k_cache, v_cache, slots, k_scales, v_scales, False)


@paged_cache_update_q8.register_fake
def _paged_cache_update_q8_fake(k, v, k_cache, v_cache, slots, k_scales, v_scales):
    return None


@torch.library.custom_op("mlx_bi::paged_cache_update_kept", mutates_args=("k_cache", "v_cache"))
def paged_cache_update_kept(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, slots: torch.Tensor, k_scales: torch.Tensor,
                            v_scales: torch.Tensor) -> None:
    from . import _paged

    _paged._update_q8_eager(k, v, k_cache, v_cache, slots, k_scales, v_scales, True)


@paged_cache_update_kept.register_fake
def _paged_cache_update_kept_fake(k, v, k_cache, v_cache, slots, k_scales, v_scales):
    return None


@torch.library.custom_op("mlx_bi::paged_cache_read", mutates_args=())
def paged_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                     k_scales: Optional[torch.Tensor], v_scales: Optional[torch.Tensor],
                     dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    from . import _paged

    return _paged._read_eager(k_cache, v_cache, slots, k_scales, v_scales, dtype)


@paged_cache_read.register_fake
def _paged_cache_read_fake(k_cache, v_cache, slots, k_scales, v_scales, dtype):
    T, Hkv = slots.shape[0], k_cache.shape[1]
    return (k_cache.new_empty((T, Hkv, k_cache.shape[3]), dtype=dtype),
            k_cache.new_empty((T, Hkv, v_cache.shape[3]), dtype=dtype))


@torch.library.custom_op("mlx_bi::rotary", mutates_args=())
def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
           interleaved: bool, offset: int, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    from . import _rotary

    return _rotary._rotary_eager(q, k, positions, inv_freq, interleaved, offset, scale)


@rotary.register_fake
def _rotary_fake(q, k, positions, inv_freq, interleaved, offset, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("mlx_bi::token_logprobs", mutates_args=())
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import _logprobs

    return _logprobs._logprobs_eager(logits, tokens, top)


@token_logprobs.register_fake
def _token_logprobs_fake(logits, tokens, top):
    f32 = dict(dtype=torch.float32)
    return (logits.new_empty(tokens.shape, **f32), logits.new_empty(tokens.shape, **f32),
            logits.new_empty((*tokens.shape, top), dtype=torch.int64),
            logits.new_empty((*tokens.shape, top), **f32))


@torch.library.custom_op("mlx_bi::paged_attention_q8", mutates_args=())
def paged_attention_q8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       block_tables: torch.Tensor, query_start: torch.Tensor,
                       seq_lens: torch.Tensor, max_query: int, max_seq: int, scale: float,
                       window: int, sink_tokens: int, sinks: Optional[torch.Tensor],
                       k_scales: torch.Tensor, v_scales: torch.Tensor) -> torch.Tensor:
    from . import _paged

    return _paged._paged_eager(q, k_cache, v_cache, block_tables, query_start, seq_lens,
                               max_query, max_seq, scale, window, sink_tokens, sinks, k_scales,
                               v_scales)


@paged_attention_q8.register_fake
def _paged_attention_q8_fake(q, k_cache, v_cache, block_tables, query_start, seq_lens, max_query,
                             max_seq, scale, window, sink_tokens, sinks, k_scales, v_scales):
    return q.new_empty((q.shape[0], q.shape[1], v_cache.shape[3]))
