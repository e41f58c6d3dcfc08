"""The two ends around the layer stack, so that a stack computes a loss from token ids:
embedding -> LayerStack -> final RMSNorm -> output layer -> cross entropy.

What the reference runs outside its partitions ("non-partition" work,
tests/bayesian/nonpartition/profile_nonpartition.py:148-486): ``LanguageModelEmbedding``
(3rdparty/Megatron-LM/megatron/core/models/common/embeddings/language_model_embedding.py:95-116,
word embeddings only — rotary positions — and the ``[b s h] -> [s b h]`` layout change), the
block's final layer norm (kareus/megatron/core/transformer/transformer_block.py:521-525), a
column-parallel output layer without bias, and ``compute_language_model_loss``
(3rdparty/Megatron-LM/megatron/core/models/common/language_module/language_module.py:71-101:
labels ``[b, s]``, logits ``[s, b, vocab]``, loss ``[b, s]``).

One GPU holds one vocabulary shard ``[vocab_start, vocab_start + vocab_rows)``.  The embedding
follows the shard semantics (ids of other shards embed to zero, which the missing all-reduce
would fill in); the loss treats the shard's columns as the whole vocabulary, which is exact for a
single shard and is what the per-shard kernels compute before the cross-shard max/sum exchange.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from .backend import get_backend
from .block import LayerConfig, LayerStack
from .partitions.streams import stream_api


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, vocab_start, backend):
        ctx.save_for_backward(ids)
        ctx.vocab_start, ctx.backend, ctx.rows = vocab_start, backend, weight.shape[0]
        return get_backend(backend).embedding_fwd(ids, weight.detach(), vocab_start)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        return None, get_backend(ctx.backend).embedding_bwd(ids, dout, ctx.rows, ctx.vocab_start), None, None


class _MainGradOrder:
    """Sums into one ``main_grad`` run one behind the other, whatever streams their forward passes ran on, and the stream that called
    ``backward()`` goes on behind them: what autograd sees to for the gradients that it accumulates itself."""

    def __init__(self) -> None:
        self.last = None    # (event behind the last sum, its stream, the captured pass that it is part of)

    def __reduce__(self):   # (a copy of a module, or one that was saved, has no sums under way)
        return _MainGradOrder, ()

    @staticmethod
    def _captured(weight: Tensor):
        """An event of a capture means nothing outside it, and one from before it nothing inside, where the device was waited for."""
        return torch._C._current_graph_task_id() if weight.is_cuda and torch.cuda.is_current_stream_capturing() else None

    def begin(self, weight: Tensor, out: Tensor) -> None:
        here = stream_api().current_stream()
        if here is not None and self.last is not None:
            event, stream, captured = self.last
            if stream != here and captured == self._captured(weight):
                self._behind(here, event, out)

    def end(self, weight: Tensor, out: Tensor) -> None:
        api = stream_api()
        here = api.current_stream()
        if here is None:
            return
        event = api.new_event()
        event.record(here)
        self.last = (event, here, self._captured(weight))

        def done() -> None:
            caller = api.current_stream()
            if caller != here:
                self._behind(caller, event, out)

        torch.autograd.Variable._execution_engine.queue_callback(done)

    @staticmethod
    def _behind(stream, event, out: Tensor) -> None:
        stream.wait_event(event)
        if out.is_cuda:
            out.record_stream(stream)


class _SortedEmbedding(torch.autograd.Function):
    """The embedding times ``scale``, its gradient by sorted tokens.  With ``order`` the gradient goes to the weight's fp32
    ``main_grad``, which the first backward pass writes whole and later ones add to, and autograd sees none."""

    @staticmethod
    def forward(ctx, ids, weight, vocab_start, scale, order, backend):
        ctx.save_for_backward(ids)
        ctx.vocab_start, ctx.scale, ctx.backend, ctx.rows = vocab_start, scale, backend, weight.shape[0]
        ctx.main, ctx.order = weight if order is not None else None, order
        return get_backend(backend).embedding_fwd(ids, weight.detach(), vocab_start, scale=scale)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        be, w = get_backend(ctx.backend), ctx.main
        out, add = None, False
        if w is not None:
            out = getattr(w, "main_grad", None)
            add = out is not None
            if not add:
                out = torch.empty(w.shape, dtype=torch.float32, device=w.device)
            ctx.order.begin(w, out)
        dw = be.embedding_bwd_sorted(ids, dout, ctx.rows, ctx.vocab_start, scale=ctx.scale, out=out, accumulate=add)
        if w is not None:
            ctx.order.end(w, out)
            w.main_grad, dw = out, None
        return None, dw, None, None, None, None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, eps, backend):
        x2d = x.reshape(-1, x.shape[-1])
        y, rstd = get_backend(backend).rmsnorm_fwd(x2d, gamma.detach(), eps)
        ctx.save_for_backward(x2d, rstd, gamma)
        ctx.backend = backend
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2d, rstd, gamma = ctx.saved_tensors
        dx, dgamma = get_backend(ctx.backend).rmsnorm_bwd(dy.reshape(x2d.shape), x2d, rstd, gamma.detach())
        return dx.view(dy.shape), dgamma, None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, backend):
        x2d = x.reshape(-1, x.shape[-1])
        ctx.save_for_backward(x2d, weight)
        ctx.backend = backend
        return get_backend(backend).linear_fwd(x2d, weight.detach()).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2d, weight = ctx.saved_tensors
        be = get_backend(ctx.backend)
        dy2d = dy.reshape(-1, dy.shape[-1])
        if not dy2d.is_contiguous():
            dy2d = dy2d.contiguous()
        dx = be.linear_dgrad(dy2d, weight.detach())
        return dx.view(*dy.shape[:-1], weight.shape[1]), be.linear_wgrad(dy2d, x2d), None


class _CrossEntropy(torch.autograd.Function):
    """logits [s, b, vocab], labels [b, s] -> loss [b, s] (fp32).  Backward overwrites the logits
    with their gradient (they are dead after the loss), as the fused implementations do."""

    @staticmethod
    def forward(ctx, logits, labels, backend):
        s, b, vocab = logits.shape
        rows = labels.transpose(0, 1).contiguous().view(-1)            # [s, b] order, like the logits
        loss, lse = get_backend(backend).cross_entropy_fwd(logits.reshape(-1, vocab), rows)
        ctx.save_for_backward(logits, rows, lse)
        ctx.backend = backend
        return loss.view(s, b).transpose(0, 1).contiguous()

    @staticmethod
    def backward(ctx, dloss):
        logits, rows, lse = ctx.saved_tensors
        s, b, vocab = logits.shape
        g = dloss.transpose(0, 1).contiguous().view(-1)
        d = get_backend(ctx.backend).cross_entropy_bwd(logits.reshape(-1, vocab), rows, lse, g,
                                                       in_place=logits.is_contiguous())
        return d.view(s, b, vocab), None, None


class LanguageModelEmbedding(torch.nn.Module):
    """Word embeddings of one vocabulary shard; ``forward(input_ids [b, s]) -> scale * rows, [s, b, hidden]``.

    ``sorted_gradient``: the weight's gradient is summed by sorted tokens instead of by vocabulary rows (always so with a scale or
    ``main_grad``), which takes as long whatever the ids are.  By rows a workgroup adds up all tokens of its rows, so that ids which come
    often cost most (us by rows and sorted, into 32064 x 4096: 16056 tokens of evenly spread ids 102, 109, as frequent as in text 1388, 112,
    with 30 % of one id 5393, 106; 512 tokens 38, 47; 64, 48; 167, 47).  ``main_grad``: it is kept over backward passes in an fp32
    ``weight.main_grad``, ``None`` until the first (set it back to ``None``, or zero it, for the next step); a pass touches the rows of
    its tokens only."""

    def __init__(self, config: LayerConfig, vocab_rows: int, vocab_start: int = 0, device=None,
                 generator=None, scale: float = 1.0, sorted_gradient: bool = False, main_grad: bool = False) -> None:
        super().__init__()
        w = torch.empty(vocab_rows, config.hidden_size, dtype=torch.float32)
        w.normal_(0.0, config.init_method_std, generator=generator)
        self.weight = torch.nn.Parameter(w.to(device=device, dtype=config.params_dtype))
        self.vocab_start, self._backend = int(vocab_start), config.backend
        self.scale, self.main_grad = float(scale), bool(main_grad)
        self.sorted_gradient = bool(sorted_gradient) or self.main_grad or self.scale != 1.0
        self._order = _MainGradOrder() if self.main_grad else None
        if self.main_grad:
            self.weight.main_grad = None

    def forward(self, input_ids: Tensor) -> Tensor:
        if self.sorted_gradient:
            return _SortedEmbedding.apply(input_ids, self.weight, self.vocab_start, self.scale, self._order, self._backend)
        return _Embedding.apply(input_ids, self.weight, self.vocab_start, self._backend)


class GPTModelShard(torch.nn.Module):
    """``forward(input_ids [b, s], labels [b, s] or None)`` -> loss ``[b, s]`` (fp32) or logits
    ``[s, b, vocab_rows]``.  ``embedding_scale``, ``embedding_sorted_gradient``, ``embedding_main_grad``: see
    :class:`LanguageModelEmbedding`."""

    def __init__(self, config: LayerConfig, vocab_rows: int, vocab_start: int = 0, device=None,
                 seed: Optional[int] = None, embedding_scale: float = 1.0, embedding_sorted_gradient: bool = False,
                 embedding_main_grad: bool = False) -> None:
        super().__init__()
        gen = torch.Generator().manual_seed(seed + 1) if seed is not None else None
        self.config = config
        self.embedding = LanguageModelEmbedding(config, vocab_rows, vocab_start, device=device, generator=gen, scale=embedding_scale,
                                                sorted_gradient=embedding_sorted_gradient, main_grad=embedding_main_grad)
        self.decoder = LayerStack(config, device=device, seed=seed)
        self.final_layernorm = torch.nn.Parameter(
            torch.ones(config.hidden_size, device=device, dtype=config.params_dtype))
        w = torch.empty(vocab_rows, config.hidden_size, dtype=torch.float32)
        w.normal_(0.0, config.init_method_std, generator=gen)
        self.output_layer = torch.nn.Parameter(w.to(device=device, dtype=config.params_dtype))

    def forward(self, input_ids: Tensor, labels: Optional[Tensor] = None) -> Tensor:
        be = self.config.backend
        hidden = self.decoder(self.embedding(input_ids))
        hidden = _RMSNorm.apply(hidden, self.final_layernorm, self.config.layernorm_epsilon, be)
        logits = _Linear.apply(hidden, self.output_layer, be)
        if labels is None:
            return logits
        return _CrossEntropy.apply(logits, labels, be)
