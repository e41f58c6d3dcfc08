"""Tensor-parallel linear layers whose three products run on operands in 8-bit blocks (``LayerConfig.linear_format = "fp8_blocks"``).

``y = x . W^T``, ``dx = dy . W`` and ``dW = dy^T . x`` as in ``linear.py``, each of ``x``, ``dy`` (a scale per 128 elements along the
contraction) and ``W`` (a scale per 128 x 128 tile) rounded to e4m3 on its way in; sums in fp32, results in the parameters' type.  What is
saved is what the backward reads: the input's columns and the weight's columns in 8-bit blocks, a byte for each element of either (the
bf16 layers save two for each of the input), and for matrices that take at most 2 MB in both orientations the rows' as well, which lie in
the same allocation.  The reference's layers take the same place with TransformerEngine quantizers
(kareus/transformer_engine/pytorch/ops/basic/basic_linear.py:391-604, 606-915).

The weight gradient over the nanobatches of a pass is one product over all their tokens, launched where ``linear.py`` launches its own.
A pass quantises a weight once: the first nanobatch to get to the layer does, the others of the pass read its result, and the last one
drops the rows' orientation; the columns are saved for the backward.  The residual add and the SwiGLU activation behind and in front of
the layers run as operators of their own.
"""

from __future__ import annotations

from ..backend import get_backend
from ..block_scaled import BlockOperand, BlockScaled
from ..partitions.streams import stream_api
from .linear import PartitionableLinear, TEColumnParallelLinearOp, TERowParallelLinearOp


def _used_on(stream, *tensors) -> None:
    """Their memory is not given away before what ``stream`` has been asked to do with them is done."""
    for t in tensors:
        if t.is_cuda:
            t.record_stream(stream)


class BlockLinear(PartitionableLinear):
    """Bias-free linear layer over 8-bit blocks; ``weight`` is ``[output_size, input_size]`` in the parameters' type."""

    fuse_activation = False

    def _weight_blocks(self, be, ctx, by_col: bool):
        """The weight in 8-bit blocks, and the stream that they were made on."""
        shared = ctx.pass_shared
        api = stream_api()
        here = None if ctx.alone else api.current_stream()
        entry = None if shared is None else shared.get(id(self))
        if entry is None:
            blocks = be.quantize_blocks(self.weight.detach(), by_row=True, by_col=by_col, tiles=True)
            if shared is not None:
                ready = None
                if here is not None:
                    ready = api.new_event()
                    ready.record(here)
                shared[id(self)] = [blocks, ready, here, shared.readers - 1]
            return blocks, here
        blocks, ready, where, left = entry
        if left == 1:
            del shared[id(self)]    # (the memory is the streams' that were asked to read it until they have)
        else:
            entry[3] = left - 1
        if here is not None and ready is not None and where != here:
            here.wait_event(ready)
            for t in blocks:
                if t is not None:
                    _used_on(here, t.data, t.scales)
        return blocks, where

    def fuser_forward(self, basic_op_ctxs, input_, *, basic_op_extra_inputs, basic_op_prev_ops,
                      basic_op_next_ops, basic_op_kwargs):
        (ctx,) = basic_op_ctxs
        n, k = self.weight.shape
        if input_.shape[-1] != k:
            raise ValueError(f"linear with in_features={k} got input of shape {tuple(input_.shape)}")
        be = get_backend(self._backend_name)
        x = be.quantize_blocks(be.rows_in_place(input_), by_row=True, by_col=ctx.requires_grad and self.weight.requires_grad)
        w, ctx.weight_stream = self._weight_blocks(be, ctx, ctx.requires_grad)
        y = be.block_matmul(x.by_row, w.by_row, dtype=self.weight.dtype)
        if ctx.requires_grad:
            # (aliases of the weight's: the engine drops the storage behind saved tensor objects, one nanobatch after the other)
            xt = (None, None) if x.by_col is None else (x.by_col.data, x.by_col.scales)
            ctx.save_for_backward(*xt, w.by_col.data.detach(), w.by_col.scales.detach())
            ctx.input_requires_grad = True
            ctx.tokens = y.shape[0]
        return y.view(*input_.shape[:-1], n), [()]

    def fuser_backward(self, basic_op_ctxs, grad_output, *, basic_op_grad_extra_outputs):
        (ctx,) = basic_op_ctxs
        dx, param_grads = self.op_backward(ctx, grad_output)
        return dx, [param_grads], [()]

    def op_backward(self, ctx, grad_output):
        xq, xs, wq, ws = ctx.saved_tensors
        n, k = self.weight.shape
        be = get_backend(self._backend_name)
        api = stream_api()
        here = None if ctx.alone else api.current_stream()
        if here is not None and ctx.weight_stream is not None and ctx.weight_stream != here:
            _used_on(here, wq, ws)
        dy = be.quantize_blocks(be.rows_in_place(grad_output), by_row=True, by_col=xq is not None)
        dx = be.block_matmul(dy.by_row, BlockOperand(wq, ws, n), dtype=grad_output.dtype)
        dw = None
        if xq is not None:
            dw = self._block_weight_grad(be, ctx, dy.by_col, BlockOperand(xq, xs, ctx.tokens))
        return dx.view(*grad_output.shape[:-1], k), (dw,)

    def _block_weight_grad(self, be, ctx, dy: BlockOperand, x: BlockOperand):
        """``dW = dy^T . x``.  With the engine's ``wgrad_sink`` (see ``PartitionableLinear._weight_grad``) the nanobatches' operands are
        contracted in one launch, with one fp32 sum and one rounding.  Where the layer's configuration asks for a product per nanobatch
        (``wgrad_over_all_nanobatches`` off), the first allocates the gradient and later ones add to it, rounding it to its type
        each time, as the bf16 layers do there."""
        sink = getattr(ctx, "wgrad_sink", None)
        if sink is None:
            return be.block_matmul(dy, x, dtype=self.weight.dtype)
        api = stream_api()
        here = None if sink.get("in_line") else api.current_stream()
        if sink.get("n", 0) > 1 and sink.get("defer", True):
            # (aliases: the engine drops the storage behind the saved tensor objects after each backward op)
            return self._over_all_nanobatches(
                sink, ctx, here, dy, x._replace(data=x.data.detach(), scales=x.scales.detach()),
                lambda dys, xs: self.weight.new_empty(self.weight.shape),
                lambda dys, xs, dw: be.block_matmul_segments(dys, xs, out=dw, dtype=dw.dtype),
                lambda pair: (t for o in pair for t in (o.data, o.scales)))
        buf = sink.get("buf")
        if buf is None:
            ret = sink["buf"] = be.block_matmul(dy, x, dtype=self.weight.dtype)
        else:
            if here is not None and sink.get("event") is not None:
                here.wait_event(sink["event"])
                _used_on(here, buf)
            be.block_matmul(dy, x, out=buf, accumulate=True, dtype=self.weight.dtype)
            ret = None
        if here is not None:
            sink["event"] = api.new_event()
            sink["event"].record(here)
        return ret


class BlockColumnParallelLinearOp(BlockLinear, TEColumnParallelLinearOp):
    """Output features are sharded; its backward input-gradient needs the all-reduce."""


class BlockRowParallelLinearOp(BlockLinear, TERowParallelLinearOp):
    """Input features are sharded; its forward output needs the all-reduce."""
