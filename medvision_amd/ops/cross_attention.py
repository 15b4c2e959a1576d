"""``cross_attention``: queries of a decoder over an encoder's states of another length.  No counterpart in the reference."""
from torch.autograd.function import once_differentiable

from .._lib import native
from ._function import NativeFunction


class CrossAttentionFunction(NativeFunction):
    @staticmethod
    def native(query, key, value, key_mask=None, key_lengths=None, scale=None):
        return native.cross_attention(query, key, value, key_mask, key_lengths, scale)

    @staticmethod
    def forward(ctx, query, key, value, key_mask=None, key_lengths=None, scale=None):
        output, lse, low = native.cross_attention_forward(query, key, value, key_mask, key_lengths, scale)
        ctx.save_for_backward(query, key, value, key_mask, key_lengths, output, lse, low)
        ctx.scale = scale
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        query, key, value, key_mask, key_lengths, output, lse, low = ctx.saved_tensors
        wanted = ctx.needs_input_grad[:3]
        grads = native.cross_attention_backward(query, key, value, key_mask, key_lengths, output, lse, low, grad_output, ctx.scale,
                                                wanted[0], wanted[1] or wanted[2])
        return (*(g if w else None for g, w in zip(grads, wanted)), None, None, None)


def cross_attention(query, key, value, key_mask=None, key_lengths=None, scale=None):
    """Attention of queries over the keys and values of another length, with the gradients of all three.

    Args:
        query (Tensor): ``[batch, queries, heads, channels]``; float32, float16 or bfloat16, 1 to 128 channels per head
        key, value (Tensor): ``[batch, keys, key_heads, channels]``; ``heads`` is a multiple of ``key_heads``, consecutive
            heads of the query share a head of the keys.  Views are read in place as long as a head's channels are neighbours
        key_mask (Tensor): bool ``[batch, keys]``, False where a key does not count
        key_lengths (Tensor): whole numbers ``[batch]``: keys from there on do not count
        scale (float): of the products of queries and keys, ``channels ** -0.5`` by default

    What keys and values that do not count hold has no effect, not even NaN.  A query without any key gets zeros.  Gradients
    are formed for the inputs that want one.  Scores, their softmax and all sums are in 32 bits; of float16 and bfloat16 the
    softmax's weights are rounded to that type before they meet the values, and in the gradients of keys and values (with
    their own gradients) from 2 ** 20 weights on, unless there are no more than 32 keys or 64 rows for a head of keys.
    """
    return CrossAttentionFunction.apply(query, key, value, key_mask, key_lengths, scale)
