"""The operators of a transformer over packed point clouds: layer normalisation, attention inside
every cloud of a batch, and a learned bias per bucket of the relative position of query and key.

Features are float32 or bfloat16 rows [N, ...] of all clouds one after the other, as everywhere in
the package; statistics, weights of the normalisation and bias tables are float32.  The kernels are
csrc/layer_norm.hip, csrc/attention.hip and csrc/attention_grads.hip; results and gradients are
summed in a fixed order."""
import torch

from . import _lib

_I32 = torch.int32

# Offsets of a bias over all its axes, axes * (2 R + 1), that the kernels' shared memory has room for
# (MCCNN_ATTENTION_MAX_OFFSETS).
MAX_OFFSETS = 1344


def layer_norm(features, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of `features` (float32 or
    bfloat16); `weight` and `bias` are float32 vectors.  Differentiable in all three."""
    return _lib.host().layer_norm(features, weight, bias, eps)


def packed_attention(queries, keys, values, query_splits=None, key_splits=None, key_sizes=None,
                     key_mask=None, causal=False, scale=None, bias_table=None, bias_buckets=None,
                     query_positions=None, key_positions=None):
    """Softmax attention inside every cloud of a packed batch -> [Nq, heads, channels].

    queries [Nq, heads, channels], keys and values [Nk, key_heads, channels] of one type, up to 128
    channels, `heads` a multiple of `key_heads`: query head h looks at key head h // (heads /
    key_heads).  Any strides with the channels one after the other (others are copied).

    query_splits, key_splits  int32 [clouds + 1] row offsets (`row_splits`), without them all rows
                are one cloud; a cloud may be empty on either side
    key_sizes   int32 [clouds]: rows in use of each cloud's keys, where the rows are a table with
                room to grow (rows behind them may hold anything)
    key_mask    bool [Nk]: False for keys that are not looked at (their rows may hold anything)
    causal      a query looks at the keys up to its own place; the last query stands at the last key
    scale       of the products, 1 / sqrt(channels) by default
    bias_table  float32 [axes, buckets, heads], one to three axes: added to a logit is the sum over
                the axes of the entry of bucket bias_buckets[offset + R], the offset key position -
                query position clamped to -R .. R; `bias_buckets` int32 [2 R + 1] (`offset_buckets`),
                axes * (2 R + 1) at most MAX_OFFSETS.  -inf hides a bucket
    query_positions, key_positions  int32 [Nq, axes], [Nk, axes], for instance grid cells; without
                them (one axis) the places of the tokens, counted as for `causal`

    A query that nothing is left for gets zeros and zero gradients.  Differentiable (once) in
    queries, keys, values and bias_table; gradients of keys that are not looked at are zero.

    Everything between operands and results is float32 (bfloat16 weights are multiplied in parts), and
    a call that records a gradient gives the same bits as one that does not.  Keys hidden by `causal`
    alone have to be finite.  A value of infinity that is looked at gives infinity in bfloat16; in
    float32 an infinity that is looked at, or a number within 2^-8 of the largest, gives NaN (such
    operands are multiplied as three bfloat16 parts)."""
    return _lib.host().packed_attention(queries, keys, values, query_splits, key_splits, key_sizes,
                                        key_mask, causal, scale, bias_table, bias_buckets,
                                        query_positions, key_positions)


def offset_buckets(num_buckets, max_offset, bidirectional=True, device="cuda"):
    """Bucket of every offset -max_offset .. max_offset, int32 [2 * max_offset + 1]: the first half of
    a direction's buckets hold one offset each, the others grow by equal ratios up to `max_offset`.
    Bidirectional: the upper half of the buckets is for offsets above 0; otherwise those share
    bucket 0 with offset 0.  `packed_attention` takes at most MAX_OFFSETS offsets over all axes of a bias.
    (Whole-number arithmetic: no offset depends on a logarithm's last bit.)"""
    side = num_buckets // 2 if bidirectional else num_buckets
    near = side // 2
    if near < 1 or max_offset < near:
        raise _lib.InvalidArgumentError(
            "offset_buckets expects at least %d buckets and offsets up to half a direction's buckets"
            % (4 if bidirectional else 2))
    wide = side - near
    # bucket near + n begins at the least offset o with o / near >= (max_offset / near) ** (n / wide)
    def bucket(size):
        if size < near:
            return size
        n = 0
        while n + 1 < wide and size ** wide >= near ** (wide - n - 1) * max_offset ** (n + 1):
            n += 1
        return near + n
    sizes = [bucket(o) for o in range(max_offset + 1)]
    after = [side + s for s in sizes] if bidirectional else [0] * (max_offset + 1)
    return torch.tensor(sizes[::-1] + after[1:], dtype=_I32, device=device)


def row_splits(point_cloud):
    """Row offsets of the clouds of a `PointCloud`, int32 [clouds + 1], for `packed_attention`; its
    points have to be stored cloud after cloud (put into `point_cloud.get_cloud_order()`)."""
    if point_cloud.get_cloud_order() is not None:
        raise _lib.InvalidArgumentError("row_splits expects points that are stored cloud after cloud")
    return _splits(point_cloud)


def _splits(point_cloud):
    sizes = point_cloud.get_sizes().reshape(-1)
    return torch.nn.functional.pad(sizes.cumsum(0), (1, 0)).to(_I32)
