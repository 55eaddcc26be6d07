"""What layer normalisation and attention refuse before anything reaches the GPU, and the buckets of
offsets.  Needs the built libraries, no GPU."""
import ctypes

import pytest
import torch

from tensorflow_graphics_point_clouds_amd import _lib, attention

_I32 = torch.int32


def _operands(nq=6, nk=9, heads=4, kv_heads=2, dim=8, dtype=torch.float32):
    return (torch.zeros(nq, heads, dim, dtype=dtype), torch.zeros(nk, kv_heads, dim, dtype=dtype),
            torch.zeros(nk, kv_heads, dim, dtype=dtype))


def _refuses(match, *operands, **more):
    with pytest.raises(_lib.InvalidArgumentError, match=match):
        attention.packed_attention(*(operands or _operands()), **more)


def test_attention_refuses_operands_that_do_not_fit():
    q, k, v = _operands()
    _refuses(r"\[rows, heads, channels\]", q[0], k, v)
    _refuses("value per key", q, k, v[:-1])
    _refuses("as many channels", q, k[..., :4], v[..., :4])
    _refuses("multiple of the key heads", q[:, :3], k, v)
    _refuses("multiple of the key heads", q[:, :1], k, v)
    _refuses("1 to 128 channels", *_operands(dim=129))
    _refuses("float32 or bfloat16", *_operands(dtype=torch.float16))
    _refuses("float32 or bfloat16", *_operands(dtype=torch.float64))
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
        _refuses("finite scale above 0", scale=scale)
    with pytest.raises(TypeError, match="one dtype"):
        attention.packed_attention(q, k.bfloat16(), v)
    with pytest.raises(TypeError, match="GPU tensors"):
        attention.packed_attention(q, k, v)


def test_attention_refuses_splits_masks_and_sizes_that_do_not_fit():
    splits = torch.tensor([0, 2, 6], dtype=_I32)
    _refuses("of both sides or of neither", query_splits=splits)
    _refuses(r"\[clouds \+ 1\]", query_splits=splits, key_splits=splits[:2])
    _refuses(r"\[clouds \+ 1\]", query_splits=splits[:0], key_splits=splits[:0])
    _refuses("key size per cloud", query_splits=splits, key_splits=splits, key_sizes=splits)
    _refuses("key size per cloud", key_sizes=splits[:2])
    _refuses("mask value per key", key_mask=torch.ones(8, dtype=torch.bool))


def test_attention_refuses_biases_that_do_not_fit():
    table, buckets = torch.zeros(1, 4, 4), torch.zeros(7, dtype=_I32)
    pos = lambda n, axes=1: torch.zeros(n, axes, dtype=_I32)
    _refuses("table and its buckets", bias_table=table)
    _refuses("table and its buckets", bias_buckets=buckets)
    _refuses(r"\[1 to 3 axes, buckets, heads\]", bias_table=table[..., :2], bias_buckets=buckets)
    _refuses(r"\[1 to 3 axes, buckets, heads\]", bias_table=torch.zeros(4, 4, 4), bias_buckets=buckets)
    _refuses("offsets -R to R", bias_table=table, bias_buckets=buckets[:6])
    _refuses("positions for a bias of 2 axes", bias_table=torch.zeros(2, 4, 4), bias_buckets=buckets)
    _refuses("position per row and axis", bias_table=table, bias_buckets=buckets,
             query_positions=pos(6), key_positions=pos(8))
    _refuses("position per row and axis", bias_table=table, bias_buckets=buckets,
             query_positions=pos(6, 2), key_positions=pos(9, 2))
    _refuses("positions of both sides", bias_table=table, bias_buckets=buckets, query_positions=pos(6))
    _refuses("positions of both sides", query_positions=pos(6), key_positions=pos(9))


def test_layer_norm_refuses():
    for bad in (torch.zeros(3, 4, dtype=torch.float16), torch.zeros(()), torch.zeros(3, 0)):
        with pytest.raises(_lib.InvalidArgumentError):
            attention.layer_norm(bad)
    x = torch.zeros(3, 4)
    for w, b in ((torch.ones(3), None), (None, torch.ones(1, 4)), (torch.ones(4), torch.ones(5))):
        with pytest.raises(_lib.InvalidArgumentError, match="per channel"):
            attention.layer_norm(x, w, b)
    with pytest.raises(_lib.InvalidArgumentError, match="epsilon"):
        attention.layer_norm(x, eps=-1e-5)
    with pytest.raises(TypeError, match="GPU tensors"):
        attention.layer_norm(x)


class _Description(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("dtype", "heads", "kv_heads", "dim", "clouds", "causal")] + \
        [(n, ctypes.c_int64) for n in ("num_q", "num_k")] + [(n, ctypes.c_void_p) for n in "qkv"] + \
        [(n, ctypes.c_int64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")] + \
        [(n, ctypes.c_void_p) for n in ("q_splits", "k_splits", "k_sizes", "key_mask")] + \
        [("scale", ctypes.c_float)] + [(n, ctypes.c_int) for n in ("axes", "num_buckets", "max_offset")] + \
        [(n, ctypes.c_void_p) for n in ("table", "buckets", "q_pos", "k_pos")]


def test_the_c_abi_refuses_with_a_status():
    lib = _lib.lib()
    lib.mccnn_attention_workspace_bytes.restype = ctypes.c_size_t
    lib.mccnn_attention_grads_workspace_bytes.restype = ctypes.c_size_t
    good = dict(dtype=0, heads=4, kv_heads=2, dim=64, clouds=1, num_q=10, num_k=10, q=4096, k=4096, v=4096,
                q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, scale=0.125)
    bias = dict(axes=1, num_buckets=4, max_offset=8, table=4096, buckets=4096)

    def status(message, **changes):
        d = _Description(**{**good, **changes})
        args = (None, ctypes.byref(d), None, ctypes.c_size_t(0), None, None, None, None)
        assert lib.mccnn_attention_forward(*args) == 1 and message in lib.mccnn_last_error(), lib.mccnn_last_error()
        assert lib.mccnn_attention_grads(None, ctypes.byref(d), *[None] * 6, ctypes.c_size_t(0), *[None] * 4) == 1
    status(b"type 2", dtype=2)
    status(b"128 channels", dim=129)
    status(b"128 channels", dim=0)
    status(b"multiple of the key heads", heads=3)
    status(b"multiple of the key heads", kv_heads=0)
    status(b"2^31 - 1024", num_k=2 ** 31)
    status(b"2^31 - 1024", num_q=-1)
    status(b"row splits", clouds=2)
    status(b"null tensor of queries", q=None)
    status(b"null tensor of keys", v=None)
    status(b"strides", k_row=-1)
    status(b"scale", scale=0.0)
    status(b"1 to 3 axes", axes=4)
    status(b"its table", **{**bias, "table": None})
    status(b"offsets over all axes", **{**bias, "max_offset": 672})
    status(b"offsets over all axes", **{**bias, "max_offset": -1})
    status(b"or neither", **{**bias, "q_pos": 4096})
    status(b"2 axes expects positions", **{**bias, "axes": 2})
    status(b"null output")
    one_token = _Description(**{**good, "num_q": 1, "num_k": 100000})
    need = lib.mccnn_attention_workspace_bytes(ctypes.byref(one_token))
    assert need > 0 and lib.mccnn_attention_workspace_bytes(ctypes.byref(_Description(**{**good, "dim": 0}))) == 0
    assert lib.mccnn_attention_forward(None, ctypes.byref(one_token), 4096, ctypes.c_size_t(need - 1), 4096, None,
                                       None, None) == 1 and b"workspace too small" in lib.mccnn_last_error()
    assert lib.mccnn_attention_forward(None, None, None, ctypes.c_size_t(0), None, None, None, None) == 1
    empty = _Description(**{**good, "num_q": 0, "q": None})
    assert lib.mccnn_attention_forward(None, ctypes.byref(empty), None, ctypes.c_size_t(0), *[None] * 4) == 0
    i64, f = ctypes.c_int64, ctypes.c_float
    assert lib.mccnn_layer_norm(None, 2, i64(4), 8, None, None, None, f(0), None, None, None) == 1
    assert lib.mccnn_layer_norm(None, 0, i64(4), 0, None, None, None, f(0), None, None, None) == 1
    assert lib.mccnn_layer_norm(None, 0, i64(4), 8, None, None, None, f(0), None, None, None) == 1
    assert b"null tensor" in lib.mccnn_last_error()
    assert lib.mccnn_layer_norm(None, 0, i64(4), 8, 4096, None, None, f(0), 4096, 4096, None) == 1
    assert b"or neither" in lib.mccnn_last_error()
    assert lib.mccnn_layer_norm(None, 0, i64(0), 8, None, None, None, f(0), None, None, None) == 0
    assert lib.mccnn_layer_norm_grads(None, 0, i64(4), 8, 4096, None, 4096, 4096, 4096, None,
                                      ctypes.c_size_t(0), None, 4096, 4096) == 1
    assert b"workspace" in lib.mccnn_last_error()


@pytest.mark.parametrize("buckets,most,both", [(4, 1, True), (8, 16, True), (32, 128, True), (10, 12, True),
                                               (16, 24, False), (2, 5, False), (7, 100, False), (2, 1, False)])
def test_offset_buckets(buckets, most, both):
    got = attention.offset_buckets(buckets, most, both, device="cpu")
    assert got.dtype == _I32 and len(got) == 2 * most + 1
    back = got[:most + 1].flip(0)                    # offsets 0, -1, -2, ...
    side = buckets // 2 if both else buckets
    assert back[0] == 0 and torch.all(back.diff() >= 0) and back.max() < side
    near = side // 2
    assert torch.equal(back[:near], torch.arange(near, dtype=_I32)) and back[near] == near
    assert torch.equal(got[most + 1:], back[1:] + side if both else torch.zeros(most, dtype=_I32))
    # the least offset of every wide bucket that has one, by powers of whole numbers
    wide = side - near
    for n in range(1, wide):
        first = (back == near + n).nonzero()
        if len(first):
            o = int(first[0])
            assert o ** wide >= near ** (wide - n) * most ** n > (o - 1) ** wide
    for bad in ((1, 5, both), (buckets, near - 1, both)):
        with pytest.raises(_lib.InvalidArgumentError):
            attention.offset_buckets(*bad, device="cpu")


def test_row_splits():
    from tensorflow_graphics_point_clouds_amd import pc
    cloud = pc.PointCloud(torch.zeros(9, 3), sizes=torch.tensor([4, 0, 5]))
    assert attention.row_splits(cloud).tolist() == [0, 4, 4, 9] and attention.row_splits(cloud).dtype == _I32


def test_row_splits_refuse_clouds_that_are_mixed():
    from tensorflow_graphics_point_clouds_amd import pc
    ordered = pc.PointCloud(torch.zeros(6, 3), batch_ids=torch.tensor([0, 0, 2, 2, 2, 3]), batch_size=5)
    assert ordered.get_cloud_order() is None and attention.row_splits(ordered).tolist() == [0, 2, 2, 5, 6, 6]
    mixed = pc.PointCloud(torch.zeros(6, 3), batch_ids=torch.tensor([1, 0, 1, 3, 0, 1]), batch_size=4)
    assert mixed.get_cloud_order().tolist() == [1, 4, 0, 2, 5, 3]
    with pytest.raises(_lib.InvalidArgumentError, match="cloud after cloud"):
        attention.row_splits(mixed)
    for cloud in (pc.PointCloud(torch.zeros(0, 3), batch_ids=torch.zeros(0), batch_size=2),
                  pc.PointCloud(torch.zeros(2, 4, 3), sizes=torch.tensor([4, 1]))):
        assert cloud.get_cloud_order() is None


def test_biases_of_more_offsets_than_the_kernels_hold():
    from tensorflow_graphics_point_clouds_amd import blocks
    lib = _lib.lib()
    for axes, most in ((1, 671), (2, 335), (3, 223)):
        d = dict(dtype=0, heads=4, kv_heads=2, dim=64, clouds=1, num_q=0, num_k=0, q_row=256, q_head=64, k_row=128,
                 k_head=64, v_row=128, v_head=64, scale=0.125, axes=axes, num_buckets=4, table=4096, buckets=4096)
        runs = lambda r: lib.mccnn_attention_forward(None, ctypes.byref(_Description(**d, max_offset=r)), None,
                                                     ctypes.c_size_t(0), *[None] * 4)
        assert axes * (2 * most + 1) <= attention.MAX_OFFSETS < axes * (2 * most + 3)
        assert runs(most) == 0 and runs(most + 1) == 1
        blocks.RelativeBias(4, 8, most, num_axes=axes, device="cpu")
        with pytest.raises(_lib.InvalidArgumentError, match="at most 1344 offsets over all axes"):
            blocks.RelativeBias(4, 8, most + 1, num_axes=axes, device="cpu")
        # refused with the other arguments, before anything is asked of a device
        pos = dict(query_positions=torch.zeros(6, axes, dtype=_I32), key_positions=torch.zeros(9, axes, dtype=_I32))
        _refuses("at most 1344 offsets over all axes", bias_table=torch.zeros(axes, 4, 4),
                 bias_buckets=torch.zeros(2 * most + 3, dtype=_I32), **pos)
