"""Paths through the attention kernels that ordinary inputs do not take: reference points that move while
there is something to keep, more clouds than a wavefront has lanes, other streams, captured graphs."""
import math

import pytest

torch = pytest.importorskip("torch")

from .test_gpu_attention import DTYPES, EPS, _inputs, _reference, _run, _sums, _table  # noqa: E402

pytestmark = pytest.mark.gpu


def _rising(dtype, q_sizes, k_sizes, heads, kv_heads, dim, jump):
    """Logits, in units of log 2, that rise along every cloud's keys: 64 keys on one level, then one key
    `jump` above them among 63 far below, then 64 on that key's level, and so on; rows see between a
    half and one and a half of it.  The 64 are 64 / 2^jump beside the one: a share that shows."""
    qs, ks = _sums(q_sizes), _sums(k_sizes)
    q, k, v, g = _inputs(dtype, qs[-1], ks[-1], heads, kv_heads, dim)
    level = []
    for n in k_sizes:
        j = torch.arange(n)
        tile, first = j // 64, j % 64 == 17
        up = jump * ((tile + 1) // 2).float()
        level.append(torch.where((tile % 2 == 1) & ~first, up - jump - 20.0, up) - jump * (n // 256))
    k *= 0.1
    k[..., 0] = (torch.cat(level).cuda() * math.log(2.0))[:, None].to(dtype)
    row = torch.arange(qs[-1], device="cuda")
    q[..., 0] = ((0.5 + (row % 16) / 15.0) * math.sqrt(dim))[:, None].to(dtype)
    return (q, k, v, g), qs, ks


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("jump", [5.0, 7.8, 8.2, 9.0, 12.0])
@pytest.mark.parametrize("q_sizes,k_sizes,heads,kv_heads,dim,causal", [
    ([130, 40], [700, 450], 2, 1, 32, False), ([600], [600], 2, 2, 64, True),
    ([1, 1], [2600, 1900], 4, 2, 64, False), ([50], [500], 2, 2, 128, False)])
def test_logits_that_rise_along_the_keys(dtype, jump, q_sizes, k_sizes, heads, kv_heads, dim, causal):
    """Sums and results so far are kept at the new reference point, in one part and in several."""
    from tensorflow_graphics_point_clouds_amd import attention
    inputs, qs, ks = _rising(dtype, q_sizes, k_sizes, heads, kv_heads, dim, jump)
    _run(*inputs, qs, ks, causal=causal)
    _run(*inputs, qs, ks, causal=causal, table=0.5 * _table(1, 8, heads), buckets=attention.offset_buckets(8, 30))
    gen = torch.Generator(device="cuda").manual_seed(3)
    pos = lambda n: torch.randint(0, 9, (n, 2), device="cuda", generator=gen, dtype=torch.int32)
    _run(*inputs, qs, ks, causal=causal, table=0.5 * _table(2, 8, heads), buckets=attention.offset_buckets(8, 9),
         qpos=pos(qs[-1]), kpos=pos(ks[-1]))


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("kind", ["plain", "causal", "places", "positions"])
def test_float32_results_carry_float32(dim, kind):
    """As a whole within 32 roundings: products in three parts of bfloat16 lose no more than float32 ones
    do (some ten roundings of sums of this length), while two parts, 2^-16 of every operand at most and
    2^-18 on average, would leave a hundred."""
    from tensorflow_graphics_point_clouds_amd import attention
    q, k, v, g = _inputs(torch.float32, 500, 500, 4, 2, dim)
    splits, more = [0, 70, 300, 500], {}
    if kind in ("places", "positions"):
        more = dict(table=_table(1 if kind == "places" else 2, 8, 4), buckets=attention.offset_buckets(8, 30))
    if kind == "positions":
        gen = torch.Generator(device="cuda").manual_seed(6)
        pos = torch.randint(0, 40, (500, 2), device="cuda", generator=gen, dtype=torch.int32)
        more.update(qpos=pos, kpos=pos)
    got = _run(q, k, v, g, splits, splits, causal=kind == "causal", **more)
    want = _reference(q, k, v, g, splits, splits, None, None, kind == "causal", more.get("table"),
                      more.get("buckets"), more.get("qpos"), more.get("kpos"))[0]
    for i, (x, value) in enumerate(zip(got, want)):
        assert float((x.double() - value).norm()) <= 32 * EPS * float(value.norm()), i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("clouds", [61, 62, 63, 64, 65, 200])
def test_a_token_each_for_many_requests(dtype, clouds):
    """Heads that share a block's rows, tables that are not full (some empty), a bias of token offsets,
    and rows before the first and behind the last table."""
    from tensorflow_graphics_point_clouds_amd import attention
    sizes = [(37 * b) % 90 + 3 * (b % 7 == 3) for b in range(clouds)]
    sizes[clouds // 2] = 700
    qs, ks = [3 + t for t in range(clouds + 1)], [5 + t for t in _sums(sizes)]
    inputs = _inputs(dtype, clouds + 9, ks[-1] + 11, 8, 2, 32)
    used = [n - n // 3 for n in sizes]
    _run(*inputs, qs, ks, sizes=used, causal=True)
    got = _run(*inputs, qs, ks, sizes=used, causal=True, table=_table(1, 12, 8), buckets=attention.offset_buckets(12, 40))
    assert torch.all(got[0][:3] == 0) and torch.all(got[0][3 + clouds:] == 0) and torch.all(got[2][:5] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("clouds", [62, 63, 130])
@pytest.mark.parametrize("causal", [False, True])
def test_many_ragged_clouds(dtype, clouds, causal):
    """Empty clouds, pieces of more than a block's rows, masks, and biases of both kinds with the gradient of
    their table, to which empty places add nothing."""
    from tensorflow_graphics_point_clouds_amd import attention
    sizes = [(29 * b) % 50 if b % 5 else 0 for b in range(clouds)]
    sizes[7], sizes[clouds - 2], sizes[clouds // 2] = 300, 257, 128
    s = [2 + t for t in _sums(sizes)]
    n = s[-1] + 4
    inputs = _inputs(dtype, n, n, 2, 1, 48)
    gen = torch.Generator(device="cuda").manual_seed(4)
    mask = torch.rand(n, device="cuda", generator=gen) < 0.8
    _run(*inputs, s, s, mask=mask, causal=causal)
    _run(*inputs, s, s, causal=causal, table=_table(1, 8, 2), buckets=attention.offset_buckets(8, 20))
    pos = torch.randint(0, 30, (n, 3), device="cuda", generator=gen, dtype=torch.int32)
    _run(*inputs, s, s, mask=mask, causal=causal, table=_table(3, 8, 2), buckets=attention.offset_buckets(8, 20),
         qpos=pos, kpos=pos)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_few_new_tokens_for_many_requests(dtype):
    """Causal, three query heads to a key head, two to four queries per cloud, of which some have no key."""
    clouds = 90
    q_sizes, k_sizes = [2 + b % 3 for b in range(clouds)], [(31 * b) % 150 for b in range(clouds)]
    qs, ks = _sums(q_sizes), _sums(k_sizes)
    _run(*_inputs(dtype, qs[-1], ks[-1], 6, 2, 40), qs, ks, causal=True)


def _training_call(dtype, bias):
    from tensorflow_graphics_point_clouds_amd import attention
    q, k, v, g = _inputs(dtype, 300, 300, 4, 2, 64)
    splits = torch.tensor([0, 130, 300], dtype=torch.int32, device="cuda")
    leaves, more = [t.requires_grad_() for t in (q, k, v)], {}
    if bias:
        leaves.append(_table(1, 8, 4).requires_grad_())
        more = dict(bias_table=leaves[3], bias_buckets=attention.offset_buckets(8, 30))

    def step():
        out = attention.packed_attention(*leaves[:3], splits, splits, causal=True, **more)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    return step, leaves, g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_gradients_on_another_stream_and_in_a_graph(dtype, bias):
    step, leaves, g = _training_call(dtype, bias)
    expect = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        fresh = _inputs(dtype, 300, 300, 4, 2, 64, seed=seed)
        with torch.no_grad():
            for a, b in zip([*leaves[:3], g], fresh):
                a.copy_(b)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_on_another_stream_and_in_a_graph(dtype):
    from tensorflow_graphics_point_clouds_amd import attention
    make = lambda seed: torch.randn(400, 72, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    x, g = make(0).to(dtype).requires_grad_(), make(1).to(dtype)
    w, b = (1 + 0.1 * make(2)[0]).requires_grad_(), make(3)[0].clone().requires_grad_()

    def step():
        y = attention.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), g)]
    expect = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        with torch.no_grad():
            x.copy_(make(seed + 10))
            g.copy_(make(seed + 20))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_gradient_of_a_table_beyond_32_bit_entries():
    """2^31 entries (8 GB), of which eight buckets are used: theirs as of a small table, zeros elsewhere."""
    from tensorflow_graphics_point_clouds_amd import attention
    heads, many = 128, 1 << 24
    q, k, v, g = _inputs(torch.float32, 20, 20, heads, 1, 8)
    small, buckets = _table(1, 8, heads), attention.offset_buckets(8, 9)
    last = (buckets + (many - 8)).int()              # the same buckets at the end of the large table
    grads = []
    for table, index in ((small, buckets), (torch.zeros(1, many, heads, device="cuda"), last)):
        if index is last:
            table[:, -8:] = small
        table.requires_grad_()
        out = attention.packed_attention(q, k, v, bias_table=table, bias_buckets=index)
        grads += torch.autograd.grad(out, table, g)
        del table, out
    assert torch.equal(grads[1][:, -8:], grads[0])
    assert not grads[1][:, :-8].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("places", [True, False])
def test_table_entries_that_are_no_ordinary_numbers(dtype, places):
    """NaN reaches the rows that meet its bucket (it is no mask), and no others; the largest finite value
    leaves a row the mean of the values that have it, as the lowest hides them."""
    from tensorflow_graphics_point_clouds_amd import attention
    q, k, v, g = _inputs(dtype, 90, 90, 2, 2, 32)
    buckets, table = attention.offset_buckets(8, 12), _table(1, 8, 2)
    gen = torch.Generator(device="cuda").manual_seed(5)
    pos = None if places else torch.randint(0, 20, (90, 1), device="cuda", generator=gen, dtype=torch.int32)
    offset = torch.arange(90, device="cuda")[None] - torch.arange(90, device="cuda")[:, None] if places else \
        pos[None, :, 0] - pos[:, None, 0]
    index = buckets[(offset.clamp(-12, 12) + 12).long()]
    bad = table.clone()
    bad[0, 7, 1] = math.nan
    out = attention.packed_attention(q, k, v, bias_table=bad, bias_buckets=buckets, query_positions=pos, key_positions=pos)
    met = (index == 7).any(1)
    assert met.any() and not met.all()
    assert torch.equal(torch.isnan(out[:, 1]).all(1), met) and torch.equal(torch.isnan(out[:, 1]).any(1), met)
    assert torch.isfinite(out[:, 0]).all()
    table[0, 5] = 3.4028234663852886e38
    got = _run(q, k, v, g, [0, 90], [0, 90], table=table, buckets=buckets, qpos=pos, kpos=pos)
    assert all(torch.isfinite(t).all() for t in got)


def test_a_million_small_clouds():
    """More blocks than one dimension of a grid takes: the same bits as half of the clouds at a time."""
    from tensorflow_graphics_point_clouds_amd import attention
    clouds, heads, dim = 1100000, 16, 4
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = torch.randint(0, 3, (clouds,), device="cuda", generator=gen)
    splits = torch.nn.functional.pad(sizes.cumsum(0), (1, 0)).int()
    n = int(splits[-1])
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(torch.bfloat16)
    q, k, v, g = (r(n, heads, dim) for _ in range(4))
    table, buckets = _table(1, 2, heads).requires_grad_(), attention.offset_buckets(2, 1, False)

    def call(cut, splits):
        leaves = [t[cut].detach().requires_grad_() for t in (q, k, v)] + [table]
        out = attention.packed_attention(*leaves[:3], splits, splits, bias_table=table, bias_buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, g[cut])]
    whole = call(slice(0, n), splits)
    middle = int(splits[clouds // 2])
    first = call(slice(0, middle), splits[:clouds // 2 + 1].clone())
    second = call(slice(middle, n), (splits[clouds // 2:] - middle).contiguous())
    for a, b, c in list(zip(whole, first, second))[:4]:
        assert torch.equal(a, torch.cat([b, c]))
    # (sums of one float32 number per block, added up in 64 bits)
    assert float((whole[4] - first[4] - second[4]).norm()) <= 8 * EPS * float(first[4].norm() + second[4].norm())
    alone = (sizes == 1).nonzero()[:, 0]
    rows = splits[alone].long()
    assert torch.equal(whole[0][rows], v[rows]) and torch.equal(whole[3][rows], g[rows])


@pytest.mark.parametrize("bias", ["none", "places", "positions"])
@pytest.mark.parametrize("nq,nk", [(70, 150), (1, 3000)])
def test_infinite_bfloat16_values_that_are_looked_at(bias, nq, nk):
    """Every weight is above 0: one infinity gives infinity in its channel, two of either sign NaN, and the
    other channels are what they are without."""
    from tensorflow_graphics_point_clouds_amd import attention
    q, k, v, _ = _inputs(torch.bfloat16, nq, nk, 4, 2, 24)
    more = {}
    if bias != "none":
        more = dict(bias_table=_table(1, 8, 4), bias_buckets=attention.offset_buckets(8, 30))
    if bias == "positions":
        gen = torch.Generator(device="cuda").manual_seed(7)
        pos = lambda n: torch.randint(0, 40, (n, 1), device="cuda", generator=gen, dtype=torch.int32)
        more.update(query_positions=pos(nq), key_positions=pos(nk))
    plain = attention.packed_attention(q, k, v, **more)
    v[40, :, 3], v[100, :, 5], v[7, :, 9], v[120, :, 9] = math.inf, -math.inf, math.inf, -math.inf
    for grad in (False, True):
        q.requires_grad_(grad)
        out = attention.packed_attention(q, k, v, **more).detach()
        assert torch.all(out[..., 3] == math.inf) and torch.all(out[..., 5] == -math.inf)
        assert torch.isnan(out[..., 9]).all()
        others = [c for c in range(24) if c not in (3, 5, 9)]
        assert torch.equal(out[..., others], plain[..., others])


def test_rows_without_any_cloud():
    from tensorflow_graphics_point_clouds_amd import attention
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in _inputs(torch.float32, 300, 500, 4, 2, 16)[:3]]
    out = attention.packed_attention(*leaves, none, none, causal=True)
    assert out.shape == leaves[0].shape and not out.any()
    assert not any(t.any() for t in torch.autograd.grad(out, leaves, torch.ones_like(out)))
