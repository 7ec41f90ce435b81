"""Drafted decoding over a quantised KV pool on the HIP kernels, against the
definitions in float64.

Bounds per element, from the roundings that the kernels make (u = 2^-24 is
fp32's, a bf16 rounding is off by at most 2^-8 of its value):

  tree attention   the output's rounding, 2^-8 |o|, and that of every weight
                   (with its V scale), 2^-8 of A = sum_j p_j |v_j|; fp32 scores
                   of unit normals are off by at most 2 D u sum_d |q_d k_d| <
                   1e-4, which moves a weight by as much: 2e-4 A. Products of
                   bf16 values with exactly converted codes add fp32 sums only.
                   Over codes, weights times scales below fp16's normal range are off
                   by 2^-25 where the largest scale is at least 32: 2^-30 of it.
  codes            half a step of the code at the exact quotient (e4m3: 2^-4 of
                   it, at least 2^-10; int8: 1/2) and what the fp32 value is off:
                   2^-22 of the quotient for values; for keys, whose norm sums D
                   squares and whose rotation adds two products, (D + 16) u of
                   twice the row's largest magnitude, that is
                   T (D + 16) 2^-22 in codes.
  scales           the same relative errors.
  read-back        one bf16 rounding of an fp32 product: 2^-8 + 2^-23.
  scores           a sum of up to 64 terms per thread and a tree over the rest:
                   80 u relative, twice that with the exponentials' own errors;
                   log probabilities 1e-5 + 4 u |x|, the entropy 2e-5 (1 + H).
  gradient         the probability's relative error 2e-5 + 2 u (|x| + |lse|),
                   taken as 4e-5, on p (|s| + |g_H| (|d| + H + 1)); the output's
                   rounding (eps / 2) of the result, fp32 sums 2^-22 of the parts.
"""

import math

import pytest
import torch

from tests.test_gpu_cyclic_pass import _check, _rel_l2, _setup
from tests.test_serving import TreeOracle
from white_matter_amd import (
    kv_pool,
    strict_causal_attention,
    token_log_probs,
    tree_attention,
    tree_mask_from_parents,
)
from white_matter_amd.cyclic_pass import GreedyDecoder, forward_cyclic, score_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
E4M3, INT8, BF16 = torch.float8_e4m3fn, torch.int8, torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen).to(DEV, dtype)


def _values(pool):
    return pool.codes.float().to(F64) * pool.scales.to(F64)[..., None]


# -------------------------------------------------------- quantised pool ----
def _exact_keys(key, weight, cos, sin, eps):
    x, dim = key.to(F64), key.shape[-1]
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.to(F64)[None, :, None, None]
    turned = torch.cat((-x[..., dim // 2 :], x[..., : dim // 2]), -1)
    return x * cos.to(F64)[:, None, None] + turned * sin.to(F64)[:, None, None]


def _check_rows(codes, scales, rows, off):
    """codes and scales of float64 rows, whose fp32 values are off by at most
    `off` of the row's largest magnitude."""
    top = TOP[codes.dtype]
    most = rows.abs().amax(-1)
    assert ((scales.to(F64) - most / top).abs() <= (off + 2**-22) * most / top).all()
    quotient = rows * (top / most)[..., None]
    half = torch.full_like(quotient, 0.5) if codes.dtype == INT8 else (quotient.abs() * 2**-4).clamp_min(2**-10)
    bound = half * (1 + 2 * off) + 2 * off * top + 2**-22 * quotient.abs()
    got = codes.float().to(F64)
    assert ((got - quotient).abs() <= bound).all(), ((got - quotient).abs() - bound).max().item()
    assert (got.abs() <= top).all()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize(("source", "tokens", "heads"), [(BF16, 1, 8), (BF16, 37, 3), (torch.float32, 5, 5), (torch.float32, 300, 2)])
@torch.no_grad()
def test_quantised_write(dtype, dim, source, tokens, heads):
    print(f"quantised write {dtype} D={dim} {source} T={tokens} H={heads}", flush=True)
    gen = _gen(dim + tokens)
    batch, channels, slots_n = 2, 3, 311
    key, value = (_randn(gen, channels, batch, tokens, heads, dim, dtype=source).permute(1, 0, 3, 2, 4) for _ in range(2))
    weight = (1 + 0.1 * torch.randn(channels, dim, generator=gen)).to(DEV)
    angle = torch.rand(batch, tokens, dim // 2, generator=gen).repeat(1, 1, 2).to(DEV) * 50
    cos, sin = angle.cos(), angle.sin()
    slots = torch.randperm(slots_n, generator=gen)[:tokens].to(DEV)
    keys, values = (kv_pool.quantize_pool(_randn(gen, batch, channels, heads, slots_n, dim), dtype) for _ in range(2))
    before = [t.clone() for t in (keys.codes.view(torch.uint8), keys.scales, values.codes.view(torch.uint8), values.scales)]
    kv_pool.write_pool_quantized(key, value, weight, cos, sin, keys, values, slots)
    off = (dim + 16) * 2**-23
    _check_rows(keys.codes.float().to(dtype)[:, :, :, slots], keys.scales[:, :, :, slots], _exact_keys(key, weight, cos, sin, 1e-6), off)
    _check_rows(values.codes.float().to(dtype)[:, :, :, slots], values.scales[:, :, :, slots], value.to(F64), 0.0)
    rest = torch.ones(slots_n, dtype=torch.bool, device=DEV)
    rest[slots] = False
    after = (keys.codes.view(torch.uint8), keys.scales, values.codes.view(torch.uint8), values.scales)
    for a, b in zip(after, before):
        assert torch.equal(a[:, :, :, rest], b[:, :, :, rest])  # other slots as they were


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@torch.no_grad()
def test_quantised_write_slots_per_row_and_tables(dtype):
    """Slots of each batch row's own, some outside the pool, RoPE tables by
    slot, keys alone, and pools that are views of larger ones."""
    gen, dim, tokens, slots_n = _gen(5), 64, 7, 20
    big = kv_pool.QuantizedPool.empty((2, 4, 6, slots_n, dim), dtype=dtype, device=DEV)
    keys = kv_pool.QuantizedPool(big.codes[:, 1:3, ::2], big.scales[:, 1:3, ::2])
    key = _randn(gen, 2, 2, 3, tokens, dim, dtype=torch.float32)
    weight = torch.ones(2, dim, device=DEV, dtype=BF16)
    tables = [f(torch.rand(slots_n, dim // 2, generator=gen).repeat(1, 2).to(DEV) * 9) for f in (torch.cos, torch.sin)]
    slots = torch.stack([torch.randperm(slots_n, generator=gen)[:tokens] for _ in range(2)])
    slots[0, 2], slots[1, 4] = -1, slots_n
    kv_pool.write_pool_quantized(key, None, weight, *tables, keys, None, slots.to(DEV), rope_by_slot=True)
    written = torch.zeros(2, slots_n, dtype=torch.bool)
    for b in range(2):
        for t in range(tokens):
            s = int(slots[b, t])
            if 0 <= s < slots_n:
                written[b, s] = True
                rows = _exact_keys(key[b : b + 1, :, :, t : t + 1], weight, *(x[s].expand(1, 1, dim) for x in tables), 1e-6)
                _check_rows(keys.codes.float().to(dtype)[b : b + 1, :, :, s : s + 1], keys.scales[b : b + 1, :, :, s : s + 1], rows, 80 * 2**-23)
    assert (keys.scales.permute(0, 3, 1, 2)[~written.to(DEV)] == 0).all()
    assert (big.scales[:, 0] == 0).all() and (big.scales[:, 1:3, 1::2] == 0).all()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@torch.no_grad()
def test_quantised_rows_of_extremes(dtype):
    rows = torch.randn(1, 1, 7, 2, 96, generator=_gen(3)).to(DEV)
    rows[0, 0, 0] = 0
    rows[0, 0, 1] *= 2.0**-110
    rows[0, 0, 2, :, 5] = math.inf
    rows[0, 0, 3, :, 95] = math.nan
    rows[0, 0, 4] *= 1e37
    rows[0, 0, 5, :, 1:] = 0
    pool = kv_pool.quantize_pool(rows, dtype)
    back = kv_pool.read_pool(pool)
    assert (back[0, 0, :2] == 0).all() and (pool.scales[0, 0, :2] == 0).all()
    assert back[0, 0, 2:4].isnan().all()
    _check_rows(pool.codes.float().to(dtype)[0, 0, [4, 6]], pool.scales[0, 0, [4, 6]], rows[0, 0, [4, 6]].to(F64), 0.0)
    assert (pool.codes[0, 0, 5].float()[:, 0].abs() == TOP[dtype]).all() and (back[0, 0, 5, :, 1:] == 0).all()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 96, 128])
@torch.no_grad()
def test_read_pool(dtype, dim):
    gen = _gen(dim)
    pool = kv_pool.quantize_pool(_randn(gen, 2, 3, 5, 41, dim), dtype)
    for view in (pool, kv_pool.QuantizedPool(pool.codes[:, 1:, ::2, 3:30], pool.scales[:, 1:, ::2, 3:30])):
        exact = _values(view)
        assert ((kv_pool.read_pool(view).to(F64) - exact).abs() <= (2**-8 + 2**-23) * exact.abs()).all()
        n = view.shape[3]
        slots = torch.tensor([n - 1, 0, 0, -1, 5, n])
        for given in (slots, slots.int(), torch.stack((slots, slots.flip(0)))):
            back = kv_pool.read_pool(view, given.to(DEV))
            for b in range(2):
                for t, s in enumerate((given if given.ndim == 1 else given[b]).tolist()):
                    want = kv_pool.read_pool(view)[b, :, :, s] if 0 <= s < n else torch.zeros_like(back[b, :, :, t])
                    assert torch.equal(back[b, :, :, t], want)
    assert kv_pool.read_pool(pool, torch.empty(0, dtype=torch.long, device=DEV)).shape == (2, 3, 5, 0, dim)


# -------------------------------------------------------- tree attention ----
def _tree_reference(query, key, value, lengths, tree, dummy, key_mask, scale):
    """(o, A) in float64, (B, n, H, D); key and value are the pool's values."""
    batch, heads, nodes, dim = query.shape
    group = heads // key.shape[1]
    out = torch.zeros(batch, nodes, heads, dim, dtype=F64, device=query.device)
    size = torch.zeros_like(out)
    for b in range(batch):
        base = min(max(int(lengths[b]), 0) + int(dummy), key.shape[2])
        end = min(base + nodes, key.shape[2]) if tree is not None else base
        seen = torch.ones(nodes, end, dtype=torch.bool, device=query.device)
        if tree is not None:
            seen[:, base:] = (tree if tree.ndim == 2 else tree[b])[:, : end - base]
        if key_mask is not None:
            seen &= key_mask[b, :end]
        for h in range(heads):
            k, v = key[b, h // group, :end].to(F64), value[b, h // group, :end].to(F64)
            for i in range(nodes):
                j = seen[i].nonzero()[:, 0]
                if len(j):
                    p = torch.softmax(k[j] @ query[b, h, i].to(F64) * scale, 0)
                    out[b, i, h], size[b, i, h] = p @ v[j], p @ v[j].abs()
    return out, size


def _assert_tree(out, reference, what=""):
    exact, size = reference
    assert torch.isfinite(out.float()).all(), what
    bound = 2**-8 * exact.abs() + (2**-8 + 2e-4) * size
    far = (out.to(F64) - exact).abs() - bound
    assert (far <= 0).all(), f"{what}: {far.max().item():.3e} past the bound"
    assert (out[size == 0] == 0).all(), what


def _random_tree(gen, *shape):
    parents = (torch.rand(*shape, generator=gen) * (torch.arange(shape[-1]) + 1)).long() - 1
    return tree_mask_from_parents(parents, device=DEV)[0]


def _pool_pair(gen, shape, kind):
    rows = [_randn(gen, *shape) for _ in range(2)]
    if kind == "bf16":
        return (*rows, *rows)
    pools = [kv_pool.quantize_pool(r[:, None], E4M3 if kind == "e4m3" else INT8).select(1, 0) for r in rows]
    return (*pools, *(_values(p) for p in pools))


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize(("heads", "kv_heads", "nodes"), [(4, 4, 1), (6, 2, 5), (4, 2, 13), (8, 2, 11), (10, 2, 13), (8, 2, 16), (10, 2, 16)])
@pytest.mark.parametrize("splits", [0, 1, 3])
@torch.no_grad()
def test_tree_attention(kind, dim, heads, kv_heads, nodes, splits):
    """Row tiles of 16, 32 and 64 query rows, several tiles, ragged lengths from
    nothing to the pool's end (drafted slots past it), NaN behind the last
    sequence."""
    print(f"tree {kind} D={dim} H={heads}/{kv_heads} n={nodes} splits={splits}", flush=True)
    gen = _gen(dim + 7 * nodes + heads)
    capacity, lengths = 333, torch.tensor([0, 1, 200, 330, 128])
    key, value, k, v = _pool_pair(gen, (5, kv_heads, capacity, dim), kind)
    query = _randn(gen, 5, heads, nodes, dim)
    for b in range(5):  # unused slots hold anything
        end = int(lengths[b]) + nodes
        if kind == "bf16":
            key[b, :, end:] = value[b, :, end:] = math.nan
        else:
            key.scales[b, :, end:] = value.scales[b, :, end:] = math.nan
    tree = _random_tree(gen, nodes) if nodes % 2 else _random_tree(gen, 5, nodes)
    out = tree_attention(query, key, value, kv_lengths=lengths.to(DEV), tree_mask=tree, num_splits=splits)
    assert out.shape == (5, nodes, heads, dim) and out.dtype == BF16
    _assert_tree(out, _tree_reference(query, k, v, lengths, tree, False, None, dim**-0.5), "tree")


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("nodes", [1, 9, 40])
@torch.no_grad()
def test_tree_attention_masks(kind, nodes):
    """Key masks that leave rows empty, the dummy slot, a mask that holds the
    diagonal, no tree mask, integer lengths and another scale."""
    gen, dim, capacity = _gen(nodes), 64, 150
    key, value, k, v = _pool_pair(gen, (3, 2, capacity, dim), kind)
    query = _randn(gen, 3, 4, nodes, dim)
    lengths = torch.tensor([100, -5, 40])
    mask = torch.rand(3, capacity, generator=gen).to(DEV) < 0.4
    mask[2] = False
    own = tree_mask_from_parents([-1] * nodes, include_self=True, device=DEV)[0]
    for tree in (None, own, _random_tree(gen, nodes)):
        for dummy in (False, True):
            for key_mask in (None, mask):
                out = tree_attention(query, key, value, kv_lengths=lengths.int().to(DEV), tree_mask=tree, use_dummy_token=dummy,
                                     key_mask=key_mask, softmax_scale=0.3)
                _assert_tree(out, _tree_reference(query, k, v, lengths, tree, dummy, key_mask, 0.3), f"{dummy} {key_mask is not None}")
    out = tree_attention(query, key, value, kv_lengths=77)
    _assert_tree(out, _tree_reference(query, k, v, [77] * 3, None, False, None, dim**-0.5), "integer length")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("nodes", [6, 30])
@torch.no_grad()
def test_a_bad_draft_stays_in_its_branch(kind, bad, nodes):
    """Keys and values of one drafted token that are not finite reach the
    queries that see it and no others."""
    gen, dim, length = _gen(nodes), 128, 45
    key, value, k, v = _pool_pair(gen, (2, 2, 100, dim), kind)
    query = _randn(gen, 2, 4, nodes, dim)
    tree = _random_tree(gen, 2, nodes)
    tree[:, 2:5, 1] = torch.tensor([True, False, True], device=DEV)
    clean = tree_attention(query, key, value, kv_lengths=length, tree_mask=tree)
    for side, pool in (("value", value), ("key", key)):
        slot = (slice(None), slice(None), length + 1)
        if kind == "bf16":
            kept = pool[slot].clone()
            pool[slot][..., 7] = bad
        else:
            kept = pool.scales[slot].clone()
            pool.scales[slot] = bad
        out = tree_attention(query, key, value, kv_lengths=length, tree_mask=tree)
        sees = tree[:, :, 1]
        assert torch.equal(out[~sees], clean[~sees])
        reached = ~torch.isfinite(out.float())
        if side == "value":
            assert reached[sees][..., 7].all()
            if kind == "bf16":
                assert not reached[..., :7].any() and not reached[..., 8:].any()
        elif math.isnan(bad):
            assert reached[sees].all()
        if kind == "bf16":
            pool[slot] = kept
        else:
            pool.scales[slot] = kept
    if kind == "e4m3":  # codes that stand for no number
        value.codes.view(torch.uint8)[:, :, length + 1, 9] = 0x7F
        out = tree_attention(query, key, value, kv_lengths=length, tree_mask=tree)
        assert torch.equal(out[~sees], clean[~sees]) and out[sees][..., 9].isnan().all()


@torch.no_grad()
def test_one_token_over_bf16_matches_the_decode():
    gen, lengths = _gen(8), torch.tensor([0, 17, 500])
    key, value, k, v = _pool_pair(gen, (3, 2, 501, 128), "bf16")
    query = _randn(gen, 3, 8, 1, 128)
    ours = tree_attention(query, key, value, kv_lengths=lengths.to(DEV), use_dummy_token=True)
    other = strict_causal_attention(query, key, value, query_start=lengths.to(DEV), kv_lengths=lengths.to(DEV), use_dummy_token=True)
    reference = _tree_reference(query, k, v, lengths, None, True, None, 128**-0.5)
    _assert_tree(ours, reference)
    _assert_tree(other, reference)


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
@torch.no_grad()
def test_tree_attention_layouts(kind):
    """Token-major storage, heads and slots taken as views, strided queries and
    masks, another query type, pools read on a stream of their own."""
    gen, dim = _gen(2), 64
    rows = [_randn(gen, 2, 90, 4, dim) for _ in range(2)]
    if kind == "bf16":
        key, value = (r.transpose(1, 2)[:, ::2, 5:] for r in rows)
        k, v = key, value
    else:
        pools = [kv_pool.quantize_pool(r[:, None], E4M3 if kind == "e4m3" else INT8).select(1, 0) for r in rows]  # (B, N, H, D)
        key, value = (kv_pool.QuantizedPool(p.codes.transpose(1, 2)[:, ::2, 5:], p.scales.transpose(1, 2)[:, ::2, 5:]) for p in pools)
        k, v = _values(key), _values(value)
    wide = _randn(gen, 2, 7, 6, 2 * dim, dtype=torch.float32)
    query = wide.transpose(1, 2)[:, :, :, dim:]  # (2, 6, 7, 64) views
    tree = _random_tree(gen, 2, 7).transpose(1, 2).contiguous().transpose(1, 2)
    mask = (torch.rand(85, 2, generator=gen) < 0.7).to(DEV).t()
    lengths = torch.tensor([30, 80])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = tree_attention(query, key, value, kv_lengths=lengths, tree_mask=tree, key_mask=mask)
    torch.cuda.current_stream().wait_stream(stream)
    assert out.dtype == torch.float32
    q = query.to(BF16)
    _assert_tree(out, _tree_reference(q, k, v, lengths, tree, False, mask, dim**-0.5))


@torch.no_grad()
def test_tree_attention_padded_head_dim():
    gen = _gen(4)
    key, value = (_randn(gen, 2, 2, 60, 80) for _ in range(2))
    query = _randn(gen, 2, 4, 5, 80)
    tree = _random_tree(gen, 5)
    out = tree_attention(query, key, value, kv_lengths=50, tree_mask=tree)
    _assert_tree(out, _tree_reference(query, key, value, [50, 50], tree, False, None, 80**-0.5))


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize(("batch", "heads", "kv_heads", "nodes"), [(1, 2, 1, 1), (6, 4, 2, 1), (6, 4, 2, 19), (70, 2, 1, 3), (256, 1, 1, 1), (257, 1, 1, 1)])
@pytest.mark.parametrize("capacity", [1700, 5200])
@torch.no_grad()
def test_tree_attention_deals_ragged_batches(kind, capacity, batch, heads, kv_heads, nodes):
    """Pools of one range a row, and long enough for work dealt out by the
    lengths: most rows short, some empty, few long, with and without a key mask
    that leaves ranges empty; the same launch captured, and replayed after the
    lengths have changed."""
    print(f"dealt {kind} N={capacity} B={batch} H={heads}/{kv_heads} n={nodes}", flush=True)
    gen, dim = _gen(batch + nodes), 64
    key, value, k, v = _pool_pair(gen, (batch, kv_heads, capacity, dim), kind)
    query = _randn(gen, batch, heads, nodes, dim)
    tree = _random_tree(gen, batch, nodes)
    mask = torch.rand(batch, capacity, generator=gen) < 0.5
    mask[:, 300:900] = False
    mask = mask.to(DEV)
    first = torch.randint(0, 140, (batch,), generator=gen)
    first[::3] = 0
    first[batch // 2 :: 7] = capacity - nodes
    second = first.flip(0).contiguous()
    second[-1] = 1300
    lengths = first.to(DEV)

    def run(key_mask):
        return tree_attention(query, key, value, kv_lengths=lengths, tree_mask=tree, key_mask=key_mask, softmax_scale=0.2)

    for key_mask in (None, mask):
        _assert_tree(run(key_mask), _tree_reference(query, k, v, first, tree, False, key_mask, 0.2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(None)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(None)
    for at in (second, first, second):
        lengths.copy_(at)
        graph.replay()
        eager = run(None)
        torch.cuda.synchronize()
        _assert_tree(out, _tree_reference(query, k, v, at, tree, False, None, 0.2))
        assert torch.equal(out, eager)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("nodes", [1, 20])
@pytest.mark.parametrize("capacity", [700, 2800])
@torch.no_grad()
def test_tree_attention_scales_of_any_size(kind, nodes, capacity):
    """V scales 2^16 apart, growing, falling and at random along the slots, around
    2^-60, 1 and 2^60; K scales of no size at all and of 2^-60."""
    gen = _gen(nodes + capacity)
    key, value, _, _ = _pool_pair(gen, (2, 1, capacity, 64), kind)
    query = _randn(gen, 2, 2, nodes, 64)
    lengths = torch.tensor([capacity - nodes, 333])
    tree = _random_tree(gen, nodes)
    key.scales[:, :, 100:140] = 0.0
    key.scales[:, :, 140:150] = 2.0**-60
    ramp = torch.arange(capacity) * 17 // capacity - 8
    for order in (ramp, ramp.flip(0), ramp[torch.randperm(capacity, generator=gen)]):
        for size in (-60, 0, 60):
            value.scales.copy_((2.0 ** (order + size)).float().expand(2, 1, -1))
            out = tree_attention(query, key, value, kv_lengths=lengths.to(DEV), tree_mask=tree)
            exact, total = _tree_reference(query, _values(key), _values(value), lengths, tree, False, None, 0.125)
            assert torch.isfinite(out.float()).all()
            small = capacity * 2.0**-30 * 448 * 2.0 ** (8 + size)
            far = (out.to(F64) - exact).abs() - 2**-8 * exact.abs() - (2**-8 + 2e-4) * total - small
            assert (far <= 0).all(), (kind, size, far.max().item())


@torch.no_grad()
def test_calls_on_two_streams_at_once():
    """Dealt and split attention and scores on two streams, each with workspaces of
    its own, against the same calls alone."""
    gen = _gen(21)
    key, value, _, _ = _pool_pair(gen, (3, 2, 5200, 64), "e4m3")
    lengths = torch.tensor([5100, 40, 2600], device=DEV)
    queries = [_randn(gen, 3, 4, 5, 64) for _ in range(2)]
    tree = _random_tree(gen, 5)
    logits = [_randn(gen, 7, 33001) for _ in range(2)]
    tokens = torch.randint(0, 33001, (7,), generator=gen).to(DEV)

    def calls(i):
        outs = [tree_attention(queries[i], key, value, kv_lengths=lengths, tree_mask=tree, num_splits=n) for n in (0, 3)]
        return [*outs, *token_log_probs(logits[i], tokens, top_k=5)]

    alone = [calls(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    together = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                together[i].append(calls(i))
    torch.cuda.synchronize()
    for i in range(2):
        for got in together[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))


@torch.no_grad()
def test_tree_attention_of_nothing():
    """No slots, no nodes, no rows, more key ranges than the pool has steps."""
    gen = _gen(8)
    for kind in ("bf16", "e4m3", "int8"):
        key, value, k, v = _pool_pair(gen, (2, 2, 40, 64), kind)
        cut = [kv_pool.QuantizedPool(p.codes[:, :, :0], p.scales[:, :, :0]) if kind != "bf16" else p[:, :, :0] for p in (key, value)]
        query = _randn(gen, 2, 4, 3, 64)
        own = tree_mask_from_parents([-1, 0, 0], device=DEV)[0]
        assert (tree_attention(query, *cut, kv_lengths=5, tree_mask=own) == 0).all()
        assert tree_attention(query[:, :, :0], key, value, kv_lengths=5).shape == (2, 0, 4, 64)
        assert tree_attention(query[:0], *(p.select(1, 0)[:0, None] if kind == "bf16" else kv_pool.QuantizedPool(*(t[:0] for t in p)) for p in (key, value)),
                              kv_lengths=5).shape == (0, 3, 4, 64)
        many = tree_attention(query, key, value, kv_lengths=17, tree_mask=own, num_splits=2**31 - 1)
        _assert_tree(many, _tree_reference(query, k, v, [17, 17], own, False, None, 0.125))
    pool = kv_pool.quantize_pool(_randn(gen, 1, 1, 1, 0, 96))
    assert kv_pool.read_pool(pool).shape == (1, 1, 1, 0, 96)
    scores = token_log_probs(_randn(gen, 0, 50), torch.zeros(0, dtype=torch.long, device=DEV), top_k=3)
    assert scores.log_probs.shape == (0,) and scores.top_indices.shape == (0, 3)


def test_forward_only_calls_refuse_gradients():
    """Queries, rows and scales that need a gradient, on the GPU."""
    pool = kv_pool.quantize_pool(_randn(_gen(1), 1, 1, 2, 30, 64))
    channel, rows = pool.select(1, 0), _randn(_gen(2), 1, 1, 2, 4, 64)
    query = _randn(_gen(3), 1, 2, 1, 64)
    grown = kv_pool.QuantizedPool(channel.codes, channel.scales.clone().requires_grad_())
    for args in ((query.clone().requires_grad_(), channel, channel), (query, grown, channel), (query, channel, grown)):
        with pytest.raises(RuntimeError, match="forward-only"):
            tree_attention(*args, kv_lengths=20)
    with pytest.raises(RuntimeError, match="forward-only"):
        kv_pool.quantize_pool(rows.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="forward-only"):
        kv_pool.read_pool(kv_pool.QuantizedPool(pool.codes, pool.scales.clone().requires_grad_()))


def test_tree_attention_refuses_unaligned_rows():
    """Rows of codes that do not start 16-byte aligned, before any launch."""
    whole = kv_pool.quantize_pool(_randn(_gen(1), 1, 1, 1, 40, 96)).select(1, 0)
    shifted = torch.zeros(1, 1, 30, 104, dtype=torch.uint8, device=DEV).view(E4M3)[..., 8:]
    bad = kv_pool.QuantizedPool(shifted, whole.scales[:, :, :30])
    query = _randn(_gen(2), 1, 1, 1, 96)
    for pair in ((bad, bad), (kv_pool.QuantizedPool(whole.codes[:, :, :30], bad.scales), bad)):
        with pytest.raises(RuntimeError, match="16-byte aligned"):
            tree_attention(query, *pair, kv_lengths=20)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@torch.no_grad()
def test_tree_attention_long_context(kind):
    """A context of many key ranges and a wide tree of several row tiles."""
    gen, length = _gen(6), 20011
    key, value, k, v = _pool_pair(gen, (1, 1, 20100, 64), kind)
    query = _randn(gen, 1, 2, 70, 64)
    tree = _random_tree(gen, 70)
    out = tree_attention(query, key, value, kv_lengths=length, tree_mask=tree)
    _assert_tree(out, _tree_reference(query, k, v, [length], tree, False, None, 0.125))


@torch.no_grad()
def test_tree_attention_and_write_far_offsets():
    """Batch rows 2^32 bytes apart."""
    gen, apart, dim, n = _gen(9), 1 << 32, 64, 40
    room = torch.empty(apart + n * dim, device=DEV, dtype=torch.uint8)
    codes = torch.as_strided(room.view(E4M3), (2, 1, 1, n, dim), (apart, n * dim, n * dim, dim, 1))
    pool = kv_pool.QuantizedPool(codes, torch.zeros(2, 1, 1, n, device=DEV))
    rows = _randn(gen, 2, 1, 1, n, dim)
    ones = torch.ones(1, dim, device=DEV)
    flat = torch.ones(2, n, dim, device=DEV), torch.zeros(2, n, dim, device=DEV)
    kv_pool.write_pool_quantized(rows, None, ones, *flat, pool, None, torch.arange(n, device=DEV))
    near = kv_pool.QuantizedPool.empty((2, 1, 1, n, dim), device=DEV)
    kv_pool.write_pool_quantized(rows, None, ones, *flat, near, None, torch.arange(n, device=DEV))
    assert torch.equal(kv_pool.read_pool(pool), kv_pool.read_pool(near))
    query, tree = _randn(gen, 2, 2, 4, dim), _random_tree(gen, 4)
    far, close = (tree_attention(query, p.select(1, 0), p.select(1, 0), kv_lengths=30, tree_mask=tree) for p in (pool, near))
    assert torch.equal(far, close)
    x = torch.as_strided(room.view(BF16), (2, 100), (apart // 2, 1)).normal_(generator=torch.Generator(DEV).manual_seed(1))
    tokens = torch.tensor([3, 99], device=DEV)
    for a, b in zip(token_log_probs(x, tokens, top_k=4), token_log_probs(x.contiguous(), tokens, top_k=4)):
        assert torch.equal(a, b)


@torch.no_grad()
def test_captured_step_replays():
    """A drafted step captured once (pool write, attention, scores) and replayed
    on other inputs, with eager work in between."""
    gen, dim, nodes, capacity = _gen(12), 64, 6, 400
    keys, values = (kv_pool.quantize_pool(_randn(gen, 2, 1, 2, capacity, dim)) for _ in range(2))
    query, new = _randn(gen, 2, 4, nodes, dim), _randn(gen, 2, 1, 2, nodes, dim)
    head = _randn(gen, 4 * dim, 1001)
    tokens = torch.randint(0, 1001, (2, nodes), generator=gen).to(DEV)
    weight, tree = torch.ones(1, dim, device=DEV), _random_tree(gen, nodes)
    lengths = torch.tensor([100, 30], device=DEV)
    angle = torch.rand(2, nodes, dim, generator=gen).to(DEV)

    def step():
        slots = lengths[:, None] + torch.arange(nodes, device=DEV)
        kv_pool.write_pool_quantized(new, new, weight, angle.cos(), angle.sin(), keys, values, slots)
        out = tree_attention(query, keys.select(1, 0), values.select(1, 0), kv_lengths=lengths, tree_mask=tree)
        return out, *token_log_probs(out.flatten(2) @ head, tokens, top_k=5)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        query.copy_(_randn(gen, *query.shape))
        new.copy_(_randn(gen, *new.shape))
        lengths.copy_(torch.tensor([390 - k, 7 * k], device=DEV))
        kept = [t.clone() for t in (keys.codes.view(torch.uint8), keys.scales)]
        graph.replay()
        got = [t.clone() for t in (*captured, keys.codes.view(torch.uint8), keys.scales)]
        torch.cuda.synchronize()
        keys.codes.view(torch.uint8).copy_(kept[0])
        keys.scales.copy_(kept[1])
        for a, b in zip(got, (*step(), keys.codes.view(torch.uint8), keys.scales)):
            assert torch.equal(a, b)


# ---------------------------------------------------------- token scores ----
def _scores(logits, tokens, top_k, ignore=-100):
    x = logits.to(F64)
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    lp = logp.gather(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None])[..., 0].masked_fill(tokens == ignore, 0.0)
    idx = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
    return lp, entropy, logp.gather(-1, idx), idx


def _assert_scores(got, logits, tokens, top_k):
    lp, entropy, top, idx = _scores(logits, tokens, top_k)
    size = logits.to(F64).masked_fill(logits == -math.inf, 0).abs().amax(-1)
    bound = 1e-5 + 4 * 2**-24 * size
    same = lp == got.log_probs  # (infinite ones)
    assert (((got.log_probs.to(F64) - lp).abs() <= bound) | same).all()
    assert ((got.entropy.to(F64) - entropy).abs() <= 2e-5 * (1 + entropy)).all()
    assert torch.equal(got.top_indices, idx)
    assert (((got.top_log_probs.to(F64) - top).abs() <= bound[..., None]) | (top == got.top_log_probs)).all()


DTYPES = [torch.float32, BF16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "vocab", "top_k"), [
    (1, 1, 1), (3, 7, 7), (2, 33, 32), (5, 2048, 1), (3, 8192, 5), (2, 8193, 32), (4, 16384, 20), (2, 16385, 8), (3, 50257, 0),
    (3, 151936, 32), (2, 200003, 3),
])
@torch.no_grad()
def test_token_log_probs(dtype, rows, vocab, top_k):
    print(f"scores {dtype} {rows} x {vocab} top {top_k}", flush=True)
    gen = _gen(vocab + rows)
    logits = (2.5 * torch.randn(rows, vocab, generator=gen)).to(DEV, dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(DEV)
    if rows > 2:
        tokens[1] = -100
    _assert_scores(token_log_probs(logits, tokens, top_k=top_k), logits, tokens, top_k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 9000, 40001])
@torch.no_grad()
def test_equal_logits_take_the_lowest_index(dtype, vocab):
    """Rows of one value, of two, of a ramp and its reverse, of signed zeros."""
    j = torch.arange(vocab, device=DEV)
    rows = [torch.zeros(vocab), torch.where(j.cpu() % 3 == 2, 1.5, -2.0), (j.cpu() // 7).float() / 64, -(j.cpu() // 7).float() / 64,
            torch.where(j.cpu() % 2 == 0, -0.0, 0.0), torch.where(j.cpu() == vocab - 1, 4.0, -1.0)]
    logits = torch.stack(rows).to(DEV, dtype)
    tokens = torch.full((len(rows),), vocab - 1, device=DEV)
    for top_k in (1, 8, 32):
        _assert_scores(token_log_probs(logits, tokens, top_k=top_k), logits, tokens, top_k)


@pytest.mark.parametrize("dtype", DTYPES)
@torch.no_grad()
def test_scores_of_banned_and_bad_rows(dtype):
    gen, vocab = _gen(1), 20000
    logits = torch.randn(8, vocab, generator=gen).to(DEV, dtype)
    logits[0, torch.rand(vocab, generator=gen).to(DEV) < 0.9] = -math.inf
    logits[1] = -math.inf
    logits[1, 19999] = 3.0
    logits[2] = torch.finfo(dtype).min
    logits[2, 5:9] = 1.0
    tokens = torch.tensor([int((logits[0] > -math.inf).nonzero()[3]), 19999, 6, 0, 1, 2, -1, vocab], device=DEV)
    logits[3] = -math.inf
    logits[4, 17] = math.nan
    logits[5, 18000] = math.inf
    got = token_log_probs(logits, tokens, top_k=6)
    _assert_scores(type(got)(*(t[:3] for t in got)), logits[:3], tokens[:3], 6)
    assert got.log_probs[3] == -math.inf and got.entropy[3] == 0
    assert (got.top_log_probs[3] == -math.inf).all() and got.top_indices[3].tolist() == list(range(6))
    assert got.log_probs[4:].isnan().all()  # NaN, +inf, and tokens outside the vocabulary
    assert got.entropy[4:6].isnan().all() and got.entropy[6:].isfinite().all() and got.top_log_probs[4:6].isnan().all()
    assert got.top_indices[4, 0] == 17 and got.top_indices[5, 0] == 18000
    assert got.top_log_probs[6:].isfinite().all()


def _gradient(logits, tokens, grads, top_k, ignore=-100):
    """The formula's gradient in float64, and the sizes its error bound takes."""
    x = logits.detach().to(F64)
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    finite = torch.where(p > 0, logp, 0.0)
    entropy = -(p * finite).sum(-1, keepdim=True)
    idx = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
    g_lp, g_h, g_top = (g.to(F64) for g in grads)
    g_lp = torch.where(tokens == ignore, 0.0, g_lp)
    reach = torch.zeros_like(x).scatter_add_(-1, tokens.clamp_min(0)[..., None], g_lp[..., None])
    reach = reach.scatter_add_(-1, idx, g_top)
    s = g_lp + g_top.sum(-1)
    grad = reach - p * (s[..., None] + g_h[..., None] * (finite + entropy))
    parts = g_lp.abs() + g_top.abs().sum(-1)
    size = p * (parts[..., None] + g_h.abs()[..., None] * (finite.abs() + entropy + 1))
    return grad, 4e-5 * size + 2**-22 * reach.abs().clamp_min(0) + 2**-21 * torch.where(reach != 0, parts[..., None], 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "vocab", "top_k"), [(1, 1, 0), (3, 33, 5), (2, 8193, 32), (3, 16391, 1), (2, 50257, 0), (2, 151936, 20)])
def test_token_log_probs_gradient(dtype, rows, vocab, top_k):
    print(f"score gradient {dtype} {rows} x {vocab} top {top_k}", flush=True)
    gen = _gen(vocab)
    logits = (2.5 * torch.randn(rows, vocab, generator=gen)).to(DEV, dtype)
    if vocab > 100:
        logits[0, 3:90:2] = -math.inf
    logits.requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(DEV)
    if vocab > 100:
        tokens[0] = 4
    if rows > 1 and top_k:
        tokens[1] = logits[1].argmax()  # the given token among the alternatives
    if rows > 2:
        tokens[2] = -100
    grads = [torch.randn(*s, generator=gen).to(DEV) for s in ((rows,), (rows,), (rows, top_k))]
    out = token_log_probs(logits, tokens, top_k=top_k)
    (got,) = torch.autograd.grad([out.log_probs, out.entropy, out.top_log_probs], logits, grads)
    assert got.dtype == dtype and got.shape == logits.shape
    exact, bound = _gradient(logits, tokens, grads, top_k)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # fp16's subnormal step
    far = (got.to(F64) - exact).abs() - (bound + torch.finfo(dtype).eps / 2 * exact.abs() + tiny)
    assert (far <= 0).all(), far.max().item()


def test_gradient_against_differences():
    gen = _gen(11)
    x = torch.randn(3, 50, generator=gen).to(DEV).requires_grad_()
    tokens = torch.tensor([4, 49, 0], device=DEV)
    w = [torch.randn(*s, generator=gen).to(DEV) for s in ((3,), (3,), (3, 4))]

    def loss(y):
        out = token_log_probs(y, tokens, top_k=4)
        return sum((a * b).sum() for a, b in zip((out.log_probs, out.entropy, out.top_log_probs), w))

    (grad,) = torch.autograd.grad(loss(x), x)
    # central differences in float64 of the formula: step 1e-5, error 1e-9
    def exact(y):
        lp, h, top, _ = _scores(y, tokens, 4)
        return sum((a * b.to(F64)).sum() for a, b in zip((lp, h, top), w))

    base = x.detach().to(F64)
    for r in range(3):
        for j in range(0, 50, 7):
            step = torch.zeros_like(base)
            step[r, j] = 1e-5
            slope = (exact(base + step) - exact(base - step)) / 2e-5
            assert abs(grad[r, j].item() - slope.item()) <= 1e-4


def test_gradient_of_some_outputs_and_layouts():
    """Only some outputs used, leading dimensions, strided rows, a row that holds
    nothing, a double backward refused, no gradient of ignored rows."""
    gen = _gen(13)
    wide = torch.randn(2, 3, 1003, generator=gen).to(DEV).requires_grad_()
    tokens = torch.randint(0, 1000, (2, 3), generator=gen).to(DEV)
    tokens[1, 2] = -7
    for use in range(3):
        logits = wide[:, :, 3:]
        out = token_log_probs(logits, tokens.int(), top_k=2, ignore_index=-7)
        (got,) = torch.autograd.grad(out[use].sum(), wide)
        grads = [torch.zeros_like(out[i]) for i in range(3)]
        grads[use] += 1
        exact, bound = _gradient(logits, tokens, grads, 2, ignore=-7)
        assert ((got[:, :, 3:].to(F64) - exact).abs() <= bound + 2**-23 * exact.abs()).all()
        assert (got[:, :, :3] == 0).all()
        if use == 0:
            assert (got[1, 2] == 0).all()
    empty = torch.full((1, 77), -math.inf, device=DEV, requires_grad=True)
    out = token_log_probs(empty, torch.tensor([3], device=DEV), top_k=1)
    (got,) = torch.autograd.grad([out.log_probs.sum() + out.entropy.sum() + out.top_log_probs.sum()], empty)
    assert (got == 0).all()
    out = token_log_probs(wide, tokens, ignore_index=-7)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.log_probs.sum(), wide, create_graph=True)
    assert token_log_probs(wide[:0], tokens[:0], top_k=2).top_indices.shape == (0, 3, 2)


def test_captured_gradient_replays():
    gen, vocab = _gen(14), 9001
    logits = torch.randn(4, vocab, generator=gen).to(DEV, BF16)
    tokens = torch.randint(0, vocab, (4,), generator=gen).to(DEV)

    def step():
        x = logits.detach().requires_grad_()
        out = token_log_probs(x, tokens, top_k=3)
        return (*out[:3], *torch.autograd.grad(out.log_probs.sum() - 0.1 * out.entropy.sum() + out.top_log_probs.sum(), x))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        logits.copy_(torch.randn(4, vocab, generator=gen).to(DEV, BF16))
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_compiled_calls():
    """The operators trace whole under torch.compile."""
    gen = _gen(15)
    key, value = (kv_pool.quantize_pool(_randn(gen, 1, 1, 2, 64, 64)) for _ in range(2))
    query, tree = _randn(gen, 1, 4, 3, 64), _random_tree(gen, 3)
    tokens = torch.tensor([[1, 2, 3]], device=DEV)

    def step(q):
        out = tree_attention(q, key.select(1, 0), value.select(1, 0), kv_lengths=20, tree_mask=tree)
        back = kv_pool.read_pool(key)
        return token_log_probs(out.flatten(2), tokens, top_k=2), back * 2

    with torch.no_grad():
        eager, compiled = step(query), torch.compile(step, fullgraph=True, backend="aot_eager")(query)
    for a, b in zip((*eager[0], eager[1]), (*compiled[0], compiled[1])):
        assert torch.equal(a, b)


# ------------------------------------------------------- drafted decoding ----
def _pool_oracle(dtype):
    """The oracle's kernel set over pools of values: stored rows are rounded to
    the grid of a quantised pool's codes (dtype None: left as they are)."""

    class Rounded(TreeOracle):
        @staticmethod
        def store(key, value, weight, cos, sin, keys, values, slots, *, eps):
            TreeOracle.store(key, value, weight, cos, sin, keys, values, slots, eps=eps)
            for pool in (keys, values) if dtype else ():
                rows = pool[..., slots, :].double()
                scale = rows.abs().amax(-1, keepdim=True) / TOP[dtype]
                x = rows / torch.where(scale > 0, scale, 1.0)
                x = x.round() if dtype == INT8 else x.float().to(dtype).double()
                pool[..., slots, :] = (x * scale).to(pool.dtype)

    return Rounded


def _check_stored(hip, ref, exact, dtype, what):
    """`_check` for pool rows. Where two runs' rows lie on two sides of the
    middle between codes they are stored one step apart, whose largest size is
    32 of a row's 448 (e4m3, top binade) or 1 of its 127: a row's largest
    magnitude times that, past the bf16 bar, is the most they differ by."""
    if dtype is None:
        return _check(hip, ref, exact, what)
    r_hip, m_hip, scale = _rel_l2(hip, exact)
    r_ref, _, _ = _rel_l2(ref, exact)
    print(f"{what}: rel_l2 hip {r_hip:.3e} bf16-oracle {r_ref:.3e}, max_abs hip {m_hip:.3e}", flush=True)
    assert r_hip <= 1.5 * r_ref + 1e-6, f"{what}: HIP rel_l2 {r_hip:.3e} vs bf16 oracle run {r_ref:.3e}"
    assert m_hip <= 1e-2 * max(1.0, scale) + scale * (1 / 127 if dtype == INT8 else 32 / 448), f"{what}: max_abs {m_hip:.3e}"


@pytest.mark.parametrize("dtype", [None, E4M3, INT8])
@torch.no_grad()
def test_prefill_decode_and_drafts_run_together(dtype):
    """A prefill's pool quantised, decoded from (captured and eager), and a tree
    of drafts run behind it and scored. Against the same weights in float32 over
    the oracle, the kernels' error is at most 1.5 times that of the bf16 model
    over the oracle, both over rows rounded to the same grid."""
    model, exact, ids, docs = _setup()
    steps, parents = 3, [-1, 0, 0, 1, -1, 4, 3, 2, 2]
    nodes, used = len(parents), ids.shape[1] + 1
    capacity = used + steps + nodes
    hidden, keys, values, positions = forward_cyclic(model, ids, docs, capacity=capacity)
    if dtype is None:
        pools, rows = (keys, values), (keys, values)
    else:
        pools = tuple(kv_pool.quantize_pool(t, dtype) for t in (keys, values))
        rows = tuple(_values(p) for p in pools)

    def copy(pool):
        return pool.clone() if dtype is None else kv_pool.QuantizedPool(*(t.clone() for t in pool))

    def read(pool):
        return kv_pool.read_pool(pool) if dtype else pool

    oracle = _pool_oracle(dtype)
    h = hidden.float()
    hip = GreedyDecoder.after_prefill(model, h, *(copy(p) for p in pools), positions, docs)
    eager = GreedyDecoder.after_prefill(model, h, *(copy(p) for p in pools), positions, docs, capture=False)
    ref = GreedyDecoder.after_prefill(model, h, *(r.bfloat16() for r in rows), positions, docs, kernels=oracle, capture=False)
    full = GreedyDecoder.after_prefill(exact, h, *(r.float() for r in rows), positions, docs, kernels=oracle, capture=False)
    for step in range(steps):
        for other in (eager, ref, full):
            other.token.copy_(hip.token)
        for decoder in (hip, eager, ref, full):
            decoder()
        torch.cuda.synchronize()
        for name in ("keys", "values"):
            got, same, want, best = (getattr(d, name) for d in (hip, eager, ref, full))
            got, same = read(got), read(same)
            at = used + step
            assert torch.equal(got, same), "graph replay and eager launches must store the same token"
            _check_stored(got[..., at, :], want[..., at, :], best[..., at, :], dtype, f"{dtype} step {step} {name}")

    drafts = torch.randint(0, 96, (2, nodes), generator=_gen(3)).to(DEV)
    context = h[:, -1:]
    results = []
    for m, d, kernels in ((model, hip, None), (model, ref, oracle), (exact, full, oracle)):
        more = {} if kernels is None else dict(kernels=kernels)
        out, scores = score_drafts(
            m, drafts, parents, context, d.keys, d.values, used + steps, d.position, d.key_mask, top_k=4, **more,
        )
        results.append((out, scores.log_probs, scores.top_log_probs, *(read(p) if kernels is None else p for p in (d.keys, d.values))))
    torch.cuda.synchronize()
    names = ("outputs", "log probabilities", "alternatives", "keys", "values")
    for name, got, want, best in zip(names, *results):
        if name in ("keys", "values"):
            got, want, best = (t[..., used + steps :, :] for t in (got, want, best))
            _check_stored(got, want, best, dtype, f"{dtype} drafts' {name}")
        else:
            _check(got, want, best, f"{dtype} drafts' {name}")
    # committed rows are left as they were
    for pool, start in zip((hip.keys, hip.values), (eager.keys, eager.values)):
        for a, b in zip((pool,) if dtype is None else pool, (start,) if dtype is None else start):
            slots = 3 if dtype is None or a.ndim == 5 else -1
            assert torch.equal(a.narrow(slots, 0, used + steps).float(), b.narrow(slots, 0, used + steps).float())


@torch.no_grad()
def test_a_drafted_chain_matches_decoding():
    """The kernels' own decoding of a chain, one token at a time, and the chain
    as one tree: the pool rows agree to a bf16 model's noise (2^-6 relative in
    the L2 norm, over 4 bf16 roundings a layer and 3 layers), the scores too."""
    model, _, ids, docs = _setup()
    nodes, used = 4, ids.shape[1] + 1
    hidden, *bf16, positions = forward_cyclic(model, ids, docs, capacity=used + nodes)
    pools = [kv_pool.quantize_pool(t) for t in bf16]
    decoder = GreedyDecoder.after_prefill(model, hidden, *(kv_pool.QuantizedPool(*(t.clone() for t in p)) for p in pools), positions, docs)
    keep, tokens = decoder.key_mask.clone(), []
    for _ in range(nodes):
        tokens.append(decoder.token.clone())
        decoder()
    drafts = torch.cat(tokens, 1)
    _, scores = score_drafts(model, drafts, [-1, 0, 1, 2], hidden[:, -1:], *pools, used, positions[:, -1:] + 1, keep, top_k=1)
    for pool, alone in zip(pools, (decoder.keys, decoder.values)):
        got, want = (_values(p)[..., used:, :] for p in (pool, alone))
        assert float((got - want).norm() / want.norm()) < 2**-6
    # greedy drafts are the top alternative of the rows above them, up to that noise
    assert (scores.log_probs - scores.top_log_probs[..., 0] >= -0.02).all()
