"""Drafted decoding over a quantised pool on the CPU: the portable paths
against loops in float64, and what each entry point refuses (before anything
reaches a GPU)."""

import ctypes
import math

import pytest
import torch

from tests.test_cyclic_pass import OracleKernels, _model
from white_matter_amd import _native, kv_pool, token_log_probs, tree_attention, tree_mask_from_parents
from white_matter_amd.cyclic_pass import GreedyDecoder, forward_cyclic, score_drafts

F64 = torch.float64


def _pool(batch=2, channels=1, heads=2, slots=12, dim=64, dtype=torch.float8_e4m3fn):
    return kv_pool.QuantizedPool.empty((batch, channels, heads, slots, dim), dtype=dtype, device="cpu")


# -------------------------------------------------------------- tree masks ----
def test_tree_mask_from_parents():
    parents = torch.tensor([[-1, 0, 0, 1, 3], [-1, -1, 1, -1, 2]])
    mask, depths = tree_mask_from_parents(parents)
    for b in range(2):
        for i in range(5):
            path, p = [], int(parents[b, i])
            while p >= 0:
                path.append(p)
                p = int(parents[b, p])
            assert mask[b, i].nonzero()[:, 0].tolist() == sorted(path) and depths[b, i] == len(path)
    own, _ = tree_mask_from_parents([-1, 0], include_self=True)
    assert own.tolist() == [[True, False], [True, True]]
    assert tree_mask_from_parents([])[0].shape == (0, 0)
    assert tree_mask_from_parents(torch.tensor([-1, 0], dtype=torch.int32))[1].tolist() == [0, 1]
    for bad in ([0], [-1, 1], [-1, -2], [-1, 0, 5]):
        with pytest.raises(ValueError, match="earlier node"):
            tree_mask_from_parents(bad)
    with pytest.raises(ValueError, match="integer"):
        tree_mask_from_parents(torch.tensor([-1.0]))


# -------------------------------------------------------- portable results ----
@pytest.mark.parametrize("quantised", [False, True])
def test_tree_attention_portable(quantised):
    gen = torch.Generator().manual_seed(3)
    batch, heads, kv_heads, nodes, slots, dim = 3, 4, 2, 5, 20, 64
    query = torch.randn(batch, heads, nodes, dim, generator=gen)
    rows = [torch.randn(batch, kv_heads, slots, dim, generator=gen) for _ in range(2)]
    if quantised:
        pools = []
        for r in rows:
            scales = r.abs().amax(-1) / 127
            pools.append(kv_pool.QuantizedPool((r / scales[..., None]).round().to(torch.int8), scales))
        key, value = pools
        rows = [p.codes.double() * p.scales.double()[..., None] for p in pools]
    else:
        key, value = rows
    tree, _ = tree_mask_from_parents([-1, 0, 0, 1, -1])
    lengths = torch.tensor([7, 0, 18])
    key_mask = torch.rand(batch, slots, generator=gen) < 0.6
    key_mask[1] = False
    for dummy in (False, True):
        for mask in (None, key_mask):
            out = tree_attention(query, key, value, kv_lengths=lengths, tree_mask=tree, use_dummy_token=dummy, key_mask=mask)
            assert out.shape == (batch, nodes, heads, dim)
            for b in range(batch):
                base = int(lengths[b]) + dummy
                for i in range(nodes):
                    seen = [j for j in range(slots) if (j < base or (j - base < nodes and tree[i, j - base])) and (mask is None or mask[b, j])]
                    for h in range(heads):
                        k, v = (r[b, h // 2, seen].double() for r in rows)
                        want = torch.softmax(k @ query[b, h, i].double() * dim**-0.5, 0) @ v if seen else torch.zeros(dim, dtype=F64)
                        assert (out[b, i, h] - want).abs().max() < 1e-5  # fp32 sums of 20 unit normals
    value_rows = value.scales if quantised else value
    value_rows[0, :, 8] = math.inf  # drafted slot 1 of row 0 (dummy off: slot 7 + 1)
    out = tree_attention(query, key, value, kv_lengths=lengths, tree_mask=tree)
    assert out[0, [0, 1, 2, 4]].isfinite().all() and not out[0, 3].isfinite().all()


def test_token_log_probs_portable():
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(2, 4, 30, generator=gen, dtype=torch.float32)
    x[0, 1, 3:] = -math.inf
    x[1, 0] = -math.inf
    tokens = torch.tensor([[0, 2, -100, 29], [5, 30, -1, 7]])
    out = token_log_probs(x, tokens, top_k=3)
    for r in range(2):
        for c in range(4):
            row, t = x[r, c].double(), int(tokens[r, c])
            if (r, c) == (1, 0):
                assert out.log_probs[r, c] == -math.inf and out.entropy[r, c] == 0 and out.top_indices[r, c].tolist() == [0, 1, 2]
                continue
            logp = row - torch.logsumexp(row, 0)
            p = logp.exp()
            assert abs(out.entropy[r, c].item() + (p * logp.masked_fill(p == 0, 0)).sum().item()) < 1e-5
            best = sorted(range(30), key=lambda j: (-row[j].item(), j))[:3]
            assert out.top_indices[r, c].tolist() == best
            assert (out.top_log_probs[r, c].double() - logp[best]).abs().max() < 1e-5
            if t == -100:
                assert out.log_probs[r, c] == 0
            elif 0 <= t < 30:
                assert abs(out.log_probs[r, c].item() - logp[t].item()) < 1e-5
            else:
                assert math.isnan(out.log_probs[r, c].item())


def test_token_log_probs_portable_gradient():
    x = torch.randn(3, 12, generator=torch.Generator().manual_seed(5), dtype=torch.float64).float().requires_grad_()
    out = token_log_probs(x, torch.tensor([1, -100, 11]), top_k=2)
    (grad,) = torch.autograd.grad(out.log_probs.sum() + 0.5 * out.entropy.sum() + out.top_log_probs[:, 1].sum(), x)
    y = x.detach().double().requires_grad_()
    logp = torch.log_softmax(y, -1)
    loss = logp[0, 1] + logp[2, 11] - 0.5 * (logp.exp() * logp).sum() + logp.sort(-1, descending=True).values[:, 1].sum()
    assert (grad.double() - torch.autograd.grad(loss, y)[0]).abs().max() < 1e-5


# ----------------------------------------------------------------- refusals ----
def test_tree_attention_refusals():
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 9, 64)
    pool = _pool().select(1, 0)
    ok = dict(kv_lengths=4)
    bad = [
        (q, k, k, dict(kv_lengths=4, backend="cuda"), "backend"),
        (q, k, k, dict(kv_lengths=4, use_dummy_token=1), "use_dummy_token"),
        (q, k, pool, ok, "both"),
        (q, pool, k, ok, "both"),
        (q[0], k, k, ok, "tensors"),
        (q, k, k[:, :, :5], ok, "matching"),
        (q[:1], k, k, ok, "batch"),
        (q[..., :32], k, k, ok, "head_dim"),
        (q[:, :3], k, k, ok, "divisible"),
        (q.long(), k, k, ok, "floating"),
        (q, k, k, dict(kv_lengths=4.0), "kv_lengths"),
        (q, k, k, dict(kv_lengths=torch.zeros(2)), "kv_lengths"),
        (q, k, k, dict(kv_lengths=torch.zeros(3, dtype=torch.long)), "kv_lengths"),
        (q, k, k, dict(kv_lengths=4, tree_mask=torch.zeros(3, 3)), "tree_mask"),
        (q, k, k, dict(kv_lengths=4, tree_mask=torch.zeros(3, 2, dtype=torch.bool)), "tree_mask"),
        (q, k, k, dict(kv_lengths=4, key_mask=torch.zeros(2, 8, dtype=torch.bool)), "key_mask"),
        (q, k, k, dict(kv_lengths=4, num_splits=-1), "num_splits"),
        (q, k[:, :, :0], k[:, :, :0], dict(kv_lengths=0, use_dummy_token=True), "dummy"),
        (q, k, k, dict(kv_lengths=4, backend="hip"), "GPU"),
        (q, kv_pool.QuantizedPool(k.to(torch.int8), torch.zeros(2, 2, 8)), pool, ok, "scales"),
        (q, kv_pool.QuantizedPool(k.half(), torch.zeros(2, 2, 9)), pool, ok, "int8"),
        (q, pool, _pool(dtype=torch.int8).select(1, 0), ok, "one type"),
    ]
    for query, key, value, options, message in bad:
        with pytest.raises(ValueError, match=message):
            tree_attention(query, key, value, **options)
    with pytest.raises(RuntimeError, match="forward-only"):
        tree_attention(q.clone().requires_grad_(), k, k, kv_lengths=4)


def test_pool_refusals():
    pool, gen = _pool(), torch.Generator().manual_seed(0)
    key = torch.randn(2, 1, 2, 3, 64, generator=gen)
    weight, cos, slots = torch.ones(1, 64), torch.ones(2, 3, 64), torch.tensor([1, 4, 2])

    def write(key=key, value=None, weight=weight, cos=cos, sin=None, keys=pool, values=None, slots=slots, **options):
        kv_pool.write_pool_quantized(key, value, weight, cos, cos if sin is None else sin, keys, values, slots, **options)

    for arguments, kind, message in [
        (dict(key=key[0]), ValueError, "of one shape"),
        (dict(value=key[:, :, :, :2]), ValueError, "of one shape"),
        (dict(key=key.half()), TypeError, "float32 or bfloat16"),
        (dict(value=key), ValueError, "exactly when"),
        (dict(values=pool), ValueError, "exactly when"),
        (dict(keys=key), TypeError, "QuantizedPool"),
        (dict(keys=_pool(heads=3)), ValueError, "B, C, H, N, D"),
        (dict(value=key, values=_pool(dtype=torch.int8)), ValueError, "code type"),
        (dict(weight=torch.ones(2, 64)), ValueError, "k_norm_weight"),
        (dict(cos=torch.ones(2, 4, 64)), ValueError, "cos and sin"),
        (dict(sin=torch.ones(2, 3, 64, dtype=torch.bfloat16)), ValueError, "cos and sin"),
        (dict(rope_by_slot=True), ValueError, "tables"),
        (dict(slots=slots[:2]), ValueError, "slots"),
        (dict(slots=slots.float()), ValueError, "slots"),
        (dict(slots=slots.expand(3, 3)), ValueError, "slots"),
        (dict(), RuntimeError, "GPU"),
    ]:
        with pytest.raises(kind, match=message):
            write(**arguments)
    with pytest.raises(RuntimeError, match="forward-only"):
        write(key=key.clone().requires_grad_())
    wide = _pool(dim=128)
    with pytest.raises(ValueError, match="unit stride"):
        kv_pool.read_pool(kv_pool.QuantizedPool(wide.codes[..., ::2], wide.scales))
    for shape, message in (((2, 1, 2, 3, 80), "head_dim"), ((2, 2, 3, 64), "B, C, H, T, D")):
        with pytest.raises(ValueError, match=message):
            kv_pool.quantize_pool(torch.zeros(shape))
    with pytest.raises(ValueError, match="codes"):
        kv_pool.quantize_pool(key, torch.float16)
    with pytest.raises(ValueError, match="codes"):
        kv_pool.QuantizedPool.empty((1, 1, 1, 4, 64), dtype=torch.bfloat16, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        kv_pool.read_pool(pool, torch.zeros(3, 5, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU"):
        kv_pool.read_pool(pool)
    with pytest.raises(ValueError, match="before the slots"):
        pool.select(3, 0)


def test_token_log_probs_refusals():
    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.long)
    for logits, tokens, options, kind, message in [
        (x.double(), t, {}, TypeError, "float32"),
        (x.long(), t, {}, TypeError, "float32"),
        (x, t[:2], {}, ValueError, "one per row"),
        (x, t.float(), {}, ValueError, "integer"),
        (x, t, dict(top_k=11), ValueError, "top_k"),
        (x, t, dict(top_k=-1), ValueError, "top_k"),
        (torch.zeros(3, 100), t, dict(top_k=33), ValueError, "top_k"),
        (x[:, :0], t, {}, ValueError, "0 logits"),
    ]:
        with pytest.raises(kind, match=message):
            token_log_probs(logits, tokens, **options)


def test_c_entry_points_refuse_before_launching():
    """NULL and inconsistent arguments of the C ABI (zeroed structs of a size
    that holds every field)."""
    lib = _native.load()
    for name in ("wmx_kv_quant_store", "wmx_kv_quant_read", "wmx_tree_attn", "wmx_score", "wmx_score_bwd"):
        entry = getattr(lib, name)
        entry.argtypes, entry.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        assert entry(None, None) == -1 and b"NULL" in lib.wmx_last_error()
        zeros = ctypes.create_string_buffer(1024)
        assert entry(zeros, None) in (-1, -2) and lib.wmx_last_error()
    for name in ("wmx_tree_workspace_size", "wmx_score_workspace_size"):
        entry = getattr(lib, name)
        entry.argtypes, entry.restype = [ctypes.c_void_p], ctypes.c_int64
        assert entry(None) == 0 and entry(ctypes.create_string_buffer(1024)) == 0


# ---------------------------------------------------------- drafted decoding ----
class TreeOracle(OracleKernels):
    @staticmethod
    def tree(q, k, v, *, lengths, tree_mask, use_dummy_token, key_mask):
        return tree_attention(
            q.cpu(), k.cpu(), v.cpu(), kv_lengths=lengths.cpu(), tree_mask=tree_mask.cpu(), use_dummy_token=use_dummy_token,
            key_mask=None if key_mask is None else key_mask.cpu(), backend="reference",
        ).to(q.device, q.dtype)


@pytest.mark.parametrize("dummy", [True, False])
@pytest.mark.parametrize("documents", [True, False])
def test_drafted_paths_match_decoding(dummy, documents):
    """Every node of a drafted tree has the output, the pool rows and the score
    that decoding its path one token at a time gives, in float64 to the portable
    path's float32 scores and weights (2^-24 on sums of up to 40 terms each)."""
    torch.manual_seed(4)
    length, parents = 12, [-1, 0, 0, 1, -1, 4, 3]
    nodes, offset = len(parents), int(dummy)
    model = _model(length, use_dummy_token=dummy)
    ids = torch.randint(0, 50, (2, length))
    docs = torch.tensor([[0] * 5 + [1] * 7, [0] * 9 + [1] * 3]) if documents else None
    capacity = length + offset + nodes + 1
    hidden, keys, values, positions = forward_cyclic(model, ids, docs, capacity=capacity, kernels=OracleKernels)
    keep = torch.zeros(2, capacity, dtype=torch.bool)
    keep[:, offset : length + offset] = True if docs is None else docs == docs[:, -1:]
    keep[:, 0] |= dummy
    drafts = torch.randint(0, 50, (2, nodes))
    drafted = [t.clone() for t in (keys, values)]
    out, scores = score_drafts(
        model, drafts, parents, hidden[:, -1:], *drafted, length + offset, positions[:, -1:] + 1, keep, top_k=3, kernels=TreeOracle,
    )
    assert out.shape == (2, nodes, 32) and scores.top_indices.shape == (2, nodes, 3)
    bound = dict(rtol=2e-5, atol=2e-6)
    for node in range(nodes):
        path = [node]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        decoder = GreedyDecoder(
            model, keys.clone(), values.clone(), length + offset, positions[:, -1:] + 1, drafts[:, :1], keep,
            kernels=OracleKernels, capture=False,
        )
        logits = model.logits(hidden[:, -1:])
        for step, i in enumerate(path):
            want = torch.log_softmax(logits[:, 0], -1)
            decoder.token.copy_(drafts[:, i : i + 1])
            decoder()
            at = length + offset + step
            for got, alone in zip(drafted, (decoder.keys, decoder.values)):
                assert torch.allclose(got[..., length + offset + i, :], alone[..., at, :], **bound)
            logits = model.logits(out[:, i : i + 1])
        given = want.gather(1, drafts[:, node : node + 1])[:, 0]
        assert torch.allclose(scores.log_probs[:, node].double(), given, rtol=0, atol=2e-5)
        assert torch.allclose(scores.entropy[:, node].double(), -(want.exp() * want).sum(-1), rtol=0, atol=2e-4)
        assert torch.allclose(scores.top_log_probs[:, node].double(), want.topk(3)[0], rtol=0, atol=2e-5)
    with pytest.raises(ValueError, match="free slot"):
        score_drafts(model, drafts, parents, hidden[:, -1:], *drafted, capacity - nodes + 1, positions[:, -1:], kernels=TreeOracle)
    with pytest.raises(ValueError, match="context"):
        score_drafts(model, drafts, parents, hidden, *drafted, length + offset, positions[:, -1:], kernels=TreeOracle)
    none, empty = score_drafts(model, drafts[:, :0], [], hidden[:, -1:], *drafted, length + offset, positions[:, -1:], kernels=TreeOracle)
    assert none.shape == (2, 0, 32) and empty.log_probs.shape == (2, 0)
