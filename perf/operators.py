"""The operators of drafted decoding over a quantised KV pool, for measuring
them: their plain forms and the calls that a program makes of this package.

  tree        attention of a tree of drafted tokens, or of one token per row,
              over a bf16, float8 or int8 pool (tree_attention)
  write       keys (norm, RoPE) and values quantised into pool slots as they
              are written (kv_pool.write_pool_quantized)
  read        pool slots read back as bf16 rows (kv_pool.read_pool)
  write_read  a token group written into the pool, then the filled prefix read
              back for a prefill over it
  score       log probabilities of given tokens, the entropy and the top
              alternatives of each row of logits (token_log_probs)
  score_grad  the same with the gradient of the logits

Queries, keys, values and gradients are unit normals, as after the norms of a
model; logits have the spread of a trained head's (standard deviation 2.5).
"""

from __future__ import annotations

import math

import torch

own = False

if torch.cuda.is_available():
    DEV = "cuda"
else:
    DEV = "cpu"
F32, F64, BF16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn
DTYPES = {"bf16": BF16, "f32": F32, "e4m3": E4M3, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}  # largest code magnitude
SMALLEST = 2.0**-100  # rows whose magnitudes stay below it are stored as zeros


# ------------------------------------------------------------------ cases ----
def listed() -> list[dict]:
    return [
        # one interactive request: its next token over a short float8 context
        dict(name="decode_one", kind="tree", pool="e4m3", batch=1, heads=16, kv_heads=8, dim=64, capacity=1153, nodes=1,
             dummy=True, masked=False),
        # a serving batch over long ragged contexts, one token per row
        dict(name="decode_batch", kind="tree", pool="e4m3", batch=32, heads=16, kv_heads=8, dim=128, capacity=8192, nodes=1,
             dummy=False, masked=False),
        # a small tree of drafted tokens for a few requests, unquantised pool
        dict(name="tree_bf16", kind="tree", pool="bf16", batch=4, heads=16, kv_heads=8, dim=128, capacity=4096, nodes=13,
             dummy=True, masked=False),
        # a wide tree over int8 contexts of packed documents, odd sizes
        dict(name="tree_int8", kind="tree", pool="int8", batch=7, heads=12, kv_heads=6, dim=96, capacity=2049, nodes=37,
             dummy=True, masked=True),
        # the widest tree over the longest contexts (the most arithmetic)
        dict(name="tree_wide", kind="tree", pool="e4m3", batch=16, heads=16, kv_heads=8, dim=128, capacity=8192, nodes=64,
             dummy=False, masked=False),
        # the pool write of a decode step: one token of every row
        dict(name="write_step", kind="write", pool="e4m3", batch=8, channels=8, kv_heads=8, dim=64, tokens=1, capacity=1153,
             key="bf16"),
        # the pool write of one token group of a prefill
        dict(name="write_group", kind="write", pool="e4m3", batch=8, channels=8, kv_heads=16, dim=64, tokens=2048, capacity=2049,
             key="bf16"),
        # a decoded context read back whole for a prefill over it
        dict(name="read_context", kind="read", pool="e4m3", batch=4, channels=8, kv_heads=8, dim=128, capacity=4096),
        # a short float32 group into an int8 pool, then its prefix back: odd sizes
        dict(name="write_read", kind="write_read", pool="int8", batch=3, channels=4, kv_heads=6, dim=96, tokens=251,
             capacity=1021, key="f32"),
        # the drafted tokens of a batch scored, with the alternatives that a sampler looks at
        dict(name="score_draft", kind="score", logits="bf16", rows=37, vocab=151936, top_k=8, banned=False, padded=False),
        # one layer of training on given tokens: log probabilities and entropy, and their gradient
        dict(name="score_train", kind="score_grad", logits="bf16", rows=2048, vocab=151936, top_k=0, banned=False, padded=True),
        # float32 logits of an odd vocabulary with banned tokens, alternatives among the outputs that get gradients
        dict(name="score_odd", kind="score_grad", logits="f32", rows=301, vocab=32003, top_k=20, banned=True, padded=True),
    ]


def draw(rng) -> dict:
    def log_int(low: int, high: int) -> int:
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    kind = rng.choice(["tree", "tree", "tree", "write", "read", "write_read", "score", "score_grad"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    dim = rng.choice([64, 96, 128])
    if kind == "tree":
        heads, kv_heads = rng.choice([(16, 16), (16, 8), (16, 4), (8, 8), (16, 2), (12, 6), (15, 3)])
        nodes = rng.choice([1, log_int(2, 64)])
        case = dict(kind=kind, pool=rng.choice(["bf16", "e4m3", "int8"]), batch=log_int(1, 32), heads=heads, kv_heads=kv_heads,
                    dim=dim, capacity=nodes + log_int(100, 8100), nodes=nodes, dummy=flag(), masked=rng.random() < 0.25)
        # no more than the largest listed: 16 rows of 64 nodes, 32 of one, 8 heads of 128
        pairs, keys = heads * nodes * case["capacity"] * dim, kv_heads * case["capacity"] * dim
        case["batch"] = max(1, min(case["batch"], (16 * 16 * 64 * 8192 * 128) // pairs, (32 * 8 * 8192 * 128) // keys))
        return case
    if kind in ("write", "read", "write_read"):
        case = dict(kind=kind, pool=rng.choice(["e4m3", "int8"] if kind != "write" else ["e4m3"]), batch=log_int(1, 8),
                    channels=rng.choice([1, 2, 4, 8]), kv_heads=rng.choice([2, 4, 6, 8, 16]), dim=dim)
        case["capacity"] = log_int(17, 2049)
        if kind != "read":
            case.update(tokens=log_int(1, case["capacity"] - 1), key=rng.choice(["bf16", "f32"]))
            if case["key"] == "f32":
                case["kv_heads"] = min(8, case["kv_heads"])
        return case
    grad = kind == "score_grad"
    vocab = log_int(1000, 151936)
    rows = log_int(1, 2048)
    logits = rng.choice(["bf16", "f32"])
    most = (2048 if grad else 512) * 151936 // (2 if logits == "f32" else 1)
    return dict(kind=kind, logits=logits, rows=max(1, min(rows, most // vocab)), vocab=vocab,
                top_k=0 if rows * vocab > 4e7 else rng.choice([0, 1, 5, 20, 32]), banned=flag(), padded=flag())


# ----------------------------------------------------------------- inputs ----
class _Normal:
    """Unit normals from one seed."""

    def __init__(self, seed: int) -> None:
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def __call__(self, *shape: int, dtype: torch.dtype = BF16, scale: float = 1.0) -> torch.Tensor:
        return (torch.randn(*shape, generator=self.gen, device=DEV) * scale).to(dtype)

    def integers(self, low: int, high: int, shape: tuple) -> torch.Tensor:
        return torch.randint(low, high, shape, generator=self.gen, device=DEV)


def _codes(x: torch.Tensor, pool: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x as codes and one float32 scale per row: scale = max|x| / the
    largest code, code = x / scale rounded to nearest even."""
    x = x.to(F32)
    most = x.abs().amax(-1, keepdim=True)
    live = most >= SMALLEST
    y = torch.where(live, x * (TOP[pool] / torch.where(live, most, 1.0)), 0.0)
    y = y.clamp(-TOP[pool], TOP[pool])
    codes = y.to(E4M3) if pool == "e4m3" else y.round().to(torch.int8)
    return codes, torch.where(live, most / TOP[pool], 0.0)[..., 0]


def _rope_tables(positions: torch.Tensor, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1e6 ** (-torch.arange(0, dim, 2, device=positions.device, dtype=F64) / dim)
    angle = (positions.to(F64)[..., None] * inv).repeat_interleave(1, dim=-1).repeat(*[1] * positions.ndim, 2)
    return angle.cos().to(F32), angle.sin().to(F32)


def prepare(case: dict, seed: int) -> dict:
    kind, normal = case["kind"], _Normal(seed)
    state: dict = {"case": case}
    if kind == "tree":
        batch, heads, kv_heads, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        nodes, capacity, offset = case["nodes"], case["capacity"], int(case["dummy"])
        room = capacity - nodes - offset  # committed tokens that leave room for the drafted ones
        state["query"] = normal(batch, heads, nodes, dim)
        for side in ("key", "value"):
            rows = normal(batch, kv_heads, capacity, dim)
            if case["pool"] == "bf16":
                state[side] = rows
            else:
                state[side], state[side + "_scales"] = _codes(rows, case["pool"])
        state["lengths"] = normal.integers(max(1, room // 16), room + 1, (batch,))
        state["mask"] = None
        if case["masked"]:  # a third of the context belongs to other documents
            state["mask"] = torch.rand(batch, capacity, generator=normal.gen, device=DEV) < 2 / 3
        # every drafted token hangs under an earlier one, or under the context; it sees its strict ancestors
        parents = [-1 if i == 0 else int(p) for i, p in enumerate((torch.rand(nodes, generator=normal.gen, device=DEV).cpu()
                                                                   * (torch.arange(nodes) + 1)).long() - 1)]
        tree = torch.zeros(nodes, nodes, dtype=torch.bool)
        for i, p in enumerate(parents):
            if p >= 0:
                tree[i] = tree[p]
                tree[i, p] = True
        state["tree"] = tree.to(DEV)
        return state
    if kind in ("write", "read", "write_read"):
        batch, channels, kv_heads, dim, capacity = (case[k] for k in ("batch", "channels", "kv_heads", "dim", "capacity"))
        for side in ("key", "value"):
            pool, scales = _codes(normal(batch, channels, kv_heads, capacity, dim), case["pool"])
            state[side + "_pool"], state[side + "_scales"] = pool, scales
        if kind == "read":
            return state
        tokens = case["tokens"]
        # the projection's output, whose channels and heads are views
        for side in ("key", "value"):
            raw = normal(channels, batch, tokens, kv_heads, dim, dtype=DTYPES[case["key"]])
            state[side] = raw.permute(1, 0, 3, 2, 4)
        state["weight"] = 1 + 0.1 * normal(channels, dim, dtype=F32)
        slots = torch.randperm(capacity - 1, generator=normal.gen, device=DEV)[:tokens] + 1
        state["slots"] = slots.sort().values
        state["cos"], state["sin"] = _rope_tables(state["slots"].expand(batch, tokens) + normal.integers(0, 4000, (batch, 1)), dim)
        state["prefix"] = torch.arange(capacity, device=DEV)[: tokens + 1]
        return state
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["logits"]]
    logits = normal(rows, vocab, dtype=dtype, scale=2.5)
    if case["banned"]:
        logits.masked_fill_(torch.rand(vocab, generator=normal.gen, device=DEV) < 0.01, -math.inf)
    state["logits"] = logits
    tokens = normal.integers(0, vocab, (rows,))
    if case["padded"]:
        tokens[torch.rand(rows, generator=normal.gen, device=DEV) < 0.1] = -100
    state["tokens"] = tokens
    if kind == "score_grad":
        state["grads"] = (normal(rows, dtype=F32), 0.1 * normal(rows, dtype=F32), normal(rows, case["top_k"], dtype=F32))
    return state


# ------------------------------------------------------------ plain forms ----
def _dequantised(codes: torch.Tensor, scales: torch.Tensor | None) -> torch.Tensor:
    return codes.to(F32) if scales is None else codes.to(F32) * scales[..., None]


def _visible(state: dict) -> torch.Tensor:
    """(B, n, N): the slots that each drafted token sees."""
    case = state["case"]
    base = (state["lengths"] + int(case["dummy"]))[:, None, None]
    slot = torch.arange(case["capacity"], device=base.device)[None, None]
    node = (slot - base).expand(-1, case["nodes"], -1)
    inside = (node >= 0) & (node < case["nodes"])
    seen = (node < 0) | (inside & torch.gather(state["tree"].expand(case["batch"], -1, -1), 2, node.clamp(0, case["nodes"] - 1)))
    return seen if state["mask"] is None else seen & state["mask"][:, None]


def _tree_plain(state: dict) -> torch.Tensor:
    case = state["case"]
    key = _dequantised(state["key"], state.get("key_scales"))
    value = _dequantised(state["value"], state.get("value_scales"))
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["dim"]
    group, nodes = case["heads"] // kv_heads, case["nodes"]
    query = state["query"].to(F32).reshape(batch, kv_heads, group * nodes, dim)
    scores = torch.matmul(query, key.transpose(-1, -2)) * dim**-0.5
    seen = _visible(state).repeat(1, group, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, value) / torch.where(total > 0, total, 1.0)
    return out.reshape(batch, case["heads"], nodes, dim).transpose(1, 2).to(BF16)


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos[:, None, None] + turned * sin[:, None, None]


def _write_plain(state: dict) -> None:
    pool, slots = state["case"]["pool"], state["slots"]
    key = state["key"].to(F32)
    key = key * torch.rsqrt(key.square().mean(-1, keepdim=True) + 1e-6) * state["weight"][None, :, None, None]
    key = _rotated(key, state["cos"], state["sin"])
    for side, rows in (("key", key), ("value", state["value"])):
        codes, scales = _codes(rows, pool)
        state[side + "_pool"].view(torch.uint8).index_copy_(3, slots, codes.view(torch.uint8))
        state[side + "_scales"].index_copy_(3, slots, scales)


def _read_plain(state: dict, side: str, slots: torch.Tensor | None) -> torch.Tensor:
    codes, scales = state[side + "_pool"], state[side + "_scales"]
    if slots is not None:
        codes = codes.view(torch.uint8).index_select(3, slots).view(codes.dtype)
        scales = scales.index_select(3, slots)
    return _dequantised(codes, scales).to(BF16)


def _score_plain(state: dict):
    case, x, tokens = state["case"], state["logits"].to(F32), state["tokens"]
    rows, vocab = x.shape
    most = x.amax(-1, keepdim=True)
    log_sum = most + (x - most).exp().sum(-1, keepdim=True).log()
    logp = x - log_sum
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    given = tokens >= 0
    log_probs = torch.where(given, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    k = case["top_k"]
    # values in order and, where they are equal, the lowest index first
    if k:
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
        unique = order * (1 << 31) + (vocab - 1 - torch.arange(vocab, device=x.device))
        indices = unique.topk(k, dim=-1).indices
    else:
        indices = tokens.new_empty(rows, 0)
    outputs = [log_probs, entropy, logp.gather(1, indices), indices]
    if case["kind"] == "score":
        return outputs
    g_token, g_entropy, g_top = state["grads"]
    g_token = torch.where(given, g_token, 0.0)
    slope = -(g_token + g_top.sum(-1))[:, None] - g_entropy[:, None] * (logp + entropy[:, None])
    grad = torch.where(p > 0, p * slope, 0.0)
    grad.scatter_add_(1, torch.cat((tokens.clamp_min(0)[:, None], indices), 1), torch.cat((g_token[:, None], g_top), 1))
    return [*outputs, grad.to(state["logits"].dtype)]


# ------------------------------------------------------------------- calls ----
def _run_own(state: dict):
    from white_matter_amd import kv_pool, token_log_probs, tree_attention

    case, kind = state["case"], state["case"]["kind"]
    if kind == "tree":
        key, value = state["key"], state["value"]
        if case["pool"] != "bf16":
            key = kv_pool.QuantizedPool(key, state["key_scales"])
            value = kv_pool.QuantizedPool(value, state["value_scales"])
        return tree_attention(
            state["query"], key, value, kv_lengths=state["lengths"], tree_mask=state["tree"], use_dummy_token=case["dummy"],
            key_mask=state["mask"],
        )
    if kind in ("write", "read", "write_read"):
        keys, values = (kv_pool.QuantizedPool(state[side + "_pool"], state[side + "_scales"]) for side in ("key", "value"))
        if kind != "read":
            kv_pool.write_pool_quantized(
                state["key"], state["value"], state["weight"], state["cos"], state["sin"], keys, values, state["slots"], eps=1e-6
            )
        if kind == "write":
            return [keys.codes, keys.scales, values.codes, values.scales]
        slots = state["prefix"] if kind == "write_read" else None
        return [kv_pool.read_pool(keys, slots), kv_pool.read_pool(values, slots)]
    if kind == "score":
        return list(token_log_probs(state["logits"], state["tokens"], top_k=case["top_k"]))
    logits = state["logits"].detach().requires_grad_()
    scores = token_log_probs(logits, state["tokens"], top_k=case["top_k"])
    outs = [scores.log_probs, scores.entropy, scores.top_log_probs]
    grads = torch.autograd.grad(outs, logits, state["grads"])
    return [*(t.detach() for t in outs), scores.top_indices, *grads]


def run(state: dict):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "tree":
        return _tree_plain(state)
    if kind in ("score", "score_grad"):
        return _score_plain(state)
    if kind != "read":
        _write_plain(state)
    if kind == "write":
        return [state["key_pool"], state["key_scales"], state["value_pool"], state["value_scales"]]
    slots = state["prefix"] if kind == "write_read" else None
    return [_read_plain(state, "key", slots), _read_plain(state, "value", slots)]


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "tree":
        # rows of the mean length; the queries, the outputs and the scales
        room = case["capacity"] - case["nodes"] - int(case["dummy"])
        mean = (max(1, room // 16) + room) / 2 + int(case["dummy"]) + case["nodes"]
        seen = 2 / 3 if case["masked"] else 1.0
        row = case["dim"] * 2 if case["pool"] == "bf16" else case["dim"] + 4
        keys = case["batch"] * mean * seen
        queries = case["batch"] * case["heads"] * case["nodes"]
        return {"bytes": 2 * keys * case["kv_heads"] * row + 4 * queries * case["dim"],
                "flops": 4 * keys * case["heads"] * case["nodes"] * case["dim"]}
    if kind in ("write", "read", "write_read"):
        rows = case["batch"] * case["channels"] * case["kv_heads"]
        dim, tokens = case["dim"], case.get("tokens", 0)
        moved = 0.0
        if kind != "read":
            moved += 2 * rows * tokens * (dim * (2 if case["key"] == "bf16" else 4) + dim + 4) + 8 * case["batch"] * tokens * dim
        if kind != "write":
            slots = case["capacity"] if kind == "read" else tokens + 1
            moved += 2 * rows * slots * (dim + 4 + 2 * dim)
        return {"bytes": moved, "flops": 0}
    size = case["rows"] * case["vocab"] * (2 if case["logits"] == "bf16" else 4)
    return {"bytes": size * (2 if kind == "score_grad" else 1) + case["rows"] * (16 + 12 * case["top_k"]), "flops": 0}


# -------------------------------------------------- the definitions, 64 bits ----
def _exact_codes(x: torch.Tensor, pool: str) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes as numbers, and the scales."""
    top = TOP[pool]
    most = x.abs().max(-1).values
    scale = torch.where(most < SMALLEST, 0.0, most / top)
    y = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0)
    if pool == "int8":
        return y.round().clamp(-top, top), scale
    # a value of e4m3 has three bits after the leading one, from 2^-6 on
    exponent = torch.frexp(y).exponent.to(F64) - 1
    step = torch.exp2(exponent.clamp_min(-6) - 3)
    return ((y / step).round() * step).clamp(-top, top), scale


def _exact_tree(state: dict) -> torch.Tensor:
    case = state["case"]
    offset, nodes, group = int(case["dummy"]), case["nodes"], case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], nodes, case["heads"], case["dim"], dtype=F64, device=DEV)
    for b in range(case["batch"]):
        base = int(state["lengths"][b]) + offset
        end = base + nodes
        seen = torch.cat((torch.ones(nodes, base, dtype=torch.bool, device=DEV), state["tree"]), 1)
        if state["mask"] is not None:
            seen = seen & state["mask"][b, :end]
        for h in range(case["kv_heads"]):
            rows = {}
            for side in ("key", "value"):
                rows[side] = state[side][b, h, :end].to(F32).to(F64)
                if case["pool"] != "bf16":
                    rows[side] = rows[side] * state[side + "_scales"][b, h, :end, None].to(F64)
            for g in range(group):
                scores = state["query"][b, h * group + g].to(F64) @ rows["key"].t() / math.sqrt(case["dim"])
                weight = torch.softmax(scores.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
                out[b, :, h * group + g] = weight @ rows["value"]
    return out


def _exact_write(state: dict) -> dict:
    """The pools after the write, as (codes as numbers, scales) per side."""
    case, dim = state["case"], state["case"]["dim"]
    x = state["key"].to(F64)
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + 1e-6) * state["weight"].to(F64)[None, :, None, None, :]
    low, high = x[..., : dim // 2], x[..., dim // 2 :]
    c, s = (state[t].to(F64)[:, None, None] for t in ("cos", "sin"))
    h = dim // 2
    key = torch.cat((low * c[..., :h] - high * s[..., :h], high * c[..., h:] + low * s[..., h:]), -1)
    pools = {}
    for side, rows in (("key", key), ("value", state["value"].to(F64))):
        codes, scales = state[side + "_pool"].to(F32).to(F64), state[side + "_scales"].to(F64)
        new, scale = _exact_codes(rows, case["pool"])
        for t, slot in enumerate(state["slots"].tolist()):
            codes[:, :, :, slot] = new[:, :, :, t]
            scales[:, :, :, slot] = scale[:, :, :, t]
        pools[side] = (codes, scales)
    return pools


def _exact_score(state: dict):
    case = state["case"]
    parts: list[list[torch.Tensor]] = []
    for at in range(0, case["rows"], 256):
        x, tokens = state["logits"][at : at + 256].to(F64), state["tokens"][at : at + 256]
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, 0.0)
        entropy = -plogp.sum(-1)
        row = torch.arange(x.shape[0], device=DEV)
        given = (tokens >= 0).to(F64)
        k = case["top_k"]
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k] if k else tokens.new_empty(len(row), 0)
        part = [torch.where(given > 0, logp[row, tokens.clamp_min(0)], 0.0), entropy, logp[row[:, None], best], best]
        if case["kind"] == "score_grad":
            g_token, g_entropy, g_top = (g[at : at + 256].to(F64) for g in state["grads"])
            # what reaches each log probability, then log_softmax's own gradient
            reach = torch.zeros_like(x)
            reach[row, tokens.clamp_min(0)] += g_token * given
            for j in range(k):
                reach[row, best[:, j]] += g_top[:, j]
            grad = reach - p * reach.sum(-1, keepdim=True)
            part.append(grad - g_entropy[:, None] * (plogp + p * entropy[:, None]))
        parts.append(part)
    return [torch.cat(column) for column in zip(*parts)]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "tree":
        return _exact_tree(state)
    if kind in ("score", "score_grad"):
        outputs = _exact_score(state)
        return [*outputs[:3], None, *outputs[4:]]
    if kind == "read":
        return [state[s + "_pool"].to(F32).to(F64) * state[s + "_scales"].to(F64)[..., None] for s in ("key", "value")]
    pools = _exact_write(state)
    if kind == "write":
        return [t for side in ("key", "value") for t in pools[side]]
    count = case["tokens"] + 1
    return [(codes * scales[..., None])[:, :, :, :count] for codes, scales in (pools["key"], pools["value"])]
