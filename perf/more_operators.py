"""Cases of the operators that answer from a 4-bit cache and check drafted tokens:

* ``write``: new keys and values go into a paged cache held in 4 bits, and are read back;
* ``attend``: attention of one token, or of a chain or tree of drafted ones, over such a cache;
* ``verify``: drafted tokens are checked against the target's probabilities with given random
  numbers; the kept path and the next token come out.

A 4-bit cache has the page table of any paged cache: token ``i`` of a sequence lies in row
``i % page_size`` of the page in slot ``i // page_size``.  A row holds one head's vector of ``D``
numbers, padded to ``P`` = 64 or 128, in four groups of ``P / 4``: a number is ``low + step * code``
with a code of 4 bits.  The row is ``P / 2`` bytes of codes, the four steps and the four lows
(bfloat16 each).  The order of the codes in a row of keys and in one of values is that in which the
matrix instruction takes them (``_place``).
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SMALLEST_STEP = 2.0 ** -100


_package = None


def _ops():
    global _package
    if _package is None:
        root = str(Path(__file__).resolve().parents[1] / "techjam-kernel_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import b200_attention as _package

    return _package


# ----------------------------------------------------------------------- cases
def _write(name, layers, batch, tokens, kv_heads, head_dim, page, lo, hi, dtype="bf16", ragged=False):
    case = {"op": "write", "layers": layers, "batch": batch, "tokens": tokens, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype, "ragged": ragged}
    return {"name": name, **case} if name else case


def _attend(name, batch, tokens, kv_heads, group, head_dim, page, lo, hi, dtype="bf16", mask="tree", ragged=False):
    case = {"op": "attend", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype, "mask": mask,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def _verify(name, batch, nodes, vocab, shape, drafter, temperature=1.0, dtype="fp32", ragged=False):
    case = {"op": "verify", "batch": batch, "nodes": nodes, "vocab": vocab, "shape": shape,
            "drafter": drafter, "temperature": temperature, "dtype": dtype, "ragged": ragged}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the drafted rows of one step of a small model, one layer: a decode loop waits for this call
        _write("write_small", 1, 4, 5, 4, 64, 16, 40, 200),
        # one new token of a full serving batch, all layers at once
        _write("write_layers", 12, 64, 1, 16, 64, 16, 30, 700, dtype="fp16"),
        # prompts of unequal length enter the cache of one layer
        _write("write_prompt", 1, 16, 2048, 8, 128, 64, 0, 100, ragged=True),
        # one sequence, one new token: the interactive decode step, where latency counts
        _attend("token_b1", 1, 1, 8, 4, 128, 16, 2000, 2000, mask="none"),
        # a serving batch of unequal lengths, one new token each, from an empty cache to a long one
        _attend("token_b64_ragged", 64, 1, 8, 4, 128, 16, 0, 8191, mask="none"),
        # as many key heads as query heads, narrow heads, a few drafted tokens, an odd page size
        _attend("tree7_mha_fp16", 24, 7, 16, 1, 64, 48, 601, 5003, dtype="fp16", ragged=True),
        # a long document under a draft tree of 16 tokens: one sequence has to fill the GPU
        _attend("tree16_long", 1, 16, 8, 4, 128, 64, 131001, 131001),
        # a batch with trees of 32 tokens, 128 rows a key head: products weigh more than bytes
        _attend("tree32_b16", 16, 32, 8, 4, 128, 64, 1001, 8100),
        # one sequence, a chain of four drafted tokens: latency counts
        _verify("chain_b1", 1, 5, 32000, "chain", "probs"),
        # a serving batch, chains of unequal length, 16-bit logits
        _verify("chain_b64", 64, 8, 32000, "chain", "probs", 0.8, "bf16", ragged=True),
        # trees of 48 nodes from a drafter that gives no probabilities
        _verify("tree_b32", 32, 48, 32000, "tree", "none"),
        # the largest: a wide vocabulary of odd size, trees of drafts that were drawn at random
        _verify("tree_b64_wide", 64, 16, 100003, "tree", "probs"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page, kind = rng.choice([16, 32, 48, 64]), rng.random()
    if kind < 0.25:
        layers, batch, kv_heads = _log(rng, 1, 16), _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16])
        head_dim, dtype = rng.choice([40, 64, 64, 96, 128, 128]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _log(rng, 1, max(2, min(2048, 16 * 2048 * 8 * 128 // (2 * layers * batch * kv_heads * head_dim))))
        lo = rng.choice([0, 1, _log(rng, 1, 300)])
        return _write(None, layers, batch, tokens, kv_heads, head_dim, page, lo, lo + _log(rng, 1, 400), dtype,
                      rng.random() < 0.5)
    if kind < 0.65:
        kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 8])
        head_dim, dtype = rng.choice([40, 64, 64, 96, 128, 128]), rng.choice(["bf16", "bf16", "fp16"])
        batch, tokens = _log(rng, 1, 64), _log(rng, 1, 32)
        hi = _log(rng, 16, max(17, min(65536, 64 * 4096 * 8 // (batch * kv_heads))))
        while batch * kv_heads * group * tokens * hi > 16 * 32 * 32 * 4000:
            batch, hi = max(1, batch // 2), max(16, hi // 2)
        lo = rng.choice([0, 1, hi // 3, hi])
        mask = rng.choice(["tree", "tree", "shared", "none"])
        return _attend(None, batch, tokens, kv_heads, group, head_dim, page, lo, hi, dtype, mask, rng.random() < 0.5)
    vocab = _log(rng, 50, 128000)
    nodes = _log(rng, 1, 48)
    batch = _log(rng, 1, max(2, min(64, 64 * 16 * 100003 // (2 * nodes * vocab))))
    return _verify(None, batch, nodes, vocab, rng.choice(["chain", "tree"]), rng.choice(["probs", "none"]),
                   rng.choice([0.0, 0.7, 1.0, 1.0]), rng.choice(["fp32", "fp32", "bf16", "fp16"]), rng.random() < 0.5)


# ----------------------------------------------------------------------- the format
def _padded(head_dim):
    return 64 if head_dim <= 64 else 128


def _place(p, keys):
    """Where the code of each of p numbers lies in its row, in half bytes.

    Keys: a quarter of the row for each of the four lanes that share a row of the product, and in
    it, for every 16 numbers of the sum, the lane's two pairs.  Values: an eighth of the row for
    each of the eight columns of a product, and in it the columns of that place, group by group."""
    d = np.arange(p)
    group, e = d // (p // 4), d % (p // 4)
    if not keys:
        each = p // 32
        return (e // each) * (p // 8) + each * group + e % each
    if p == 128:
        lane, word, pair = e // 8, group, 2 * (e % 8 // 4) + e % 4 // 2
    else:
        lane, word, pair = e // 4, group // 2, 2 * (group % 2) + e % 4 // 2
    return lane * (p // 4) + 8 * word + pair + 4 * (e % 2)


def _pack(codes, step, low, keys):
    """Rows of bytes from codes [..., P] and the groups' steps and lows [..., 4]."""
    p = codes.shape[-1]
    where = torch.from_numpy(np.argsort(_place(p, keys))).to(codes.device)
    codes = codes[..., where].view(*codes.shape[:-1], p // 2, 2)
    meta = torch.cat([step, low], -1).to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([codes[..., 0] | codes[..., 1] << 4, meta], -1)


def _unpack(rows, head_dim, keys):
    """The values of rows of bytes, in 32 bits."""
    p = _padded(head_dim)
    codes = torch.stack([rows[..., :p // 2] & 15, rows[..., :p // 2] >> 4], -1).flatten(-2)
    codes = codes[..., torch.from_numpy(_place(p, keys)).to(rows.device)].float().unflatten(-1, (4, p // 4))
    meta = rows[..., p // 2:].contiguous().view(torch.bfloat16).float()
    return (codes * meta[..., :4, None] + meta[..., 4:, None]).flatten(-2)[..., :head_dim]


def _bf16_down(x):
    """The largest bfloat16 that is not above x (in 64 bits)."""
    y = x.float().to(torch.bfloat16)
    return torch.where(y.double() > x, torch.nextafter(y, torch.full_like(y, -math.inf)), y)


def _quantise(x):
    """The values that rows x [..., D] have in the cache, in 32 bits."""
    d, p = x.shape[-1], _padded(x.shape[-1])
    x = x.double()
    at = torch.arange(p, device=x.device).view(4, p // 4)
    present = at < d
    parts = torch.nn.functional.pad(x, (0, p - d)).unflatten(-1, (4, p // 4))
    lo = torch.where(present, parts, math.inf).amin(-1)
    hi = torch.where(present, parts, -math.inf).amax(-1)
    empty = ~present[:, 0]
    lo, hi = torch.where(empty, 0.0, lo), torch.where(empty, 0.0, hi)
    low = _bf16_down(lo).double()
    step = -_bf16_down((low - hi) / 15).double()
    step = torch.where((step > 0) & (step < _SMALLEST_STEP), _SMALLEST_STEP, step)
    codes = torch.round((parts - low[..., None]) / torch.where(step > 0, step, 1.0)[..., None]).clamp(0, 15)
    return (codes * step[..., None] + low[..., None]).float().flatten(-2)[..., :d]


# ----------------------------------------------------------------------- inputs
def _lengths(lo, hi, n):
    """n lengths from lo to hi, evenly spaced and then made mostly odd: the same for every seed."""
    if n == 1:
        return [hi]
    return [min(hi, max(lo, lo + (hi - lo) * i // (n - 1) - (i % 3 == 1))) for i in range(n)]


def _counts(case, most):
    """New tokens of each sequence: all of them, or, ragged, from all of them down to none."""
    b = case["batch"]
    return [max(0, most - (most * i) // max(1, b - 1)) if case["ragged"] and b > 1 else most for i in range(b)]


def _parents(nodes, shape, rng, n):
    """Parents [n, nodes] of drafted nodes; the first is the root, and parents come before children."""
    if shape == "chain":
        return np.broadcast_to(np.arange(nodes, dtype=np.int32) - 1, (n, nodes)).copy()
    parents = np.full((n, nodes), -1, dtype=np.int32)
    for i in range(1, nodes):  # about three children a node, the first nodes' first
        parents[:, i] = np.maximum(0, (i - 1) // 3 - rng.integers(0, 2, n))
    return parents


def _trees(tokens, rng, n):
    """Ancestor masks [n, T, T] of random trees whose nodes come after their parents."""
    mask = np.zeros((n, tokens, tokens), dtype=bool)
    for b in range(n):
        for i in range(tokens):
            if i:
                mask[b, i] = mask[b, rng.integers(max(0, i - 6), i)]
            mask[b, i, i] = True
    return mask


def _table(pages_of, slots, total, rng):
    """A page table that gives each sequence its number of pages, scattered over the pool."""
    order = rng.permutation(total)[:sum(pages_of)].astype(np.int32)
    table, at = np.full((len(pages_of), slots), -1, dtype=np.int32), 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _normal(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _pool(shape, head_dim, gen, keys):
    """Pages of a 4-bit cache that has been in use: the codes, steps and lows of normal numbers."""
    p = _padded(head_dim)
    codes = torch.empty((*shape, p), dtype=torch.float16, device="cuda").normal_(7.5, 3.6, generator=gen)
    codes = codes.round_().clamp_(0, 15).to(torch.uint8)
    codes[..., head_dim:] = 0
    step = torch.rand((*shape, 4), generator=gen, device="cuda") * 0.12 + 0.2
    low = step * -(torch.rand((*shape, 4), generator=gen, device="cuda") * 2 + 6.5)
    return _pack(codes, step, low, keys)


def _softmax(x):
    return torch.softmax(x, -1)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype, op, b = _DTYPES[case["dtype"]], case["op"], case["batch"]
    state = {"op": op}

    if op == "verify":
        t, v = case["nodes"], case["vocab"]
        # the target: a few likely tokens and a long tail; the drafter is near it
        logits = torch.randn((b, t, v), generator=gen, device="cuda").mul_(5)
        near = (logits[:, :max(1, t - 1)] + torch.randn((b, max(1, t - 1), v), generator=gen, device="cuda")).contiguous()
        parents = _parents(t, case["shape"], rng, b)
        at = _cuda(parents[:, 1:].astype(np.int64).clip(0))
        if case["drafter"] == "probs":  # children are drawn from their parent's distribution
            probs = _softmax(near)
            rows = probs.flatten(0, 1)[(at + torch.arange(b, device="cuda")[:, None] * probs.shape[1]).flatten()]
            drawn = torch.multinomial(rows, 1, generator=gen).view(b, t - 1) if t > 1 else at
            state["draft_probs"] = probs[:, :t - 1]
        else:  # children are their parent's likeliest tokens, in order
            rank = np.zeros((b, t), dtype=np.int64)
            for i in range(1, t):
                rank[:, i] = (parents[:, 1:i] == parents[:, i:i + 1]).sum(1)
            order = near.topk(min(v, 16), dim=-1).indices
            drawn = order[torch.arange(b, device="cuda")[:, None], at, _cuda(rank[:, 1:]) % order.shape[-1]]
            state["draft_probs"] = None
        root = torch.randint(0, v, (b, 1), generator=gen, device="cuda")
        state["logits"] = logits.to(dtype)
        state["tokens"] = torch.cat([root, drawn], 1)
        state["parents"] = None if case["shape"] == "chain" else _cuda(parents)
        state["uniforms"] = torch.rand((b, t), generator=gen, device="cuda")
        state["drafts"] = _cuda(np.array(_counts(case, t), dtype=np.int32)) if case["ragged"] else None
        state["temperature"] = case["temperature"]
        return state

    page, kv, d = case["page"], case["kv_heads"], case["head_dim"]
    t, order = case["tokens"], rng.permutation(b)
    lens = np.array(_lengths(case["lo"], case["hi"], b), dtype=np.int32)[order]
    drafts = np.array(_counts(case, t), dtype=np.int32)[order]
    pages_of = [-(-int(x + y) // page) for x, y in zip(lens, drafts)]
    total = sum(pages_of) + 3
    state["table"] = _cuda(_table(pages_of, max(1, max(pages_of)), total, rng))
    state["lens"] = _cuda(lens)
    state["drafts"] = _cuda(drafts) if case["ragged"] else None

    if op == "write":
        # heads lie next to each other, as a projection leaves them; keys have an offset of their own
        new = (case["layers"], b, t, kv, d)
        offset = 2 * torch.randn((1, 1, 1, kv, d), generator=gen, device="cuda")
        state["k_new"] = (_normal(new, torch.float32, gen) + offset).to(dtype).transpose(2, 3)
        state["v_new"] = _normal(new, dtype, gen).transpose(2, 3)
        pool = (case["layers"], total, kv, page, _padded(d) // 2 + 16)
        state["k"], state["v"] = (torch.zeros(pool, dtype=torch.uint8, device="cuda") for _ in range(2))
        return state

    state["k"], state["v"] = _pool((total, kv, page), d, gen, True), _pool((total, kv, page), d, gen, False)
    # queries that make a softmax with some weight on few keys, as trained heads do
    state["q"] = _normal((b, t, kv * case["group"], d), dtype, gen).mul_(2).transpose(1, 2)
    state["mask"] = (None if case["mask"] == "none" else _cuda(_trees(t, rng, 1)[0]) if case["mask"] == "shared"
                     else _cuda(_trees(t, rng, b)))
    state["scale"] = d ** -0.5
    return state


# ----------------------------------------------------------------------- plain forms
def _plain_write(s):
    k, v = _quantise(s["k_new"]).to(s["k_new"].dtype), _quantise(s["v_new"]).to(s["v_new"].dtype)
    if s["drafts"] is not None:  # rows that no sequence has are zero
        kept = torch.arange(k.shape[3], device=k.device)[None, :] < s["drafts"][:, None]
        kept = kept[None, :, None, :, None]
        k, v = torch.where(kept, k, 0.0), torch.where(kept, v, 0.0)
    return {"k": k, "v": v}


def _plain_attend(s):
    q, table, page = s["q"], s["table"].long(), s["k"].shape[2]
    b, heads, t, d = q.shape
    kv = s["k"].shape[1]
    keys = table.shape[1] * page
    # every sequence's rows in order, from its pages
    k, v = (_unpack(x[table.clamp(min=0)], d, first).permute(0, 2, 1, 3, 4).reshape(b, kv, keys, d)
            for x, first in ((s["k"], True), (s["v"], False)))
    drafts = s["drafts"] if s["drafts"] is not None else torch.full_like(s["lens"], t)
    at = torch.arange(keys, device=q.device)[None, None, :] - s["lens"][:, None, None]  # place in the draft
    row = torch.arange(t, device=q.device)[None, :, None]
    inside = (at >= 0) & (at < drafts[:, None, None])
    if s["mask"] is None:
        shown = inside & (at <= row)
    else:
        shown = inside & torch.gather(s["mask"].expand(b, t, t), 2, at.clamp(0, t - 1).expand(b, t, keys))
    shown = ((at < 0) | shown) & (row < drafts[:, None, None])
    scores = q.float().reshape(b, kv, heads // kv * t, d) @ k.transpose(2, 3) * s["scale"]
    scores = scores.view(b, kv, heads // kv, t, keys).masked_fill(~shown[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.view(b, kv, heads // kv * t, keys) @ v
    out = out.view(b, kv, heads // kv, t, d) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(b, heads, t, d).to(q.dtype)}


def _plain_verify(s):
    """Speculative sampling in 64 bits: a drawn token sits next to a border of the cumulated weights."""
    logits, tokens, u = s["logits"], s["tokens"], s["uniforms"].double()
    b, t, v = logits.shape
    batch = torch.arange(b, device=logits.device)
    if s["temperature"] > 0:
        x = logits.double() / s["temperature"]
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
    else:  # all weight on the likeliest token
        p = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
        first = torch.where(logits == logits.amax(-1, keepdim=True), torch.arange(v, device=logits.device), v).amin(-1)
        p.scatter_(2, first[..., None], 1.0)
    node = torch.arange(t, device=logits.device)
    parents = s["parents"] if s["parents"] is not None else (node - 1).expand(b, t)
    drafts = s["drafts"].long() if s["drafts"] is not None else torch.full_like(batch, t)
    left, at = p[:, 0], torch.zeros_like(batch)  # the node reached, and what is left of its distribution
    paths = torch.full((b, t), -1, dtype=torch.int32, device=logits.device)
    paths[:, 0] = torch.where(drafts > 0, 0, -1)
    counts = (drafts > 0).int()
    for i in range(1, t):
        asked = (parents[:, i] == at) & (i < drafts)
        x = tokens[:, i, None]
        if s["draft_probs"] is not None and s["temperature"] > 0:
            q = s["draft_probs"][batch, at.clamp(max=t - 2)].double()
        else:
            q = torch.zeros_like(left).scatter_(1, x, 1.0)
        taken = asked & (u[:, i] * q.gather(1, x)[:, 0] < left.gather(1, x)[:, 0])
        rest = (left - q).clamp(min=0)
        total = rest.sum(-1, keepdim=True)
        refused = (asked & ~taken)[:, None] & (total > 0)
        left = torch.where(taken[:, None], p[:, i], torch.where(refused, rest / torch.where(total > 0, total, 1.0), left))
        at = torch.where(taken, i, at)
        paths = paths.scatter(1, counts.long().clamp(max=t - 1)[:, None],
                              torch.where(taken, i, paths.gather(1, counts.long().clamp(max=t - 1)[:, None])[:, 0])[:, None].int())
        counts = counts + taken.int()
    cum = left.cumsum(-1)
    past = (cum > u[:, :1] * cum[:, -1:]) & (left > 0)
    last = v - 1 - (left > 0).flip(-1).int().argmax(-1)
    drawn = torch.where(past.any(-1), past.int().argmax(-1), last)
    return {"paths": paths, "counts": counts, "next": torch.where(drafts > 0, drawn, -1)}


_PLAIN = {"write": _plain_write, "attend": _plain_attend, "verify": _plain_verify}


# ----------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return _PLAIN[s["op"]](s)
    ops = _ops()
    if s["op"] == "write":
        _, _, _, t, d = s["k_new"].shape
        ops.b200_cache_append(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["lens"], s["drafts"])
        k, v = ops.b200_cache_read(s["k"], s["v"], s["table"], s["lens"], t, d, s["k_new"].dtype, s["drafts"])
        return {"k": k, "v": v}
    if s["op"] == "attend":
        return {"out": ops.b200_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["mask"], s["drafts"], s["scale"])}
    paths, counts, following = ops.b200_verify_drafts(s["logits"], s["tokens"], s["uniforms"], s["draft_probs"],
                                                      s["parents"], s["drafts"], s["temperature"])
    return {"paths": paths, "counts": counts, "next": following}


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "verify":
        # Rows of the target that cannot be left out: those of the nodes on the path, the root's always, and a
        # draft is kept about two times in three; of the drafter, the row where the path ends.
        b, t = case["batch"], case["nodes"]
        counts = _counts(case, t)
        depth = [n if case["shape"] == "chain" else math.log(2 * n + 1, 3) for n in counts]
        rows = sum((1 - (2 / 3) ** x) * 3 for x in depth)
        drafter = sum(n > 1 for n in counts) if case["drafter"] == "probs" and case["temperature"] > 0 else 0
        moved = (rows * size + drafter * 4) * case["vocab"]
        return {"bytes": moved + sum(counts) * 12 + b * (t * 4 + 12), "flops": 6 * rows * case["vocab"]}
    kv, d = case["kv_heads"], case["head_dim"]
    row = d / 2 + 16  # of the cache
    counts = _counts(case, case["tokens"])
    if case["op"] == "write":
        rows = 2 * case["layers"] * kv
        # numbers in, rows of the cache out, rows of the cache in, numbers out
        moved = rows * (sum(counts) * (d * size + 2 * row) + case["batch"] * case["tokens"] * d * size)
        return {"bytes": moved + 4 * sum(-(-n // case["page"]) for n in counts), "flops": 8 * rows * sum(counts) * d}
    b, t, heads = case["batch"], case["tokens"], kv * case["group"]
    lens = _lengths(case["lo"], case["hi"], b)
    rows = sum(x + y for x, y in zip(lens, counts) if y)
    masks = {"none": 0, "shared": 1, "tree": b}[case["mask"]] * t * t
    moved = rows * kv * 2 * row + (sum(counts) + b * t) * heads * d * size + masks + 4 * (rows // case["page"]) + 8 * b
    # a drafted token sees the committed tokens and itself at least
    return {"bytes": moved, "flops": 4 * heads * d * sum(y * (x + 1) for x, y in zip(lens, counts))}


# ----------------------------------------------------------------------- in 64 bits
def _number(rows, d, head_dim, keys):
    """Number d of every row of bytes [..., bytes], in 64 bits, from the format's definition."""
    p = 64 if head_dim <= 64 else 128
    g, e = divmod(d, p // 4)
    if not keys:
        n = e // (p // 32) * (p // 8) + p // 32 * g + e % (p // 32)
    elif p == 128:
        n = 32 * (e // 8) + 8 * g + 2 * (e % 8 // 4) + e % 4 // 2 + 4 * (e % 2)
    else:
        n = 16 * (e // 4) + 8 * (g // 2) + 2 * (g % 2) + e % 4 // 2 + 4 * (e % 2)
    code = (rows[..., n // 2].int() >> 4 * (n % 2)) & 15

    def at(byte):  # a bfloat16
        bits = rows[..., byte].int() << 16 | rows[..., byte + 1].int() << 24
        return bits.view(torch.float32).double()

    return at(p // 2 + 2 * g) * code + at(p // 2 + 8 + 2 * g)


def _exact_write(case, s):
    """Group by group: the low is the bfloat16 at or below the smallest number, the step the one at or
    above a fifteenth of the way from it to the largest."""
    out = {}
    counts = _counts(case, case["tokens"])
    if s["drafts"] is not None:
        counts = s["drafts"].tolist()
    for name in ("k", "v"):
        x = s[name + "_new"].double()
        d, y = x.shape[-1], torch.zeros_like(x)
        each = (64 if d <= 64 else 128) // 4
        for at in range(0, d, each):
            part = x[..., at:at + each]
            lo, hi = part.aminmax(dim=-1, keepdim=True)

            def toward(a, up):  # the next bfloat16 up or down, by its bits
                bits = a.float().view(torch.int32) & -65536
                near = [(bits + n * 65536).view(torch.float32).double() for n in (-1, 0, 1)]
                if up:
                    return torch.stack([torch.where(n >= a, n, math.inf) for n in near]).amin(0)
                return torch.stack([torch.where(n <= a, n, -math.inf) for n in near]).amax(0)

            low = torch.where(lo == 0, 0.0, toward(lo, False))
            span = (hi - low) / 15
            step = torch.where(span == 0, 0.0, toward(span, True))
            code = torch.where(step > 0, torch.round((part - low) / step), 0.0).clamp(0, 15)
            y[..., at:at + each] = low + step * code
        for i, n in enumerate(counts):
            y[:, i, :, n:] = 0
        out[name] = y
    return out


def _exact_attend(case, s):
    """One sequence and drafted token at a time."""
    b, heads, t, d = s["q"].shape
    kv, page = case["kv_heads"], case["page"]
    out = torch.zeros((b, heads, t, d), dtype=torch.float64, device="cuda")
    table, lens = s["table"].cpu().numpy(), s["lens"].cpu().numpy()
    drafts = s["drafts"].cpu().numpy() if s["drafts"] is not None else np.full(b, t)
    if s["mask"] is None:
        mask = np.tril(np.ones((t, t), dtype=bool))[None].repeat(b, 0)
    else:
        mask = np.broadcast_to(s["mask"].cpu().numpy(), (b, t, t))
    for i in range(b):
        n = int(lens[i] + drafts[i])
        if not drafts[i]:
            continue
        ids = torch.from_numpy(table[i, :-(-n // page)].astype(np.int64)).cuda()
        k, v = (torch.stack([_number(x[ids], j, d, first) for j in range(d)], -1).transpose(0, 1).reshape(kv, -1, d)[:, :n]
                for x, first in ((s["k"], True), (s["v"], False)))
        for j in range(int(drafts[i])):
            seen = np.concatenate([np.arange(lens[i]), lens[i] + np.nonzero(mask[i, j, :drafts[i]])[0]]).astype(np.int64)
            if not len(seen):
                continue
            at = torch.from_numpy(seen).cuda()
            q = s["q"][i, :, j].double().view(kv, heads // kv, d)
            w = torch.softmax(torch.einsum("hgd,hkd->hgk", q, k[:, at]) * s["scale"], dim=-1)
            out[i, :, j] = torch.einsum("hgk,hkd->hgd", w, v[:, at]).reshape(heads, d)
    return {"out": out}


def exact(case, seed):
    """What was written, and the attention, from their definitions.  None for the check of drafts, whose
    results are whole numbers."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    return _exact_write(case, s) if case["op"] == "write" else _exact_attend(case, s)
