"""Cases of the paged-cache operators: drafted-token (tree) attention over a paged
key/value cache, and the cache's page operations (append, accept, reserve, fork, free, compact).

A cache is a pool of pages ``[layers, pages, kv_heads, page_size, head_dim]`` for keys and one for
values, a page table ``[batch, slots]`` (-1: no page), the number of committed tokens of each
sequence and a reference count for each page.  Token ``i`` of a sequence lies in row
``i % page_size`` of the page in slot ``i // page_size``; drafted tokens follow the committed ones.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


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
def _attend(name, batch, tokens, kv_heads, group, head_dim, page, lo, hi, dtype="bf16", mask="tree", ragged=False):
    case = {"op": "attend", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype, "mask": mask,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def _step(name, layers, batch, tokens, kv_heads, head_dim, page, lo, hi, dtype="bf16"):
    case = {"op": "step", "layers": layers, "batch": batch, "tokens": tokens, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype}
    return {"name": name, **case} if name else case


def _fork(name, layers, parents, children, tokens, kv_heads, head_dim, page, lo, hi, dtype="bf16"):
    case = {"op": "fork", "layers": layers, "parents": parents, "children": children, "tokens": tokens,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype}
    return {"name": name, **case} if name else case


def _compact(name, layers, batch, finished, kv_heads, head_dim, page, lo, hi, dtype="bf16"):
    case = {"op": "compact", "layers": layers, "batch": batch, "finished": finished, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lo": lo, "hi": hi, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one sequence, one new token: the interactive decode step, where latency counts
        _attend("token_b1", 1, 1, 8, 4, 128, 16, 1000, 1000, mask="none"),
        # a serving batch of unequal lengths, one new token each, from an empty cache to a long one
        _attend("token_b64_ragged", 64, 1, 8, 4, 128, 16, 0, 8191, mask="none"),
        # a long document under one 16-token draft tree: one sequence has to fill the GPU
        _attend("tree16_long", 1, 16, 8, 4, 128, 64, 131001, 131001),
        # as many key heads as query heads, narrow heads, wide trees of unequal size, an odd page size
        _attend("tree63_mha_fp16", 5, 63, 16, 1, 64, 48, 601, 5003, dtype="fp16", ragged=True),
        # 32-bit cache, narrow odd-sized heads, a small batch: the check run of a small model
        _attend("tree5_fp32", 3, 5, 4, 3, 40, 16, 33, 700, dtype="fp32", ragged=True),
        # the largest: a full batch with 64-token trees, where products weigh as much as bytes
        _attend("tree64_b32", 32, 64, 8, 4, 128, 64, 1001, 8100),
        # one draft step of a small model: write the drafted rows, keep the accepted path
        _step("step_small", 2, 2, 5, 4, 64, 16, 40, 200),
        # one draft step of all layers of a large model at full batch
        _step("step_large", 32, 64, 16, 8, 128, 16, 30, 300),
        # four continuations of one prompt: re-fork the branches and reserve room for their next token
        _fork("fork_small", 2, 1, 4, 1, 4, 64, 16, 75, 75),
        # many continuations of many prompts over all layers: copies of the partly filled last pages count
        _fork("fork_large", 32, 32, 224, 1, 8, 128, 16, 39, 170),
        # a few short sequences, one has finished: release it and close the gaps in the pool
        _compact("compact_small", 2, 4, 1, 4, 64, 16, 50, 200),
        # a full batch, a third has finished: close the gaps over all layers
        _compact("compact_large", 32, 48, 16, 8, 128, 16, 60, 500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice([16, 32, 48, 64])
    kind = rng.random()
    if kind < 0.55:
        kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 8])
        head_dim = rng.choice([40, 64, 64, 96, 128, 128])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":  # small check runs
            batch, tokens, hi = _log(rng, 1, 4), _log(rng, 1, 16), _log(rng, 16, 1000)
        else:
            batch, tokens = _log(rng, 1, 64), _log(rng, 1, 64)
            # no more keys in all than the largest listed case has
            hi = _log(rng, 16, max(17, min(65536, 32 * 8100 * 8 // (batch * kv_heads) // 2)))
            while batch * kv_heads * group * tokens * hi > 32 * 32 * 64 * 4000:
                batch, hi = max(1, batch // 2), max(16, hi // 2)
        lo = rng.choice([0, 1, hi // 3, hi])
        mask = rng.choice(["tree", "tree", "shared", "none"])
        return _attend(None, batch, tokens, kv_heads, group, head_dim, page, lo, hi, dtype, mask, rng.random() < 0.5)
    layers, kv_heads, head_dim = _log(rng, 1, 32), rng.choice([2, 4, 8]), rng.choice([64, 96, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind < 0.7:
        lo = _log(rng, 1, 60)
        return _step(None, layers, _log(rng, 1, 32), _log(rng, 3, 16), kv_heads, head_dim, page, lo, _log(rng, lo, 300), dtype)
    if kind < 0.85:
        parents = _log(rng, 1, 16)
        return _fork(None, layers, parents, parents * rng.randint(1, 5), _log(rng, 1, 8), kv_heads, head_dim, page,
                     _log(rng, 1, 40), _log(rng, 40, 170), dtype)
    batch = _log(rng, 2, 24)
    return _compact(None, layers, batch, rng.randint(1, batch - 1), kv_heads, head_dim, page, _log(rng, 1, 60), _log(rng, 60, 400), dtype)


# ----------------------------------------------------------------------- inputs
def _lengths(lo, hi, n):
    """n lengths from lo to hi, evenly spaced and then made mostly odd: the same for every seed."""
    if n == 1:
        return [hi]
    return [min(hi, max(lo, lo + (hi - lo) * i // (n - 1) - (i % 3 == 1))) for i in range(n)]


def _drafts(case):
    """Drafted tokens of each sequence; the first has the full tree, ragged ones go down to none."""
    t, b = case["tokens"], case["batch"]
    return [max(0, t - (t * i) // max(1, b - 1)) if case.get("ragged") and b > 1 else t for i in range(b)]


def _counts(case):
    """Accepted tokens of each sequence of a draft step, at most one less than the drafted ones."""
    most = max(1, min(8, case["tokens"] - 1))
    return [i % (most + 1) for i in range(1, case["batch"] + 1)]


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


def _pool(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16).to(dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype, page, op = _DTYPES[case["dtype"]], case["page"], case["op"]
    kv, d = case["kv_heads"], case["head_dim"]
    state = {"op": op, "page": page}

    if op == "attend":
        b, t = case["batch"], case["tokens"]
        order = rng.permutation(b)
        lens = np.array(_lengths(case["lo"], case["hi"], b), dtype=np.int32)[order]
        drafts = np.array(_drafts(case), dtype=np.int32)[order]
        pages_of = [-(-int(x + y) // page) for x, y in zip(lens, drafts)]
        total = sum(pages_of) + 3
        pool = (total, kv, page, d)
        state["k"], state["v"] = _pool(pool, dtype, gen), _pool(pool, dtype, gen)
        # queries that make a softmax with some weight on few keys, as trained heads do
        state["q"] = _pool((b, t, kv * case["group"], d), dtype, gen).mul_(2).transpose(1, 2)
        state["table"] = _cuda(_table(pages_of, max(1, max(pages_of)), total, rng))
        state["lens"] = _cuda(lens)
        state["drafts"] = _cuda(drafts) if case["ragged"] else None
        state["mask"] = (None if case["mask"] == "none" else _cuda(_trees(t, rng, 1)[0]) if case["mask"] == "shared"
                         else _cuda(_trees(t, rng, b)))
        state["scale"] = d ** -0.5
        return state

    layers = case["layers"]
    if op == "step":
        b, t = case["batch"], case["tokens"]
        lens = np.array(_lengths(case["lo"], case["hi"], b), dtype=np.int32)[rng.permutation(b)]
        pages_of = [-(-int(x + t) // page) for x in lens]
        counts = np.array(_counts(case), dtype=np.int32)[rng.permutation(b)]
        paths = np.zeros((b, max(1, int(counts.max()))), dtype=np.int32)
        for i in range(b):  # the root, then a path that leaves out the root's first child
            if paths.shape[1] > 1:
                paths[i, 1:] = 2 + np.sort(rng.permutation(t - 2)[:paths.shape[1] - 1])
        new = (layers, b, t, kv, d)
        state["k_new"], state["v_new"] = (_pool(new, dtype, gen).transpose(2, 3) for _ in range(2))
        state["counts"], state["paths"] = _cuda(counts), _cuda(paths)
        table = _table(pages_of, max(pages_of), sum(pages_of) + 5, rng)
        total = sum(pages_of) + 5
    elif op == "fork":
        p, c = case["parents"], case["children"]
        parent_lens = _lengths(case["lo"], case["hi"], p)
        lens = np.array([parent_lens[i] for i in range(p)] + [parent_lens[i % p] for i in range(c)], dtype=np.int32)
        pages_of = [-(-x // page) for x in parent_lens]
        grow = -(-(max(parent_lens) + case["tokens"]) // page) + 1
        slots = max(grow, max(pages_of))
        total = sum(pages_of) + c * (2 + case["tokens"] // page) + 7
        table = np.full((p + c, slots), -1, dtype=np.int32)
        table[:p] = _table(pages_of, slots, total, rng)
        for i in range(c):  # the branches hold what their parent holds: a fork without a write yet
            table[p + i] = table[i % p]
        state["src"] = _cuda((np.arange(c, dtype=np.int32) % p).astype(np.int32))
        state["dst"] = _cuda(np.arange(p, p + c, dtype=np.int32))
        state["tokens"] = _cuda(np.array([0] * p + [case["tokens"]] * c, dtype=np.int32))
    else:
        b = case["batch"]
        lens = np.array(_lengths(case["lo"], case["hi"], b), dtype=np.int32)[rng.permutation(b)]
        pages_of = [-(-int(x) // page) for x in lens]
        total = sum(pages_of) + 4
        table = _table(pages_of, max(pages_of), total, rng)
        state["rows"] = _cuda(np.sort(rng.permutation(b)[:case["finished"]]).astype(np.int32))
    pool = (layers, total, kv, page, d)
    state["k"], state["v"] = _pool(pool, dtype, gen), _pool(pool, dtype, gen)
    refs = np.bincount(table[table >= 0].reshape(-1), minlength=total).astype(np.int32)
    state["table"], state["lens"], state["refs"] = _cuda(table), _cuda(lens), _cuda(refs)
    if op == "compact":  # the scheduler's copy of the bookkeeping, which each pass starts from
        state["table0"], state["lens0"], state["refs0"] = (state[n].clone() for n in ("table", "lens", "refs"))
    return state


# ----------------------------------------------------------------------- plain forms
def _plain_attend(s):
    q, table, page = s["q"], s["table"].long(), s["page"]
    b, heads, t, d = q.shape
    kv = s["k"].shape[1]
    keys = table.shape[1] * page
    # every sequence's rows in order, from its pages
    k, v = (x[table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(b, kv, keys, d).float() for x in (s["k"], s["v"]))
    drafts = s["drafts"] if s["drafts"] is not None else torch.full_like(s["lens"], t)
    at = torch.arange(keys, device=q.device)[None, None, :] - s["lens"][:, None, None]  # place in the draft
    row = torch.arange(t, device=q.device)[None, :, None]
    inside = (at >= 0) & (at < drafts[:, None, None])
    if s["mask"] is None:
        shown = inside & (at <= row)
    else:
        mask = s["mask"].expand(b, t, t)
        shown = inside & torch.gather(mask, 2, at.clamp(0, t - 1).expand(b, t, keys))
    shown = ((at < 0) | shown) & (row < drafts[:, None, None])
    # rows that no key of this sequence fills may hold anything
    used = (at < drafts[:, None, None])[:, 0, None, :, None]
    v = torch.where(used, v, 0.0)
    scores = q.float().reshape(b, kv, heads // kv * t, d) @ k.transpose(2, 3) * s["scale"]
    scores = scores.view(b, kv, heads // kv, t, keys).masked_fill(~shown[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.view(b, kv, heads // kv * t, keys) @ v
    out = out.view(b, kv, heads // kv, t, d) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(b, heads, t, d).to(q.dtype)}


def _places(table, lens, tokens, page):
    """Page and row of tokens lens + 0..tokens-1 of each sequence."""
    at = lens.long()[:, None] + tokens
    return table.long().gather(1, at // page), at % page


def _plain_step(s):
    k, v, table, lens, page = s["k"], s["v"], s["table"], s["lens"], s["page"]
    t = s["k_new"].shape[3]
    pages, rows = _places(table, lens, torch.arange(t, device=lens.device)[None, :], page)
    k[:, pages, :, rows] = s["k_new"].permute(1, 3, 0, 2, 4)
    v[:, pages, :, rows] = s["v_new"].permute(1, 3, 0, 2, 4)
    kept = torch.arange(s["paths"].shape[1], device=lens.device)[None, :] < s["counts"][:, None]
    to_pages, to_rows = _places(table, lens, torch.arange(kept.shape[1], device=lens.device)[None, :], page)
    from_pages, from_rows = _places(table, lens, s["paths"].long(), page)
    a, r, c, f = to_pages[kept], to_rows[kept], from_pages[kept], from_rows[kept]
    k[:, a, :, r] = k[:, c, :, f]
    v[:, a, :, r] = v[:, c, :, f]
    return {"k": k, "v": v, "lens": lens + s["counts"]}


def _plain_fork(s):
    k, v, table, lens, refs, page = s["k"], s["v"], s["table"], s["lens"], s["refs"], s["page"]
    src, dst = s["src"].long(), s["dst"].long()
    slot = torch.arange(table.shape[1], device=table.device)[None, :]
    one = torch.ones((), dtype=refs.dtype, device=refs.device)
    # the branches let go of what they held and share their parent's pages
    old = table[dst]
    held = old >= 0
    refs.index_add_(0, old[held].long(), -one.expand(int(held.sum())))
    rows = torch.where(slot * page < lens[src][:, None], table[src], -1)
    held = rows >= 0
    refs.index_add_(0, rows[held].long(), one.expand(int(held.sum())))
    table[dst] = rows
    lens[dst] = lens[src]
    # pages of their own for the tokens to come
    more = s["tokens"]
    wanted = (slot >= (lens // page)[:, None]) & (slot * page < (lens + more)[:, None]) & (more > 0)[:, None]
    held = table >= 0
    shared = wanted & held & (refs[table.clamp(min=0).long()] > 1)
    need = (wanted & ~held) | shared
    free = refs == 0
    lack = need.sum() > free.sum()
    full = ((more > 0) & (lens + more > table.shape[1] * page)).any()
    need, shared = need & ~(lack | full), shared & ~(lack | full)
    order = torch.argsort((~free).int(), stable=True)
    rank = (need.flatten().cumsum(0) - 1).clamp(0, refs.numel() - 1).view_as(table)
    given = order[rank]
    part = lens % page
    copied = shared & (slot == (lens // page)[:, None]) & (part > 0)[:, None]
    a, c = given[copied], table[copied].long()
    filled = torch.arange(page, device=table.device)[None, :] < part[:, None].expand_as(table)[copied][:, None]
    filled = filled[None, :, None, :, None]
    k[:, a] = torch.where(filled, k[:, c], k[:, a])
    v[:, a] = torch.where(filled, v[:, c], v[:, a])
    refs.index_add_(0, table[shared].long(), -one.expand(int(shared.sum())))
    refs[given[need]] = 1
    table.copy_(torch.where(need, given.int(), table))
    return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "status": (lack.int() + 2 * full.int()).view(1)}


def _plain_compact(s):
    k, v, table, lens, refs = s["k"], s["v"], s["table"], s["lens"], s["refs"]
    for name in ("table", "lens", "refs"):
        s[name].copy_(s[name + "0"])
    rows = s["rows"].long()
    old = table[rows]
    held = old[old >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=refs.dtype))
    table[rows] = -1
    lens[rows] = 0
    live = refs > 0
    count = int(live.sum())
    holes = torch.nonzero(~live[:count])[:, 0]
    movers = torch.nonzero(live[count:])[:, 0] + count
    k[:, holes] = k[:, movers]
    v[:, holes] = v[:, movers]
    place = torch.arange(refs.numel(), device=refs.device)
    place[movers] = holes
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].int(), -1))
    refs[holes] = refs[movers]
    refs[movers] = 0
    return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "live": torch.full_like(lens[:1], count)}


_PLAIN = {"attend": _plain_attend, "step": _plain_step, "fork": _plain_fork, "compact": _plain_compact}


# ----------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return _PLAIN[s["op"]](s)
    ops = _ops()
    if s["op"] == "attend":
        return {"out": ops.b200_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["mask"], s["drafts"], s["scale"])}
    k, v, table, lens = s["k"], s["v"], s["table"], s["lens"]
    if s["op"] == "step":
        ops.b200_cache_append(s["k_new"], s["v_new"], k, v, table, lens)
        return {"k": k, "v": v, "lens": ops.b200_cache_accept(k, v, table, lens, s["paths"], s["counts"])}
    refs = s["refs"]
    if s["op"] == "fork":
        ops.b200_cache_fork(table, lens, refs, s["src"], s["dst"], s["page"])
        status = ops.b200_cache_reserve(k, v, table, lens, refs, s["tokens"])
        return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "status": status}
    for name in ("table", "lens", "refs"):
        s[name].copy_(s[name + "0"])
    ops.b200_cache_free(table, lens, refs, s["rows"])
    live = ops.b200_cache_compact(k, v, table, refs)
    return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "live": live}


def work(case):
    size, page, kv, d = (4 if case["dtype"] == "fp32" else 2), case["page"], case["kv_heads"], case["head_dim"]
    if case["op"] == "attend":
        b, t = case["batch"], case["tokens"]
        lens, drafts, heads = _lengths(case["lo"], case["hi"], b), _drafts(case), kv * case["group"]
        rows = sum(x + y for x, y in zip(lens, drafts) if y)
        masks = {"none": 0, "shared": 1, "tree": b}[case["mask"]] * t * t
        moved = rows * kv * d * 2 * size + sum(drafts) * heads * d * size + b * heads * t * d * size + masks + 4 * (rows // page) + 8 * b
        # a drafted token sees the committed tokens and itself at least
        return {"bytes": moved, "flops": 4 * heads * d * sum(y * (x + 1) for x, y in zip(lens, drafts))}
    token = case["layers"] * kv * d * 2 * size  # one token's keys and values in all layers
    if case["op"] == "step":
        counts = _counts(case)
        moved = case["batch"] * case["tokens"] + sum(max(0, c - 1) for c in counts)
        return {"bytes": 2 * moved * token + 8 * sum(counts) + 16 * case["batch"], "flops": 0}
    if case["op"] == "fork":
        parents = _lengths(case["lo"], case["hi"], case["parents"])
        lens = [parents[i % len(parents)] for i in range(case["children"])]
        return {"bytes": sum(2 * (x % page) * token + 8 * -(-x // page) for x in lens), "flops": 0}
    pages = [-(-x // page) for x in _lengths(case["lo"], case["hi"], case["batch"])]
    total = sum(pages) + 4
    live = sum(pages) * (1 - case["finished"] / case["batch"])
    # pages lie at random: so many of the live ones, on average, lie past the first `live` places
    return {"bytes": 2 * live * (1 - live / total) * page * token + 8 * total + 8 * sum(pages), "flops": 0}


# ----------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The drafted tokens' attention from its definition, one sequence and drafted token at a time;
    None for the page operations, which only move rows."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
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
        k, v = (x.index_select(0, ids).transpose(0, 1).reshape(kv, -1, d)[:, :n].double() for x in (s["k"], s["v"]))
        for j in range(int(drafts[i])):
            seen = np.concatenate([np.arange(lens[i]), lens[i] + np.nonzero(mask[i, j, :drafts[i]])[0]]).astype(np.int64)
            if not len(seen):
                continue
            at = torch.from_numpy(seen).cuda()
            q = s["q"][i, :, j].double().view(kv, heads // kv, d)
            w = torch.softmax(torch.einsum("hgd,hkd->hgk", q, k[:, at]) * s["scale"], dim=-1)
            out[i, :, j] = torch.einsum("hgk,hkd->hgd", w, v[:, at]).reshape(heads, d)
    return {"out": out}
