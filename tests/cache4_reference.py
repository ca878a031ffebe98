"""Plain 64-bit restatements of the 4-bit cache's format and of attention over it, and of the
check of drafted tokens, for the tests."""

import numpy as np
import torch


def padded(head_dim):
    return 64 if head_dim <= 64 else 128


def half_byte(d, p, keys):
    """Where number d of a row of p lies, from the header's formulas."""
    g, e = divmod(d, p // 4)
    if not keys:
        n = p // 32
        return e // n * (p // 8) + n * g + e % n
    if p == 128:
        return 32 * (e // 8) + 8 * g + 2 * (e % 8 // 4) + e % 4 // 2 + 4 * (e % 2)
    return 16 * (e // 4) + 8 * (g // 2) + 2 * (g % 2) + e % 4 // 2 + 4 * (e % 2)


def rows_of(pool):
    return np.ascontiguousarray(pool.cpu().numpy())


def bf16_at(rows, byte):
    bits = rows[..., byte].astype(np.uint32) << 16 | rows[..., byte + 1].astype(np.uint32) << 24
    return bits.view(np.float32).astype(np.float64)


def decode(pool, head_dim, keys):
    """Values of rows of bytes [..., bytes] and |low| + step code, both float64."""
    rows, p = rows_of(pool), padded(head_dim)
    value = np.zeros((*rows.shape[:-1], head_dim))
    size = np.zeros_like(value)
    for d in range(head_dim):
        n, g = half_byte(d, p, keys), d // (p // 4)
        code = rows[..., n // 2] >> (4 * (n % 2)) & 15
        step, low = bf16_at(rows, p // 2 + 2 * g), bf16_at(rows, p // 2 + 8 + 2 * g)
        value[..., d] = low + step * code
        size[..., d] = np.abs(low) + step * code
    return torch.from_numpy(value), torch.from_numpy(size)


def _bf16_toward(x, down):
    """The bf16 number at or below (above) each x."""
    bits = x.astype(np.float32).view(np.uint32) & np.uint32(0xffff0000)
    best = np.full(x.shape, -np.inf if down else np.inf)
    for off in (-65536, 0, 65536):
        near = (bits.astype(np.int64) + off).clip(0, 0xffffffff).astype(np.uint32).view(np.float32).astype(np.float64)
        near = np.where(np.isfinite(near), near, best)
        best = np.where(near <= x, np.maximum(best, near), best) if down else \
            np.where(near >= x, np.minimum(best, near), best)
    return best


def quantise(x):
    """Values that vectors [..., D] have in the cache, and the groups' steps spread over their
    numbers; groups with a number that is not finite are NaN."""
    x = x.detach().cpu().double().numpy()
    d, each = x.shape[-1], padded(x.shape[-1]) // 4
    value, steps = np.zeros_like(x), np.zeros_like(x)
    for at in range(0, d, each):
        part = x[..., at:at + each]
        odd = ~np.isfinite(part).all(-1, keepdims=True)
        part = np.where(odd, 0.0, part)
        lo, hi = part.min(-1, keepdims=True), part.max(-1, keepdims=True)
        low = np.where(lo == 0, 0.0, _bf16_toward(lo, True))
        span = (hi - low) / 15
        step = np.where(span == 0, 0.0, _bf16_toward(np.where(span == 0, 1.0, span), False))
        step = np.where((step > 0) & (step < 2.0 ** -100), 2.0 ** -100, step)
        code = np.clip(np.rint((part - low) / np.where(step > 0, step, 1.0)), 0, 15)
        value[..., at:at + each] = np.where(odd, np.nan, low + step * code)
        steps[..., at:at + each] = np.where(odd, np.nan, step)
    return torch.from_numpy(value), torch.from_numpy(steps)


def attention64(q, k, v, table, lens, mask=None, drafts=None, scale=None):
    """Attention of drafted tokens in float64 over decoded pools k = (values, sizes) and v
    likewise: the output, sum_p weight size, and the largest visible scale sum_d |q| size."""
    q = q.detach().cpu().double()
    table, lens = table.cpu().long(), lens.cpu().tolist()
    B, H, T, D = q.shape
    group, page = H // k[0].shape[1], k[0].shape[2]
    scale = D ** -0.5 if scale is None else scale
    drafts = [T] * B if drafts is None else drafts.cpu().tolist()
    mask = (torch.ones(T, T, dtype=torch.bool).tril() if mask is None else mask.cpu()).expand(B, T, T)
    out, size, grow = torch.zeros(B, H, T, D).double(), torch.zeros(B, H, T, D).double(), \
        torch.zeros(B, H, T, 1).double()
    for b in range(B):
        at = torch.arange(lens[b] + drafts[b])
        pages, rows = table[b, at // page], at % page
        for h in range(H):
            kk, ks, vv, vs = (x[pages, h // group, rows] for x in (*k, *v))
            for i in range(drafts[b]):
                seen = torch.cat([torch.ones(lens[b], dtype=torch.bool), mask[b, i, :drafts[b]]])
                if not seen.any():
                    continue
                p = torch.softmax(kk[seen] @ q[b, h, i] * scale, 0)
                out[b, h, i] = p @ vv[seen]
                size[b, h, i] = p @ vs[seen]
                grow[b, h, i] = (ks[seen] @ q[b, h, i].abs() * scale).max()
    return out, size, grow


def attention_bound(dtype, out, size, grow, head_dim, keys, rows=1):
    """How far the kernel may be from the 64-bit result.  w = 2^-24.  A score is a sum of
    head_dim exact products and 4 steps and lows in fp32 (the queries' 16-bit form and the lows'
    three bf16 parts add less than w each): off by (head_dim + 12) w grow, a weight by that and a few w
    for the exponential, and normalising doubles it; sums over the keys add keys w.  A weight
    times a step is rounded to fp16, 2^-11; so is the output to its type.

    bf16 queries of more than 16 rows a key head take the kernel whose operands are rounded: keys to
    fp16 (a score is off by 2^-11 grow more, a weight by that, and normalising doubles it), values
    and weights to bf16, 2^-8 each (the sum is of the rounded weights)."""
    w = 2.0 ** -24
    weight = 2 * ((head_dim + 12) * w * grow + 16 * w) + 2 * keys * w + 2.0 ** -11
    if dtype == torch.bfloat16 and rows > 16:
        weight = weight + 2 * 2.0 ** -11 * grow + 3 * 2.0 ** -8
    rounding = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return rounding * out.abs() + (1 + rounding) * weight * size + tiny


def verify64(logits, tokens, uniforms, draft_probs=None, parents=None, drafts=None, temperature=1.0):
    """The check of drafted tokens, a sequence and node at a time, in float64."""
    logits, tokens, uniforms = (x.detach().cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()
                                for x in (logits, tokens, uniforms))
    B, T, V = logits.shape
    if parents is None:
        parents = np.broadcast_to(np.arange(T) - 1, (B, T))
    else:
        parents = np.broadcast_to(parents.cpu().numpy(), (B, T))
    drafts = [T] * B if drafts is None else drafts.cpu().tolist()
    probs = None if draft_probs is None or temperature == 0 else draft_probs.detach().cpu().double().numpy()
    paths, counts, following = np.full((B, T), -1), np.zeros(B, dtype=int), np.full(B, -1)
    for b in range(B):
        if drafts[b] == 0:
            continue
        at, path = 0, [0]
        while True:
            row = logits[b, at]
            if not (row < np.inf).all() or row.max() == -np.inf:
                break
            if temperature == 0:
                p = np.zeros(V)
                p[row.argmax()] = 1.0
            else:
                p = np.exp((row - row.max()) / temperature)
                p /= p.sum()
            kept = -1
            for c in range(at + 1, drafts[b]):
                if parents[b, c] != at:
                    continue
                x = tokens[b, c]
                if probs is None:
                    q = np.zeros(V)
                    q[x] = 1.0
                else:
                    q = np.where(probs[b, at] > 0, probs[b, at], 0.0)
                if uniforms[b, c] * q[x] < p[x]:
                    kept = c
                    break
                rest = np.maximum(p - q, 0.0)
                if rest.sum() > 0:
                    p = rest / rest.sum()
            if kept < 0:
                cum = p.cumsum()
                past = np.nonzero((cum > uniforms[b, 0] * cum[-1]) & (p > 0))[0]
                following[b] = past[0] if len(past) else np.nonzero(p > 0)[0][-1]
                break
            at = kept
            path.append(kept)
        paths[b, :len(path)] = path
        counts[b] = len(path)
    return torch.from_numpy(paths).int(), torch.from_numpy(counts).int(), torch.from_numpy(following)
