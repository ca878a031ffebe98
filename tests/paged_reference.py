"""Plain 64-bit and Python restatements of the paged-cache operators, for the tests."""

import numpy as np
import torch


def attention64(q, k_pages, v_pages, table, lens, mask=None, drafts=None, scale=None):
    """Drafted-token attention from its definition, in float64 on the CPU.  Returns
    the output, sum_p weight |v| and the largest visible scale * sum_d |q k| (each
    like the output or broadcastable to it), which the error bounds are made of."""
    q, k_pages, v_pages = (t.detach().cpu().double() for t in (q, k_pages, v_pages))
    table, lens = table.cpu().long(), lens.cpu().tolist()
    B, H, T, D = q.shape
    group, page = H // k_pages.shape[1], k_pages.shape[2]
    scale = D ** -0.5 if scale is None else scale
    drafts = [T] * B if drafts is None else drafts.cpu().tolist()
    if mask is None:
        mask = torch.ones(T, T, dtype=torch.bool).tril()
    mask = mask.cpu().expand(B, T, T)
    out, size, grow = torch.zeros(B, H, T, D).double(), torch.zeros(B, H, T, D).double(), \
        torch.zeros(B, H, T, 1).double()
    for b in range(B):
        n = lens[b] + drafts[b]
        at = torch.arange(n)
        pages, rows = table[b, at // page], at % page
        for i in range(drafts[b]):
            seen = torch.cat([torch.arange(lens[b]),
                              lens[b] + mask[b, i, :drafts[b]].nonzero()[:, 0]]).long()
            if len(seen) == 0:
                continue
            for h in range(H):
                k = k_pages[pages[seen], h // group, rows[seen]]
                v = v_pages[pages[seen], h // group, rows[seen]]
                s = (k @ q[b, h, i]) * scale
                p = torch.softmax(s, 0)
                out[b, h, i] = p @ v
                size[b, h, i] = p @ v.abs()
                grow[b, h, i] = ((k.abs() @ q[b, h, i].abs()) * scale).max()
    return out, size, grow


def attention_bound(dtype, out, size, grow, head_dim, keys):
    """How far the kernels' output may be from the 64-bit one, element by element.

    With 2u the largest relative error of one rounding to the type, and w = 2^-24: a
    score is a sum of head_dim products, off by at most head_dim w grow, so a weight by
    that and a few w for the exponential; normalising doubles it.  Sums over the keys add
    keys w.  16-bit weights are rounded, so is the output: 3u of the size of the sum in
    all, which is one and a half times the largest error of one rounding (the
    weights' errors are independent, and do not all point one way).  Half a smallest
    subnormal at least."""
    u = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12, torch.float32: 2.0 ** -24}[dtype]
    tiny = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}[dtype]
    w = 2.0 ** -24
    weight = 2 * ((head_dim + 4) * w * grow + 16 * w) + 2 * keys * w
    if dtype != torch.float32:
        weight = weight + 2 * u
    return u * out.abs() + (1 + u) * weight * size + tiny


class CacheModel:
    """The page operations in plain Python on numpy copies of the tensors."""

    def __init__(self, k, v, table, lens, refs):
        self.k, self.v = (t.detach().float().cpu().numpy().copy() for t in (k, v))
        self.table, self.lens, self.refs = (t.cpu().numpy().copy() for t in (table, lens, refs))
        self.page = self.k.shape[3]

    def _rows(self, b, token):
        return self.table[b, token // self.page], token % self.page

    def append(self, k_new, v_new, counts=None):
        k_new, v_new = k_new.float().cpu().numpy(), v_new.float().cpu().numpy()
        for b in range(self.table.shape[0]):
            for j in range(k_new.shape[3] if counts is None else int(counts[b])):
                p, r = self._rows(b, int(self.lens[b]) + j)
                self.k[:, p, :, r] = k_new[:, b, :, j]
                self.v[:, p, :, r] = v_new[:, b, :, j]

    def accept(self, paths, counts):
        for b in range(self.table.shape[0]):
            moved = []
            for j in range(int(counts[b])):
                p, r = self._rows(b, int(self.lens[b]) + int(paths[b][j]))
                moved.append((self.k[:, p, :, r].copy(), self.v[:, p, :, r].copy()))
            for j, (k, v) in enumerate(moved):
                p, r = self._rows(b, int(self.lens[b]) + j)
                self.k[:, p, :, r], self.v[:, p, :, r] = k, v
        return self.lens + np.asarray(counts, dtype=np.int32)

    def fork(self, src, dst):
        for s, d in zip(src, dst):
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] -= 1
            held = -(-int(self.lens[s]) // self.page)
            self.table[d] = -1
            self.table[d, :held] = self.table[s, :held]
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] += 1
            self.lens[d] = self.lens[s]

    def free(self, rows):
        for r in dict.fromkeys(rows):
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r] = -1
            self.lens[r] = 0

    def reserve(self, tokens):
        """Status; shared pages are counted as the call finds them."""
        wanted, status = [], 0
        for b, n in enumerate(tokens):
            if n == 0:
                continue
            if self.lens[b] + n > self.table.shape[1] * self.page:
                status |= 2
                continue
            for s in range(int(self.lens[b]) // self.page, (int(self.lens[b]) + n - 1) // self.page + 1):
                p = self.table[b, s]
                if p < 0 or self.refs[p] > 1:
                    wanted.append((b, s))
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        if len(free) < len(wanted):
            status |= 1
        if status:
            return status
        for (b, s), p in zip(wanted, free):
            old = self.table[b, s]
            if old >= 0:
                self.refs[old] -= 1
                rows = max(0, min(self.page, int(self.lens[b]) - s * self.page))
                self.k[:, p, :, :rows] = self.k[:, old, :, :rows]
                self.v[:, p, :, :rows] = self.v[:, old, :, :rows]
            self.refs[p] = 1
            self.table[b, s] = p
        return 0

    def compact(self):
        held = int((self.refs > 0).sum())
        holes = [p for p in range(held) if self.refs[p] <= 0]
        movers = [p for p in range(held, len(self.refs)) if self.refs[p] > 0]
        for h, m in zip(holes, movers):
            self.k[:, h], self.v[:, h] = self.k[:, m], self.v[:, m]
            self.refs[h], self.refs[m] = self.refs[m], 0
            self.table[self.table == m] = h
        return held

    def check(self, k, v, table, lens, refs):
        np.testing.assert_array_equal(table.cpu().numpy(), self.table)
        np.testing.assert_array_equal(refs.cpu().numpy(), self.refs)
        np.testing.assert_array_equal(lens.cpu().numpy(), self.lens)
        np.testing.assert_array_equal(k.float().cpu().numpy(), self.k)
        np.testing.assert_array_equal(v.float().cpu().numpy(), self.v)
