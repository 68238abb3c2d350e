"""Restatement in 64 bits of the serving operators: rotary positions, the 4-bit paged cache and
the attention over it, and the bookkeeping of its pages.  Plain loops over sequences and heads,
written from the definitions; test infrastructure only."""
from __future__ import annotations

import math

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def rotary(x, positions, radians, *, head_dim, interleaved=False, magnitude=1.0, in_scale=1.0,
           weight=None, weight_offset=1.0, eps=1e-6, inverse=False):
    """x [rows, heads * head_dim] -> f64 of the same shape."""
    y = x.double().unflatten(-1, (-1, head_dim)) * in_scale
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (weight.double()
                                                                       + weight_offset)
    w = torch.tensor(radians, dtype=torch.float64)
    a = positions.double()[:, None, None] * w * (-1 if inverse else 1)
    n = 2 * len(radians)
    out = y.clone()
    first = slice(0, n, 2) if interleaved else slice(0, n // 2)
    second = slice(1, n, 2) if interleaved else slice(n // 2, n)
    out[..., first] = magnitude * (y[..., first] * a.cos() - y[..., second] * a.sin())
    out[..., second] = magnitude * (y[..., second] * a.cos() + y[..., first] * a.sin())
    return out.flatten(1)


def pack(x, scale):
    """x [..., D] -> (codes [..., D] in 0..15, scale bytes [..., D / 16], values f64)."""
    g = x.double().unflatten(-1, (-1, 16))
    s8 = (g.abs().amax(-1) / (6 * scale)).clamp(max=448).float().to(torch.float8_e4m3fn)
    s = (s8.double() * scale).unsqueeze(-1)
    y = torch.where(s > 0, g / s, torch.zeros_like(g)).clamp(-6, 6)
    grid = torch.tensor(E2M1, dtype=torch.float64)
    far = (y.abs().unsqueeze(-1) - grid).abs()
    # nearest; of two equally near the one with the even code
    code = torch.argmin(far + 1e-9 * (torch.arange(8) % 2) * (far == far.amin(-1, keepdim=True)), -1)
    value = grid[code] * torch.where(torch.signbit(y), -1.0, 1.0) * s
    code = code + 8 * torch.signbit(y)
    return code.flatten(-2), s8.view(torch.uint8), value.flatten(-2)


def unpack_block(block, page_size, head_dim, k_scale, v_scale):
    """uint8 [..., page_size * head_dim * 9 / 8] -> K, V f64 [..., page_size, head_dim]."""
    c, s = page_size * head_dim // 2, page_size * head_dim // 16
    grid = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64)
    out = []
    for part, scale in ((block[..., :c + s], k_scale), (block[..., c + s:], v_scale)):
        codes, scales = part[..., :c], part[..., c:]
        v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
        f = scales.contiguous().view(torch.float8_e4m3fn).double() * scale
        v = v.unflatten(-1, (-1, 16)) * f.unsqueeze(-1)
        out.append(v.flatten(-2).unflatten(-1, (page_size, head_dim)))
    return out


def cached(storage, table_row, length, page_size, head_dim, k_scale, v_scale):
    """K, V f64 [length, kv_heads, head_dim] of one sequence of one layer."""
    pages = [int(p) for p in table_row[:-(-length // page_size)]]
    k, v = unpack_block(storage[pages], page_size, head_dim, k_scale, v_scale)
    flat = lambda x: x.transpose(1, 2).flatten(0, 1)[:length]  # noqa: E731
    return flat(k), flat(v)


def attention(q, k, v, *, causal=True, sm_scale=None, gate=None):
    """q f64 [n, Hq, D] (the last n tokens), k, v f64 [L, Hk, D] -> (out [n, Hq, D], lse [n, Hq],
    sum of p |v| / sum of p, the sum of |q k| of the largest kind).  What a token may not see
    does not enter its sums."""
    n, hq, d = q.shape
    length, hk = k.shape[:2]
    out = torch.zeros_like(q)
    mass = torch.zeros_like(q)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    size = 0.0
    scale = 1 / math.sqrt(d) if not sm_scale else sm_scale
    for i in range(n):
        seen = max(0, length - n + i + 1) if causal else length
        if seen == 0:
            continue
        for h in range(hq):
            g = h * hk // hq
            s = k[:seen, g] @ q[i, h] * scale
            size = max(size, float((k[:seen, g].abs() @ q[i, h].abs()).nan_to_num().max()) * scale)
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[i, h])
            out[i, h] = p @ v[:seen, g]
            mass[i, h] = p @ v[:seen, g].abs()
    if gate is not None:
        gate = torch.sigmoid(gate.double())
        out, mass = out * gate, mass * gate
    return out, lse, mass, size


class Pages:
    """The bookkeeping of the pages in plain Python."""

    def __init__(self, pages, rows, cols, page_size):
        self.refs, self.page = [0] * pages, page_size
        self.table, self.lens = [[-1] * cols for _ in range(rows)], [0] * rows
        self.copies = []

    def _take(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(free) < n:
            return None
        for p in free[:n]:
            self.refs[p] = 1
        return free[:n]

    def extend(self, rows, counts):
        ceil = lambda n: -(-n // self.page)  # noqa: E731
        if len(set(rows)) < len(rows) or any(not 0 <= r < len(self.lens) for r in rows) or any(
                c < 0 or self.lens[r] + c > len(self.table[r]) * self.page
                for r, c in zip(rows, counts)):
            return False
        need = [ceil(self.lens[r] + c) - ceil(self.lens[r]) for r, c in zip(rows, counts)]
        got = self._take(sum(need))
        if got is None:
            return False
        for r, c, n in zip(rows, counts, need):
            at = ceil(self.lens[r])
            self.table[r][at:at + n] = got[:n]
            got = got[n:]
            self.lens[r] += c
        return True

    def fork(self, src, dst):
        n = len(self.lens)
        if len(set(dst)) < len(dst) or set(src) & set(dst) or any(
                not 0 <= r < n for r in src + dst) or any(self.lens[d] for d in dst):
            return False
        got = self._take(sum(self.lens[s] % self.page > 0 for s in src))
        if got is None:
            return False
        for s, d in zip(src, dst):
            full = self.lens[s] // self.page
            for c in range(full):
                self.table[d][c] = self.table[s][c]
                self.refs[self.table[s][c]] += 1
            if self.lens[s] % self.page:
                self.table[d][full] = got.pop(0)
                self.copies.append((self.table[s][full], self.table[d][full]))
            self.lens[d] = self.lens[s]
        return True

    def free(self, rows):
        for r in rows:
            for c in range(-(-self.lens[r] // self.page)):
                self.refs[self.table[r][c]] -= 1
                self.table[r][c] = -1
            self.lens[r] = 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        moves = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(moves, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.copies.append((a, b))
        self.table = [[to.get(p, p) for p in row] for row in self.table]
