"""The operators of a paged cache on the CPU: the table as lists, one row after another, the attention in 64 bits, and
the bounds that the GPU results are held to.

Rounding of a type is off by at most u = eps / 2 of the value.  A level of the attention, per token:

* a score is a product of d terms summed in fp32 (d + 2 roundings of 2^-24 of sum |q k|), scaled, clamped and
  shifted by a bias (4 more of its size), then exp2 in fp32 (2^-22 relative): a weight and the weights' sum are
  off by at most r = 2 (largest score error) + 2^-21, relatively;
* in 16-bit types the weights enter the second product rounded to the type: u;
* the sum itself: (n + 64) 2^-24 for n terms in fp32;
* the level below: its stored averages' bounds enter linearly, its logsumexps' bound b as 2 b in r;
* a product with the next level's projected values: 2^-24 of it;
* the stored result is rounded once: u of it, and where the type's steps stop shrinking (below its smallest normal
  number tiny) u tiny.

The definition has the next level read what is stored.  The oracle keeps its averages unrounded and counts the
rounding among their bounds, so that it need not round as the kernel did.
"""

import math

import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def stored(y, dtype):
    """Half a step of the type at y."""
    return unit(dtype) * y.abs().clamp(min=torch.finfo(dtype).tiny)


class Table:
    """The state of a PageTable in lists, and its calls one row after another."""

    def __init__(self, rows, pool, page_size, capacity):
        self.ps, self.most = page_size, -(-capacity // page_size)
        self.pages = [[] for _ in range(rows)]
        self.counts, self.new = [0] * rows, [0] * rows
        self.starts = [0] * (rows + 1)
        self.refs = [0] * pool
        self.overflow = False

    def need(self, n):
        return -(-n // self.ps)

    def extend(self, more):
        """Copies as a list of (from, to, positions)."""
        free = [p for p, r in enumerate(self.refs) if r == 0]
        copies, asked, at = [], [], 0
        starved = False  # a row did not get its pages: neither does any behind it that needs some
        for b, m in enumerate(more):
            asked.append(max(m, 0))
            m = max(m, 0)
            self.new[b] = 0
            n = self.counts[b]
            if n + m > self.most * self.ps:
                self.overflow = True
                continue
            if m == 0:
                continue
            tail = self.pages[b][-1] if n % self.ps else None
            # rows before this one that were about to write the page and could not leave it
            waits = tail is not None and tail in getattr(self, "_stuck", ())
            copy = tail is not None and self.refs[tail] > 1
            want = self.need(n + m) - self.need(n) + copy
            if (want and (starved or want > len(free) - at)) or waits:
                starved = True
                self.overflow = True
                if tail is not None:
                    self._stuck = (*getattr(self, "_stuck", ()), tail)
                continue
            if copy:
                to = free[at]
                at += 1
                copies.append((tail, to, n % self.ps))
                self.refs[tail] -= 1
                self.refs[to] = 1
                self.pages[b][-1] = to
            for _ in range(self.need(n + m) - self.need(n)):
                self.pages[b].append(free[at])
                self.refs[free[at]] = 1
                at += 1
            self.counts[b] = n + m
            self.new[b] = m
        self._stuck = ()
        self.starts = [sum(asked[:k]) for k in range(len(asked) + 1)]
        return copies

    def select(self, index, lengths=None):
        pages, counts = [], []
        for b, i in enumerate(index):
            n = self.counts[i] if 0 <= i < len(index) else 0
            if lengths is not None:
                n = min(n, max(lengths[b], 0))
            pages.append(self.pages[i][:self.need(n)] if n else [])
            counts.append(n)
        self.pages, self.counts, self.new = pages, counts, [0] * len(index)
        self.refs = [0] * len(self.refs)
        for row in pages:
            for p in row:
                self.refs[p] += 1

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        self.pages = [[to.get(p, p) for p in row] for row in self.pages]
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        return list(zip(movers, holes))

    def check(self, table):
        """Everything a PageTable holds is as here."""
        most = table.pages.shape[1]
        assert table.counts.tolist() == self.counts
        assert table.pages.tolist() == [row + [-1] * (most - len(row)) for row in self.pages]
        assert table.refs.tolist() == self.refs
        assert table.new.tolist() == self.new


def row_of(array, pages, n, ps):
    """Positions 0 .. n of a row, [heads, n, ...], of an array of pages."""
    if n == 0:
        return array[:0].transpose(0, 1).flatten(1, 2)
    return torch.cat([array[p] for p in pages], 1)[:, :n]


def put(array, pages, p, x, ps):
    array[pages[p // ps], :, p % ps] = x


def places(starts, new, packed):
    """(row, token of the row, batch row of the inputs, token of the inputs)."""
    for b, m in enumerate(new):
        for i in range(m):
            yield b, i, (0 if packed else b), (starts[b] + i if packed else i)


def attend(q1, vs, cache, table, packed, scale, softclamp):
    """Results and bounds from CPU copies: cache a dict of keys, values, lses; table a Table.  (out, values, lses) as
    (result, bound) pairs, values and lses whole arrays in 64 bits whose untouched places are what they were."""
    H, d = q1.shape[1], q1.shape[3]
    hk, order, ps = cache["keys"][0].shape[1], len(cache["keys"]), table.ps
    dt = q1.dtype
    up = unit(dt) if dt != torch.float32 else 0.0
    rep = H // hk
    out = torch.zeros(q1.shape, dtype=torch.float64)
    out_tol = torch.zeros_like(out)
    values = [x.double() for x in cache["values"]]
    values_tol = [torch.zeros_like(x) for x in values]
    lses = [x.double() for x in cache["lses"]]
    lses_tol = [torch.zeros_like(x) for x in lses]
    for b, m in enumerate(table.new):
        if m == 0:
            continue
        n, pages = table.counts[b], table.pages[b]
        first, src, tok = n - m, 0 if packed else b, table.starts[b] if packed else 0
        pos = torch.arange(first, n)
        hidden = torch.arange(n) > pos[:, None]
        page = torch.tensor(pages)[pos // ps]
        for t in range(order):
            last = t == order - 1
            k = row_of(cache["keys"][t], pages, n, ps).double()
            v, v_tol = row_of(values[t], pages, n, ps), row_of(values_tol[t], pages, n, ps)
            if last:
                q = q1[src, :, tok:tok + m].double().view(hk, rep, m, d)
            else:
                q = row_of(cache["keys"][t + 1], pages, n, ps)[:, first:].double()[:, None]
            raw = torch.einsum("grid,gjd->grij", q, k) * scale
            off = (d + 2) * F32 * torch.einsum("grid,gjd->grij", q.abs(), k.abs()) * abs(scale)
            s = softclamp * torch.tanh(raw / softclamp) if softclamp else raw
            bias_tol = 0.0
            if t:
                bias = row_of(lses[t - 1], pages, n, ps)[:, None, None]
                bias_tol = row_of(lses_tol[t - 1], pages, n, ps)[:, None, None]
                s = s + bias
                off = off + 4 * F32 * bias.abs()
            off = off + 6 * F32 * (raw.abs() + s.abs()) + bias_tol
            s = s.masked_fill(hidden, -math.inf)
            off = off.masked_fill(hidden, 0.0).amax(-1)             # [g, r, i]
            z = torch.logsumexp(s, -1)
            w = torch.exp(s - z[..., None])
            v = torch.where(hidden[:, :, None].all(0)[None], 0.0, v)
            # a token's own mask: what it does not see may be no number
            clean = torch.where(torch.isfinite(v), v, 0.0)
            o = torch.einsum("grij,gjd->grid", w, clean)
            size = torch.einsum("grij,gjd->grid", w, clean.abs())
            below = torch.einsum("grij,gjd->grid", w, v_tol)
            rel = (2 * off + 2.0 ** -21 + (n + 64) * F32 + up)[..., None]
            tol = size * rel + below * (1 + rel)
            z_tol = off + 2.0 ** -21 + (n + 64) * F32 + 6 * F32 * z.abs()
            if last:
                o, tol = (x.reshape(H, m, d) for x in (o, tol))
                out[src, :, tok:tok + m] = o
                out_tol[src, :, tok:tok + m] = tol + stored(o.abs() + tol, dt)
                continue
            o, tol, z, z_tol = o[:, 0], tol[:, 0], z[:, 0], z_tol[:, 0]
            if t + 1 < order - 1:
                by = vs[order - 3 - t][src, :, tok:tok + m].double()
                o, tol = o * by, tol * by.abs() + F32 * (o * by).abs()
            tol = tol + stored(o.abs() + tol, dt)
            for i in range(m):
                values[t + 1][page[i], :, pos[i] % ps] = o[:, i]
                values_tol[t + 1][page[i], :, pos[i] % ps] = tol[:, i]
                lses[t][page[i], :, pos[i] % ps] = z[:, i]
                lses_tol[t][page[i], :, pos[i] % ps] = z_tol[:, i]
    return (out, out_tol), list(zip(values, values_tol)), list(zip(lses, lses_tol))


def append(q, weight, eps, angles, dtype):
    """A token's norm and rotation, [heads, d] -> (result, bound): the mean of squares is a sum of d terms in fp32
    ((d + 2) 2^-24 of it, half of that in its root), rsqrt and three products 8 2^-24 more; a rotation two products and a
    sum of sines and cosines that are 2^-22 off; the result is rounded once."""
    x = q.double()
    d = x.shape[-1]
    if weight is not None:
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    else:
        y = x
    tol = y.abs() * (d / 2 + 10) * F32
    if angles is not None and angles.numel():
        r = angles.numel()
        a = angles.double()
        z, zt = y[:, :r], tol[:, :r]
        turned = torch.stack([-z[:, 1::2], z[:, 0::2]], -1).flatten(-2)
        swap = torch.stack([zt[:, 1::2], zt[:, 0::2]], -1).flatten(-2)
        y = torch.cat([z * a.cos() + turned * a.sin(), y[:, r:]], -1)
        extra = (z.abs() + turned.abs()) * (2.0 ** -22 + 4 * F32)
        tol = torch.cat([zt + swap + extra, tol[:, r:]], -1)
    return y, tol + stored(y.abs() + tol, dtype)
