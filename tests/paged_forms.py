"""The paged-cache operators in 64 bits on the CPU, row by row from their definitions, and random caches to try them on."""
from __future__ import annotations

import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype) -> float:
    """Largest relative error of one rounding to the type."""
    return torch.finfo(dtype).eps / 2


def frequencies(n_rot, base=1.0e6, scaling="none", factor=1.0, original_context=32768, beta_fast=32.0, beta_slow=1.0,
                attention_factor=0.0):
    """(angle per position of each pair, size of the rotated values)"""
    f, size = [], 1.0
    if scaling == "ntk":
        base = base * factor ** (n_rot / (n_rot - 2))
    if scaling == "yarn":
        size = attention_factor or 0.1 * math.log(factor) + 1
        lo, hi = (n_rot * math.log(original_context / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (beta_fast, beta_slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n_rot - 1)
    for i in range(n_rot // 2):
        w = base ** (-2 * i / n_rot)
        if scaling == "linear":
            w /= factor
        if scaling == "yarn":
            r = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            w = w * (1 - r) + w / factor * r
        f.append(w)
    return torch.tensor(f, dtype=torch.float64), size


def rotate(x, positions, n_rot, layout="half", **kw):
    """x [rows, heads, dim] (any type) rotated, f64, and the bound |a| + |b| of each rotated value's terms."""
    f, size = frequencies(n_rot, **kw)
    y = x.double().clone()
    terms = torch.zeros_like(y)
    angle = positions.double()[:, None] * f
    c, s = (angle.cos() * size)[:, None], (angle.sin() * size)[:, None]
    i = torch.arange(n_rot // 2)
    lo, hi = (i, i + n_rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    terms[..., lo] = terms[..., hi] = (a.abs() + b.abs()) * size
    return y, terms


# Rotated values: cos and sin carry the rounding of the angle to a float (2^-25 half turns, 9.4e-8 rad) and sincospi's own
# error (below 2 steps, 1.2e-7), the size, products and sum three more roundings of 2^-24: below 4.0e-7 of |a| + |b|.
ROTATION = 4.0e-7


def rotation_bound(y, terms, dtype):
    # the smallest normal's step covers results below f16's normal range
    return half_step(dtype) * (y.abs() + ROTATION * terms) + ROTATION * terms + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


class Sequences:
    """A random cache and step. rows[s] new rows of sequence s, lengths[s] slots with them; pages in random order, the
    pool padded with pages of nobody; absent: (sequence, page number) pairs whose table entry is no page."""

    def __init__(self, rows, lengths, kv_heads, dim, page, dtype, seed=0, order="pages", absent=(), pad_rows=0, extra_pages=3,
                 wide_table=0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.page, self.kv_heads, self.dim, self.dtype = list(rows), list(lengths), page, kv_heads, dim, dtype
        per = max(1, -(-max(lengths) // page)) + wide_table
        self.n_pages = len(self.rows) * per + extra_pages
        self.table = torch.randperm(self.n_pages, generator=g)[:len(self.rows) * per].to(torch.int32).reshape(len(self.rows), per)
        for n, (s, p) in enumerate(absent):
            self.table[s, p] = [-1, self.n_pages, 2**31 - 1, -2**31][n % 4]
        starts = [0]
        for r in self.rows:
            starts.append(starts[-1] + r)
        self.starts, self.total = starts, starts[-1] + pad_rows
        self.row_starts = torch.tensor(starts, dtype=torch.int32)
        self.lengths = torch.tensor(self.lens, dtype=torch.int32)
        self.order = order
        size = (self.n_pages, kv_heads, page, dim)
        self.k = torch.randn(size, generator=g).to(dtype)
        self.v = torch.randn(size, generator=g).to(dtype)
        self.weights = torch.rand(size[:3], generator=g)
        self.positions = torch.randint(0, 1 << 20, size[:3], generator=g, dtype=torch.int32)
        self.max_rows, self.max_length = max(self.rows), max(self.lens)

    def slot(self, s, t):
        """(page, place) of slot t of sequence s, None on an absent page."""
        p = int(self.table[s, t // self.page])
        return (p, t % self.page) if 0 <= p < self.n_pages else None

    def to_gpu(self):
        """The pool on the GPU (as [pages, heads, page, dim] views of storage in the asked order), table, lengths, starts."""
        def pool(x):
            if self.order == "tokens":  # [pages, page, heads, dim]
                return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            if self.order == "padded":  # heads and slots further apart than they need to be
                big = torch.zeros(x.shape[0], x.shape[1] + 1, x.shape[2] + 2, x.shape[3] + 8, dtype=x.dtype)
                big[:, :x.shape[1], :x.shape[2], :x.shape[3]] = x
                return big.cuda()[:, :x.shape[1], :x.shape[2], :x.shape[3]]
            return x.cuda()
        return (pool(self.k), pool(self.v), self.weights.cuda(), self.positions.cuda(), self.table.cuda(),
                self.lengths.cuda(), self.row_starts.cuda())

    def rows_of(self, s):
        """(row, slot) of the sequence's new rows that have a slot."""
        for i in range(self.rows[s]):
            t = self.lens[s] - self.rows[s] + i
            if t >= 0:
                yield self.starts[s] + i, t

    def poison(self):
        """NaN and infinities in every slot that no sequence uses, and in the pages of nobody."""
        used = torch.zeros(self.n_pages, self.page, dtype=torch.bool)
        for s in range(len(self.rows)):
            for t in range(self.lens[s]):
                at = self.slot(s, t)
                if at is not None:
                    used[at] = True
        bad = ~used[:, None, :, None].expand_as(self.k)
        values = torch.tensor([math.nan, math.inf, -math.inf], dtype=self.dtype).repeat(self.k.numel() // 3 + 1)
        self.k[bad] = values[:self.k.numel()].reshape(self.k.shape)[bad]
        self.v[bad] = values[1:self.k.numel() + 1].reshape(self.k.shape)[bad]
        return self

    def gather(self, s):
        """K and V [K/V heads, slots, dim] (f64) of a sequence, and which slots are there."""
        n = self.lens[s]
        k, v = (torch.zeros(self.kv_heads, n, self.dim, dtype=torch.float64) for _ in range(2))
        there = torch.zeros(n, dtype=torch.bool)
        for p in range(-(-n // self.page)):
            at = self.slot(s, p * self.page)
            t0, t1 = p * self.page, min(n, (p + 1) * self.page)
            if at is not None:
                k[:, t0:t1], v[:, t0:t1] = self.k[at[0], :, :t1 - t0].double(), self.v[at[0], :, :t1 - t0].double()
                there[t0:t1] = True
        return k, v, there

    def sees(self, s, causal, there):
        """[rows, slots] what each new row of a sequence sees."""
        n, r = self.lens[s], self.rows[s]
        t = torch.arange(n)
        end = torch.arange(n - r + 1, n + 1)[:, None] if causal else torch.full((r, 1), n)
        return (t < end) & there

    def attend(self, q, scale, causal=True):
        """out, lse (f64) and their bounds for q [rows, heads, dim]."""
        group = q.shape[1] // self.kv_heads
        out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
        bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
        step, tiny = half_step(self.dtype), 2.0**-25 if self.dtype == torch.float16 else 0.0
        for s in range(len(self.rows)):
            k, v, there = self.gather(s)
            sees = self.sees(s, causal, there)
            r = slice(self.starts[s], self.starts[s + 1])
            for h in range(q.shape[1]):
                x, kh, vh = q[r, h].double(), k[h // group], v[h // group]
                score = (x @ kh.T * scale).masked_fill(~sees, -math.inf)
                # a score: dim products and sums in f32, its product with the scale and the difference to the maximum
                off = ((self.dim + 2) * 2.0**-24 * scale * (x.abs() @ kh.abs().T) + 2.0**-22 * score.abs()).masked_fill(~sees, 0)
                off = off.amax(-1, keepdim=True) if off.shape[1] else torch.zeros(len(x), 1)
                some = sees.any(-1)
                lse[r, h] = torch.logsumexp(score, -1)
                p = torch.where(some[:, None], torch.softmax(score, -1), 0.0)
                p = torch.where(sees, p, 0.0)
                n = sees.shape[1]
                out[r, h] = p @ vh
                size = p @ vh.abs()
                # weights: a half step of their rounding, their score, exp2 (2^-22); sums of n terms and 64 parts in f32
                bound[r, h] = size * (step + 2 * off + 2.0**-21 + (n + 64) * 2.0**-23)
                bound[r, h] += tiny * (sees.double() @ vh.abs())  # weights below f16's normal range, of a sum of 1 at least
                bound[r, h] += step * (out[r, h].abs() + bound[r, h]) + 2.0**-25
                lse_bound[r, h] = off[:, 0] + 2.0**-21 + (n + 64) * 2.0**-23 + 2.0**-22 * lse[r, h].abs().nan_to_num(posinf=0)
        return out, lse, bound, lse_bound

    def weigh(self, q, lse, scale, causal=True):
        """weights (f64) after the rows q with lse [rows, heads] (float32), and their bounds."""
        group = q.shape[1] // self.kv_heads
        w, bound = self.weights.double().clone(), torch.zeros(self.weights.shape, dtype=torch.float64)
        for s in range(len(self.rows)):
            k, _, there = self.gather(s)
            sees = self.sees(s, causal, there)
            r = slice(self.starts[s], self.starts[s + 1])
            sums, offs = torch.zeros(self.kv_heads, self.lens[s], dtype=torch.float64), torch.zeros(self.kv_heads, self.lens[s])
            for h in range(q.shape[1]):
                x, kh, l = q[r, h].double(), k[h // group], lse[r, h].double()[:, None]
                score = x @ kh.T * scale
                p = torch.where(sees & (l > -math.inf), torch.exp(score - l), 0.0)
                # as for attention's scores, and the rounding of lse in base 2
                off = (self.dim + 2) * 2.0**-24 * scale * (x.abs() @ kh.abs().T) + 2.0**-22 * (score.abs() + l.abs()) + 2.0**-21
                sums[h // group] += p.sum(0)
                offs[h // group] += torch.where(p > 0, p * off, 0.0).sum(0)
            terms = self.rows[s] * group / 16 + 24  # sums of a lane, over lanes and into the total
            for t in range(self.lens[s]):
                at = self.slot(s, t)
                if at is not None:
                    w[at[0], :, at[1]] += sums[:, t]
                    bound[at[0], :, at[1]] = offs[:, t] + (terms * sums[:, t] + w[at[0], :, at[1]].abs()) * 2.0**-24
        return w, bound

    def evict(self, budget, first, recent):
        """k, v, weights, positions and lengths after a cut."""
        k, v, w, pos = self.k.clone(), self.v.clone(), self.weights.clone(), self.positions.clone()
        lens = [min(n, budget) for n in self.lens]
        for s, n in enumerate(self.lens):
            if n <= budget:
                continue
            at = [self.slot(s, t) for t in range(n)]
            for h in range(self.kv_heads):
                there = [t for t in range(n) if at[t] is not None]
                newest = max((int(self.positions[at[t][0], h, at[t][1]]) for t in there), default=0)

                def order(t):
                    if at[t] is None:  # holds its place below the budget, never moves
                        return (0 if t < budget else 3, 0, 0.0, t)
                    p, weight = int(self.positions[at[t][0], h, at[t][1]]), float(self.weights[at[t][0], h, at[t][1]])
                    kind = 1 if p < first or p > newest - recent else 2
                    return (kind, 1, 0.0, t) if math.isnan(weight) else (kind, 0, -weight, t)

                stay = set(sorted(range(n), key=order)[:budget])
                to = [t for t in range(budget) if t not in stay]
                come = [t for t in range(budget, n) if t in stay]
                assert len(to) == len(come)
                for a, b in zip(to, come):
                    for x, y in ((k, self.k), (v, self.v), (w, self.weights), (pos, self.positions)):
                        x[at[a][0], h, at[a][1]] = y[at[b][0], h, at[b][1]]
        return k, v, w, pos, lens
