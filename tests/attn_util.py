"""Plain 64-bit attention over a paged cache, its error bound, and builders for the GPU tests."""
import math

import torch

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS32 = 2.0 ** -24  # half a step of f32, relative


def lengths_to_start(rows):
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    return start


class Setup:
    """A cache, its page lists and the new rows of some sequences, built on the CPU (so the reference
    reads them there) and copied to `dev`.

    kv: cached tokens of each sequence with the new ones; rows: new rows of each (None: decode).
    order "hnd" ([page][head][token]), "nhd" ([page][token][head]) or "mixed" (keys and values of a
    page side by side, padded).  junk: what every place holds that no sequence uses."""

    def __init__(self, hq, hkv, d, page, type, kv, rows=None, order="hnd", junk=float("nan"), seed=0, spare=3,
                 q_scale=1.5, extra_rows=0, pad_pages=2, dev="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.page, self.type = hq, hkv, d, page, TYPES[type]
        self.kv, self.rows = list(kv), None if rows is None else list(rows)
        need = [-(-max(n, 0) // page) for n in kv]
        self.wide = max(need + [1]) + pad_pages
        n_pages = sum(need) + spare
        perm = torch.randperm(n_pages, generator=g).tolist()
        # behind a list's last used page: ids far outside, never to be read
        self.pages = torch.full((len(kv), self.wide), 2 ** 30 + 7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.pages[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.unused = perm[at:]
        self.n_rows = (len(kv) if rows is None else sum(rows)) + extra_rows
        self.K = [torch.randn(max(n, 0), hkv, d, generator=g).to(self.type) for n in kv]
        self.V = [(torch.randn(max(n, 0), hkv, d, generator=g) + 0.2).to(self.type) for n in kv]
        self.q = (q_scale * torch.randn(self.n_rows, hq, d, generator=g)).to(self.type)
        self.start = None if rows is None else torch.tensor(lengths_to_start(rows), dtype=torch.int32)
        self.kv_len = torch.tensor(self.kv, dtype=torch.int32)
        self.order, self.junk, self.n_pages, self.dev = order, junk, n_pages, dev

    def pools(self, filled=True):
        """(k, v) views [n_pages][hkv][page][d] on the device in the wanted order."""
        n, h, p, d = self.n_pages, self.hkv, self.page, self.d
        if self.order == "hnd":
            k, v = (torch.full((n, h, p, d), self.junk, dtype=self.type) for _ in range(2))
        elif self.order == "nhd":
            k, v = (torch.full((n, p, h, d), self.junk, dtype=self.type).transpose(1, 2) for _ in range(2))
        else:
            both = torch.full((n, 2, h, p, d + 8), self.junk, dtype=self.type)
            k, v = both[:, 0, :, :, :d], both[:, 1, :, :, :d]
        if filled:
            for b, m in enumerate(self.kv):
                for t in range(max(m, 0)):
                    pg = int(self.pages[b, t // self.page])
                    k[pg, :, t % self.page] = self.K[b][t]
                    v[pg, :, t % self.page] = self.V[b][t]
        if self.order == "hnd":
            return k.to(self.dev), v.to(self.dev)
        if self.order == "nhd":
            return tuple(x.transpose(1, 2).contiguous().to(self.dev).transpose(1, 2) for x in (k, v))
        both = both.to(self.dev)
        return both[:, 0, :, :, :d], both[:, 1, :, :, :d]

    def seqs(self, pkg):
        start = None if self.start is None else self.start.to(self.dev)
        return pkg.SeqBatch(self.pages.to(self.dev), self.kv_len.to(self.dev), start,
                            None if start is None else self.n_rows)

    def context(self, pkg, max_seqs=None):
        return pkg.AttnContext(self.hq, self.hkv, self.d, self.page, max_seqs or len(self.kv), dtype=self.type)

    def row_seen(self):
        """(row, sequence, tokens it sees) of every row of a sequence."""
        if self.rows is None:
            return [(b, b, max(n, 0)) for b, n in enumerate(self.kv)]
        out, row = [], 0
        for b, (r, n) in enumerate(zip(self.rows, self.kv)):
            for i in range(r):
                out.append((row, b, max(0, n - r + i + 1)))
                row += 1
        return out

    def reference(self, scale=None, only=None):
        """(o, bound, lse, lse_bound) in 64 bits; rows of no sequence stay NaN in o.

        bound, element by element, of a kernel that holds scores, maxima, sums and products in f32,
        rounds each softmax weight to the type and the result once:
          scores: f32 products are exact, their sum of d terms and the scaling by two more
            roundings are off by e_s <= (d + 4) 2^-24 scale sum |q_i k_i|;
          weights: e^s off by a factor of e_s + 2^-22 (base-2 exponential, its argument's
            subtraction under 2^-23 |s - m|), over the sum's, so twice that;
          sums of n weights or products: (n + 64) 2^-24 (every order of summation, the rescaling of a
            running maximum and the joining of pieces included), twice;
          the weight's rounding: u = eps / 2 of the type, and where f16 runs out of exponent half a step of
            its smallest numbers, 2^-25, over what the largest weight is scaled to: 2^15 in the decode
            form (2^-40), 2^7 at least in the prompt form (2^-32); the result's: u |o|."""
        scale = self.d ** -0.5 if scale is None else scale
        u = torch.finfo(self.type).eps / 2
        tiny = torch.finfo(self.type).smallest_normal * torch.finfo(self.type).eps / 2
        lost = 2.0 ** -40 if self.rows is None else 2.0 ** -32
        group = self.hq // self.hkv
        o = torch.full((self.n_rows, self.hq, self.d), float("nan"), dtype=torch.float64)
        bound = torch.zeros_like(o)
        lse = torch.full((self.n_rows, self.hq), float("nan"), dtype=torch.float64)
        lse_bound = torch.zeros_like(lse)
        K = [x.double().repeat_interleave(group, 1).permute(1, 0, 2) for x in self.K]  # [hq][n][d]
        V = [x.double().repeat_interleave(group, 1).permute(1, 0, 2) for x in self.V]
        for row, b, n in self.row_seen():
            if only is not None and row not in only:
                continue
            if n == 0:
                o[row], lse[row] = 0.0, -math.inf
                continue
            q = self.q[row].double().unsqueeze(1)  # [hq][1][d]
            k, v = K[b][:, :n], V[b][:, :n]
            s = scale * (q * k).sum(-1)
            e_s = (self.d + 4) * EPS32 * abs(scale) * (q.abs() * k.abs()).sum(-1)
            m = s.amax(-1, keepdim=True)
            e_w = (e_s + e_s.amax(-1, keepdim=True) + 2.0 ** -22 + (s - m).abs() * 2.0 ** -22)
            w = torch.softmax(s, -1)
            off = (w * e_w).sum(-1, keepdim=True) + 2 * (n + 64) * EPS32
            o[row] = (w.unsqueeze(-1) * v).sum(1)
            av = v.abs()
            mass = (w.unsqueeze(-1) * av).sum(1)
            bound[row] = (u * o[row].abs() + (u + off) * mass * (1 + u) + (w * e_w).unsqueeze(-1).mul(av).sum(1)
                          + lost * av.sum(1) + tiny)
            lse[row] = torch.logsumexp(s, -1)
            lse_bound[row] = off.squeeze(-1) + 4 * EPS32 * (1 + lse[row].abs() + m.squeeze(-1).abs())
        return o, bound, lse, lse_bound


def check(name, got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bound, first {at}: {float(got[at])} "
                             f"for {float(want[at])}, bound {float(bound[at]):.3g}")
