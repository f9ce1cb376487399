"""Plain float64 forms of the dense operators, and the bounds that follow from the kernels' roundings."""

import torch

PAGE = 16


def _attend(q, k, v):
    """q [hkv, g, d], k and v [hkv, s, d] -> (out, lse, weighted mean of |v|, largest sum |q_i k_i| / sqrt(d))."""
    scale = q.shape[-1] ** -0.5
    s = torch.einsum("hgd,hsd->hgs", q, k) * scale
    w = torch.softmax(s, dim=-1)
    mag = float((torch.einsum("hgd,hsd->hgs", q.abs(), k.abs()) * scale).max())
    return torch.einsum("hgs,hsd->hgd", w, v), torch.logsumexp(s, dim=-1), torch.einsum("hgs,hsd->hgd", w, v.abs()), mag


class Reference:
    def __init__(self, rows, hq, d):
        self.out = torch.zeros((rows, hq, d), dtype=torch.float64)
        self.mean_abs = torch.zeros((rows, hq, d), dtype=torch.float64)
        self.lse = torch.full((rows, hq), float("-inf"), dtype=torch.float64)
        self.mag, self.keys, self.d = 0.0, 0, d

    def row(self, i, q, k, v):
        hq = self.out.shape[1]
        o, lse, mean_abs, mag = _attend(q, k, v)
        self.out[i], self.mean_abs[i], self.lse[i] = o.reshape(hq, -1), mean_abs.reshape(hq, -1), lse.reshape(hq)
        self.mag, self.keys = max(self.mag, mag), max(self.keys, k.shape[1])

    def weight_error(self):
        """Relative error of a softmax weight in fp32, u = half a step = 2^-24: a logit is a sum of d products and a scaling,
        off by (d + 2) u times the sum of the products' magnitudes; exp turns that into a relative error, and
        numerator and denominator both have it; the sum over the keys adds keys * u to each; 16 u for the exponentials,
        rescalings and the division (2 units in the last place each)."""
        u = torch.finfo(torch.float32).eps / 2
        return 2 * (self.d + 2) * u * self.mag + 2 * self.keys * u + 16 * u

    def check(self, got, dtype):
        """bf16 adds one rounding of each weight before the second product and one of the result, half a step (2^-8
        relative) each."""
        half = torch.finfo(dtype).eps / 2
        bound = self.weight_error() * self.mean_abs + half * self.out.abs()
        if dtype == torch.bfloat16:
            bound = bound + half * self.mean_abs
        err = (got.double().cpu() - self.out).abs()
        worst = float((err - 1.01 * bound).max())   # second-order terms: a hundredth
        assert worst <= 0, f"off by {float(err.max()):.3g}, {worst:.3g} past the bound"

    def check_lse(self, got):
        got = got.double().cpu()
        assert torch.equal(torch.isinf(got), torch.isinf(self.lse))
        seen = ~torch.isinf(self.lse)
        u = torch.finfo(torch.float32).eps / 2
        bound = 1.01 * (self.weight_error() + 4 * u * self.lse[seen].abs())
        assert bool(((got[seen] - self.lse[seen]).abs() <= bound).all())


def prompt_reference(q, k, v, q_lens, kv_lens):
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    ref = Reference(q.shape[0], hq, d)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    q0 = k0 = 0
    for n, m in zip(q_lens, kv_lens):
        for t in range(n):
            seen = min(max(m - n + t + 1, 0), m)
            if seen:
                ref.row(q0 + t, q[q0 + t].view(hkv, hq // hkv, d), k[k0:k0 + seen].transpose(0, 1),
                        v[k0:k0 + seen].transpose(0, 1))
        q0, k0 = q0 + n, k0 + m
    return ref


def decode_reference(q, k_pool, v_pool, table, lens):
    hq, hkv, d = q.shape[1], k_pool.shape[1], q.shape[2]
    ref = Reference(q.shape[0], hq, d)
    k_pool, v_pool, table, q = k_pool.cpu(), v_pool.cpu(), table.cpu(), q.double().cpu()
    for b, n in enumerate(lens):
        if n:
            pages = table[b, :(n + PAGE - 1) // PAGE].long()
            ref.row(b, q[b].view(hkv, hq // hkv, d), k_pool[pages].double().transpose(0, 1).reshape(hkv, -1, d)[:, :n],
                    v_pool[pages].double().transpose(0, 1).reshape(hkv, -1, d)[:, :n])
    return ref


class PagesModel:
    """The page cache's rules on Python lists."""

    def __init__(self, n_pages, n_rows, max_pages):
        self.refs, self.rows, self.lens, self.max_pages = [0] * n_pages, [[] for _ in range(n_rows)], [0] * n_rows, max_pages
        self.contents = list(range(n_pages))     # what a page holds, as the number of the page it came from
        self.bad = self.full = False

    def _take(self, wants):
        """wants: pages wanted per entry -> pages per entry, or None from the first that does not fit on."""
        free, out, at = [p for p, r in enumerate(self.refs) if r == 0], [], 0
        for w in wants:
            at += w
            if at > len(free):
                self.full = True
            out.append(free[at - w:at] if at <= len(free) else None)
        return out

    def extend(self, rows, counts):
        wants, ok = [], []
        for i, (r, c) in enumerate(zip(rows, counts)):
            good = 0 <= r < len(self.rows) and r not in rows[:i] and 0 <= c <= self.max_pages * PAGE - self.lens[r]
            ok.append(good)
            self.bad |= not good
            wants.append(-(-(self.lens[r] + c) // PAGE) - len(self.rows[r]) if good else 0)
        for r, c, good, pages in zip(rows, counts, ok, self._take(wants)):
            if good and pages is not None:
                self.rows[r] += pages
                self.lens[r] += c
                for p in pages:
                    self.refs[p] = 1

    def fork(self, parents, children, share):
        before, lens = [list(r) for r in self.rows], list(self.lens)
        wants, ok = [], []
        for i, (p, c) in enumerate(zip(parents, children)):
            n = len(self.rows)
            good = 0 <= p < n and 0 <= c < n and p != c and c not in children[:i] and lens[c] == 0
            ok.append(good)
            self.bad |= not good
            kept = lens[p] // PAGE if good and share else 0
            wants.append(len(before[p]) - kept if good else 0)
        for p, c, good, pages in zip(parents, children, ok, self._take(wants)):
            if good and pages is not None:
                kept = before[p][:len(before[p]) - len(pages)]
                for x in kept:
                    self.refs[x] += 1
                for src, x in zip(before[p][len(kept):], pages):
                    self.refs[x] = 1
                    self.contents[x] = self.contents[src]
                self.rows[c], self.lens[c] = kept + pages, lens[p]

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.rows):
                self.bad = True
                continue
            for p in self.rows[r]:
                self.refs[p] -= 1
            self.rows[r], self.lens[r] = [], 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        movers = [p for p in range(n, len(self.refs)) if self.refs[p]]
        holes = [p for p in range(n) if not self.refs[p]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.contents[b] = self.refs[a], 0, self.contents[a]
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
