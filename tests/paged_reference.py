"""Plain implementations of the paged cache's operators for the tests: attention in 64 bits, page bookkeeping as loops
over Python integers, written from the operators' documentation."""

import math

import numpy as np
import torch

DONE, INVALID, NO_ROOM, NOT_OWN = 0, 1, 2, 3


class Cache:
    """A paged cache on the CPU with any contents (numpy): what a test starts from and what it expects."""

    def __init__(self, layers, pages, kv_heads, ps, dim, seqs, max_pages, seed=0, dtype=torch.bfloat16):
        self.ps, self.pages, self.max_pages, self.dtype = ps, pages, max_pages, dtype
        g = torch.Generator().manual_seed(seed)
        shape = (layers, pages, kv_heads, ps, dim)
        self.k, self.v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        self.table = np.full((seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__.update(self.__dict__)
        c.k, c.v, c.table, c.lens, c.refs = self.k.clone(), self.v.clone(), self.table.copy(), self.lens.copy(), self.refs.copy()
        return c

    def hold(self, seq, length, ids):
        """Sequence seq gets `length` positions on the pages `ids`."""
        n = -(-length // self.ps)
        self.table[seq, :n] = ids[:n]
        self.lens[seq] = length
        for p in ids[:n]:
            if 0 <= p < self.pages:
                self.refs[p] += 1

    def to(self, device):
        t = lambda a: torch.from_numpy(a.copy()).to(device)
        return [self.k.to(device), self.v.to(device), t(self.table), t(self.lens), t(self.refs)]

    def same(self, got):
        """Whether the five device tensors hold this cache, bit for bit."""
        bits = lambda t: t.cpu().contiguous().view(torch.uint8)
        return [torch.equal(bits(got[0]), bits(self.k)), torch.equal(bits(got[1]), bits(self.v)),
                np.array_equal(got[2].cpu().numpy(), self.table), np.array_equal(got[3].cpu().numpy(), self.lens),
                np.array_equal(got[4].cpu().numpy(), self.refs)]

    def real(self, page):
        return 0 <= page < self.pages

    def used(self, n):
        return -(-n // self.ps)

    def fits(self, n):
        return 0 <= n <= self.max_pages * self.ps


def _grant(cache, needs):
    """Which requests get their pages (a list each, or None), lowest free page first, all or nothing, in order."""
    free = [p for p in range(cache.pages) if cache.refs[p] == 0]
    got, at, short = [], 0, False
    for n in needs:
        if n and at + n > len(free):
            short = True
        if n and short:
            got.append(None)
        else:
            got.append(free[at:at + n])
            at += n
    return got


def append(cache, k_new, v_new, rows, starts):
    """PagedAppend on `cache` in place; the status of each sequence."""
    ps, status, needs = cache.ps, [], []
    for s in range(len(cache.lens)):
        n, count = int(cache.lens[s]), starts[s + 1] - starts[s]
        st = DONE
        if count and not max(0, *starts[:s + 1]) <= starts[s] <= starts[s + 1] <= len(rows):
            st, count = INVALID, 0  # leaves the rows, ends before its start, or starts before an earlier range did or ended
        elif not cache.fits(n):
            st = INVALID
        elif not cache.fits(n + count):
            st = NO_ROOM
        elif count and n % ps:
            page = cache.table[s, n // ps]
            if not cache.real(page) or cache.refs[page] != 1:
                st = NOT_OWN
        status.append(st)
        needs.append(cache.used(n + count) - cache.used(n) if st == DONE else 0)
    for s, pages in enumerate(_grant(cache, needs)):
        if status[s] != DONE:
            continue
        if pages is None:
            status[s] = NO_ROOM
            continue
        n = int(cache.lens[s])
        for i, p in enumerate(pages):
            cache.table[s, cache.used(n) + i] = p
            cache.refs[p] = 1
        for i, r in enumerate(rows[starts[s]:starts[s + 1]]):
            page, at = cache.table[s, (n + i) // ps], (n + i) % ps
            inside = 0 <= r < k_new.shape[1]
            cache.k[:, page, :, at] = k_new[:, r] if inside else 0
            cache.v[:, page, :, at] = v_new[:, r] if inside else 0
        cache.lens[s] = n + starts[s + 1] - starts[s]
    return status


def fork(cache, forks, share):
    """PageFork on `cache` in place; the status of each pair."""
    ps, S, status, needs = cache.ps, len(cache.lens), [], []
    was = cache.copy()
    for i, (a, b) in enumerate(forks):
        ok = 0 <= a < S and 0 <= b < S and a != b and was.lens[b] == 0 and cache.fits(int(was.lens[a]))
        ok = ok and all(f[1] != b for f in forks[:i])
        status.append(DONE if ok else INVALID)
        n = int(was.lens[a]) if ok else 0
        if not ok:
            needs.append(0)
        elif share:
            needs.append(int(n % ps != 0 and cache.real(was.table[a, n // ps])))
        else:
            needs.append(sum(cache.real(p) for p in was.table[a, :cache.used(n)]))
    for i, ((a, b), pages) in enumerate(zip(forks, _grant(was, needs))):
        if status[i] != DONE:
            continue
        if pages is None:
            status[i] = NO_ROOM
            continue
        n, pages = int(was.lens[a]), list(pages)
        for e in range(cache.used(n)):
            p = was.table[a, e]
            if not cache.real(p):
                cache.table[b, e] = p
            elif share and (e + 1) * ps <= n:
                cache.table[b, e] = p
                cache.refs[p] += 1
            else:
                q, rows = pages.pop(0), min(ps, n - e * ps)
                cache.table[b, e], cache.refs[q] = q, 1
                cache.k[:, q, :, :rows] = was.k[:, p, :, :rows]
                cache.v[:, q, :, :rows] = was.v[:, p, :, :rows]
        cache.lens[b] = n
    return status


def compact(cache):
    """PageCompact on `cache` in place; how many pages moved."""
    used = int((cache.refs != 0).sum())
    src = [p for p in range(used, cache.pages) if cache.refs[p] != 0]
    dst = [p for p in range(used) if cache.refs[p] == 0]
    new = dict(zip(src, dst))
    for a, b in new.items():
        cache.k[:, b], cache.v[:, b] = cache.k[:, a].clone(), cache.v[:, a].clone()
        cache.refs[b], cache.refs[a] = cache.refs[a], 0
    for s in range(len(cache.lens)):
        if cache.fits(int(cache.lens[s])):
            for e in range(cache.used(int(cache.lens[s]))):
                cache.table[s, e] = new.get(int(cache.table[s, e]), cache.table[s, e])
    return len(src)


def free(cache, slots):
    """PageFree on `cache` in place; the status of each entry."""
    status = []
    for i, s in enumerate(slots):
        if not 0 <= s < len(cache.lens) or s in slots[:i] or not cache.fits(int(cache.lens[s])):
            status.append(INVALID)
            continue
        for e in range(cache.used(int(cache.lens[s]))):
            p = cache.table[s, e]
            if cache.real(p):
                cache.refs[p] = max(0, cache.refs[p] - 1)
            cache.table[s, e] = -1
        cache.lens[s] = 0
        status.append(DONE)
    return status


def attention(q, k_new, v_new, k_pages, v_pages, table, lens, starts, sees, scale, prior, max_nodes):
    """TreeAttention in 64 bits on CPU tensors, with the bound of its rounding: (out, tolerance), both float64.

    A score is a dot product of D terms in fp32, in any order: off by at most (D + 2) 2^-24 of the sum of the terms'
    sizes (times scale); its product with log2(e) and the subtraction of a maximum add 2^-22 of the largest score. A
    weight is off by that, the exponential's 2^-22, and its own rounding before the second product: 2^-16 for the two
    parts that it goes in as, or, where a KV head has more than 32 rows (max_nodes times the heads of its group), half
    a step of its type, as MHA rounds it; each shows in the sum of the weights too, hence twice. Sums of n terms in fp32 add n 2^-24. In fp16 a weight's
    lower part may lie under the normal range: n 2^-24 of the largest value. All of it is relative to sum(p |v|).
    The result is then rounded once: half a step of its type.
    """
    out, tol = prior.double().clone(), torch.zeros(prior.shape, dtype=torch.float64)
    D, ps = q.shape[-1], k_pages.shape[2]
    G, half = q.shape[1] // k_new.shape[1], torch.finfo(prior.dtype).eps / 2
    weight = half if max_nodes * G > 32 else 2.0 ** -16
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        pos = [t for t in range(n) if 0 <= table[s][t // ps] < k_pages.shape[0]]
        page, at = torch.tensor([int(table[s][t // ps]) for t in pos], dtype=torch.long), torch.tensor([t % ps for t in pos], dtype=torch.long)
        for i in range(a, b):
            mine = torch.tensor([j for j in range(b - a) if sees[i][j]], dtype=torch.long)
            for h in range(q.shape[1]):
                k = torch.cat([k_pages[page, h // G, at], k_new[a + mine, h // G]]).double()
                v = torch.cat([v_pages[page, h // G, at], v_new[a + mine, h // G]]).double()
                if not len(k):
                    out[i, h] = 0
                    continue
                x = q[i, h].double()
                w = k @ x * scale
                p = torch.softmax(w, 0)
                out[i, h] = p @ v
                size = float((k.abs() @ x.abs()).max()) * scale
                each = (D + 2) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + float(w.abs().max()) * 1.5)
                rel = 2 * (each + weight) + (len(k) + 8) * 2.0 ** -24
                tol[i, h] = half * out[i, h].abs() + rel * (p @ v.abs()) * (1 + half)
                if prior.dtype == torch.float16:
                    tol[i, h] += len(k) * 2.0 ** -24 * float(v.abs().max()) + 2.0 ** -25
    return out, tol
