"""Plain restatements of the paged 8-bit cache for the tests: bookkeeping on Python
lists, quantisation step by step in FP32 as engine_b200.h defines it, attention in
64 bits with a derived error bound."""
from __future__ import annotations

import numpy as np
import torch

U16, U32 = 2.0 ** -11, 2.0 ** -24
Q = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def codes_from(x: torch.Tensor, dtype) -> torch.Tensor:
    """Nearest code, ties to even, of FP32 x within the type's range."""
    if dtype == torch.int8:
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(dtype)


class Model:
    """A cache on the host, its operators written out."""

    def __init__(self, n_layers, n_pages, hk, page, d, n_slots, max_pages, dtype):
        self.dims = (n_layers, n_pages, hk, page, d)
        self.page, self.max_pages, self.dtype = page, max_pages, dtype
        self.code = torch.zeros(2, *self.dims, dtype=torch.float32)  # K, V: codes as numbers
        self.scale = torch.zeros(2, n_layers, n_pages, hk)
        self.rows = [[] for _ in range(n_slots)]
        self.length = [0] * n_slots
        self.ref = [0] * n_pages

    def _take(self):
        i = self.ref.index(0)
        self.ref[i] = 1
        return i

    def _pages(self, n):
        return -(-n // self.page)

    def extend(self, slots, n_new):
        n_slots = len(self.rows)
        if (any(not 0 <= s < n_slots for s in slots) or len(set(slots)) < len(slots)
                or any(n < 0 for n in n_new)
                or any(self.length[s] + n > self.max_pages * self.page for s, n in zip(slots, n_new))):
            return -1
        want = sum(self._pages(self.length[s] + n) - self._pages(self.length[s])
                   for s, n in zip(slots, n_new))
        missing = max(0, want - self.ref.count(0))
        if missing:
            return missing
        for s, n in zip(slots, n_new):
            for _ in range(self._pages(self.length[s] + n) - self._pages(self.length[s])):
                self.rows[s].append(self._take())
            self.length[s] += n
        return 0

    def fork(self, parents, children):
        n_slots = len(self.rows)
        if (any(not 0 <= s < n_slots for s in (*parents, *children))
                or len(set(children)) < len(children) or any(self.length[c] for c in children)
                or set(children) & set(parents)):
            return -1
        want = sum(self.length[p] % self.page != 0 for p in parents)
        missing = max(0, want - self.ref.count(0))
        if missing:
            return missing
        for p, c in zip(parents, children):
            full = self.length[p] // self.page
            self.rows[c] = self.rows[p][:full]
            if self.length[p] % self.page:
                i = self._take()
                self.code[:, :, i] = self.code[:, :, self.rows[p][full]]
                self.scale[:, :, i] = self.scale[:, :, self.rows[p][full]]
                self.rows[c].append(i)
            self.length[c] = self.length[p]
        for c in children:
            for i in self.rows[c][:self.length[c] // self.page]:
                self.ref[i] += 1
        return 0

    def free(self, slots):
        for s in slots:
            for i in self.rows[s]:
                self.ref[i] -= 1
            self.rows[s], self.length[s] = [], 0

    def compact(self):
        live = [i for i, r in enumerate(self.ref) if r]
        n = len(live)
        holes = [i for i in range(n) if not self.ref[i]]
        remap = [i if self.ref[i] and i < n else -1 for i in range(len(self.ref))]
        for src, dst in zip([i for i in live if i >= n], holes):
            remap[src] = dst
            self.code[:, :, dst], self.scale[:, :, dst] = self.code[:, :, src], self.scale[:, :, src]
            self.ref[dst], self.ref[src] = self.ref[src], 0
        self.rows = [[remap[i] for i in r] for r in self.rows]
        return remap

    def write(self, layer, k, v, slots, cu):
        """k, v [tokens, hk * d] FP16 on the host."""
        hk, page, d = self.dims[2:]
        inv_q = torch.tensor(1.0 / Q[self.dtype], dtype=torch.float32)
        for kv, x in enumerate((k, v)):
            x = x.float().view(-1, hk, d)
            for i, s in enumerate(slots):
                n = cu[i + 1] - cu[i]
                p = self.length[s] - n
                r = cu[i]
                while p < self.length[s]:
                    end = min(self.length[s], (p // page + 1) * page)
                    new = x[r:r + end - p].transpose(0, 1)  # [hk, rows, d]
                    w, off = self.rows[s][p // page], p % page
                    old = self.scale[kv, layer, w].clone() if off else torch.zeros(hk)
                    m = new.abs().amax((1, 2)) * inv_q
                    sc = torch.where(torch.isfinite(m) & ~old.isnan(), torch.maximum(old, m), float("nan"))
                    ratio = torch.where(sc > old, old / sc, 1.0)
                    if off:
                        c = self.code[kv, layer, w]
                        self.code[kv, layer, w] = torch.where((sc > old)[:, None, None],
                                                              codes_from(c * ratio[:, None, None], self.dtype).float(), c)
                    inv = torch.where(sc > 0, 1.0 / sc, 0.0)
                    y = torch.where(sc.isnan()[:, None, None], 0.0, new * inv[:, None, None])
                    self.code[kv, layer, w, :, off:off + end - p] = codes_from(y, self.dtype).float()
                    self.scale[kv, layer, w] = sc
                    r += end - p
                    p = end

    def load(self, kv):
        """Copies the model's state into a PagedKV on the device."""
        for t, i in ((kv.k, 0), (kv.v, 1)):
            t.copy_(self.code[i].to(self.dtype))
        kv.k_scale.copy_(self.scale[0])
        kv.v_scale.copy_(self.scale[1])
        kv.table.copy_(self.table())
        kv.length.copy_(torch.tensor(self.length, dtype=torch.int32))
        kv.ref.copy_(torch.tensor(self.ref, dtype=torch.int32))

    def table(self):
        t = torch.full((len(self.rows), self.max_pages), -1, dtype=torch.int32)
        for s, r in enumerate(self.rows):
            t[s, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return t

    def same_books(self, kv):
        assert kv.table.cpu().equal(self.table())
        assert kv.length.cpu().tolist() == self.length
        assert kv.ref.cpu().tolist() == self.ref

    def same_data(self, kv):
        """Codes and scales of every slot's positions, bit for bit."""
        got = [t.cpu().float() for t in (kv.k, kv.v)]
        sc = [t.cpu() for t in (kv.k_scale, kv.v_scale)]
        for s, r in enumerate(self.rows):
            for e, w in enumerate(r):
                n = min(self.page, self.length[s] - e * self.page)
                for i in range(2):
                    assert torch.equal(got[i][:, w, :, :n], self.code[i][:, w, :, :n]), (s, e, i)
                    assert torch.equal(sc[i][:, w].nan_to_num(-1), self.scale[i][:, w].nan_to_num(-1))


def attend64(kv, layer, q, slot, last, scale):
    """Rows q [m, H, d] of one sequence, row i over positions [0, last[i]]: output, lse
    and the output's error bound, in 64 bits on the host.

    The bound: x_j (the scaled score) is off by at most dx = 2 d u32 scale sum|q||k|
    (FP32 accumulation in an unspecified order, c = 2) plus 8 u32 |x| for its few FP32
    operations; 2^x by 2^-21.  A weight enters the product rounded to FP16 (u16 of
    itself, or half of FP16's smallest step where it is below 2^-14 of the largest);
    the sums over n keys add n u32 each.  With A = sum p |v|:
      |err| <= u16 |out| + (u16 + 2 (dx + 2^-21) + 2 n u32) (A + |out|) + n 2^-25 max|v|
    """
    cpu = {n: getattr(kv, n)[layer].cpu() for n in ("k", "v", "k_scale", "v_scale")}
    page, hk, d = kv.k.shape[3], kv.n_kv_heads, kv.head_dim
    n_keys = int(max(last)) + 1
    m, H, _ = q.shape
    out = np.zeros((m, H, d))
    lse = np.full((m, H), -np.inf)
    bound = np.zeros((m, H, d))
    if n_keys <= 0:
        return out, lse, bound
    ids = kv.table[slot].cpu()[: -(-n_keys // page)].long()
    k, v = ((cpu[n][ids].double() * cpu[n + "_scale"][ids].double()[..., None, None])
            .transpose(0, 1).reshape(hk, -1, d)[:, :n_keys].numpy() for n in ("k", "v"))
    q = q.double().cpu().numpy()
    G = H // hk
    for i in range(m):
        n = int(last[i]) + 1
        if n <= 0:
            continue
        for h in range(H):
            kk, vv = k[h // G, :n], v[h // G, :n]
            x = (kk @ q[i, h]) * scale
            dx = (2 * d * U32 * scale * (np.abs(kk) @ np.abs(q[i, h])) + 8 * U32 * np.abs(x)).max()
            e = np.exp(x - x.max())
            p = e / e.sum()
            out[i, h] = p @ vv
            lse[i, h] = x.max() + np.log(e.sum())
            a = p @ np.abs(vv)
            o = np.abs(out[i, h])
            bound[i, h] = (U16 * o + (U16 + 2 * (dx + 2.0 ** -21) + 2 * n * U32) * (a + o)
                           + n * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -25)
    return out, lse, bound


def check_attention(kv, layer, q, got, slots, cu, scale, causal=True, lse=None):
    """Every row against attend64; rows of sequence i are [cu[i], cu[i+1])."""
    lengths = kv.length.cpu().tolist()
    got = got.double().cpu().numpy()
    for i, s in enumerate(slots):
        rows = range(cu[i], cu[i + 1])
        if not len(rows):
            continue
        n = lengths[s]
        last = [n - len(rows) + j if causal else n - 1 for j in range(len(rows))]
        out, want_lse, bound = attend64(kv, layer, q[cu[i]:cu[i + 1]], s, last, scale)
        err = np.abs(got[cu[i]:cu[i + 1]] - out)
        assert (err <= bound).all(), (i, s, n, float(np.nanmax(err / np.maximum(bound, 1e-30))),
                                      int((~(err <= bound)).sum()))
        if lse is not None:
            g = lse[cu[i]:cu[i + 1]].double().cpu().numpy()
            assert np.array_equal(np.isneginf(g), np.isneginf(want_lse))
            ok = np.isfinite(want_lse)
            # the sums' relative error, as above, and the logarithm's own roundings
            tol = 2.0 ** -19 + 4 * n * U32 + 2.0 ** -19 * np.abs(want_lse[ok])
            assert (np.abs(g[ok] - want_lse[ok]) <= tol).all(), np.abs(g[ok] - want_lse[ok]).max()
