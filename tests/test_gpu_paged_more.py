"""GPU: calls of more sequences than one launch takes, many query heads to a KV head, and what the
8 bits of the paged cache cost against the FP16 keys and values that were written."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

I8, E4M3 = torch.int8, torch.float8_e4m3fn


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def filled(pkg, dev, lens, *, hk, d, page, max_pages, dtype, spare=0):
    """A cache whose slots have the given lengths, its codes and scales drawn."""
    n_pages = sum(-(-n // page) for n in lens) + 1
    kv = pkg.ops.PagedKV.empty(1, n_pages, hk, page, d, len(lens) + spare, max_pages, dtype, dev)
    g = torch.Generator().manual_seed(len(lens))
    for t, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        x = torch.randn(t.shape, generator=g) * (30 if dtype == I8 else 60)
        t.copy_(ref.codes_from(x, dtype))
        s.copy_(0.01 + 0.02 * torch.rand(s.shape, generator=g))
    assert int(pkg.ops.kv_pages_extend(kv, i32(range(len(lens)), dev), i32(lens, dev))) == 0
    return kv


@pytest.mark.parametrize("wide", [False, True])  # a CTA to an item; items cut and joined
def test_more_sequences_than_a_launch_takes(pkg, dev, wide):
    """1040 sequences: the last 16 are a launch of their own.  Decode, a few rows each and many rows
    each, with the slots in order and permuted."""
    n, page, d, heads = 1040, 16, 64, 2
    lens = [1 + (i * 37) % 60 for i in range(1024)] + [500 + 60 * i if wide else 100 + 50 * i for i in range(16)]
    kv = filled(pkg, dev, lens, hk=1, d=d, page=page, max_pages=100 if wide else 64, dtype=I8)
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(3)).tolist()
    perm = [s for s in perm if s < 1024] + [s for s in perm if s >= 1024]  # the long ones stay last
    for slots in (None, perm):
        order = list(range(n)) if slots is None else slots
        on = None if slots is None else i32(slots, dev)
        look = list(range(0, 1024, 73)) + list(range(1022, n))
        q = torch.randn(n, heads, d, generator=torch.Generator().manual_seed(1)).half().to(dev)
        out, lse = pkg.ops.attention_paged_decode(kv, 0, q, on, want_lse=True)
        at = [order[i] for i in look]
        ref.check_attention(kv, 0, q[look], out[look], at, list(range(len(at) + 1)), d ** -0.5, lse=lse[look])
        for rows in ([1 + i % 4 for i in range(n)], [18 + i % 7 for i in range(n)]):
            cu = [0]
            for r in rows:
                cu.append(cu[-1] + r)
            q = torch.randn(cu[-1], heads, d, generator=torch.Generator().manual_seed(2)).half().to(dev)
            out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, on, i32(cu, dev), want_lse=True)
            for i in look:  # the last rows of some
                last = min(rows[i], 3)
                a = slice(cu[i + 1] - last, cu[i + 1])
                ref.check_attention(kv, 0, q[a], out[a], [order[i]], [0, last], d ** -0.5, lse=lse[a])
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("group", [129, 160])
def test_more_query_heads_to_a_kv_head_than_a_tile_has_rows(pkg, dev, dtype, group):
    """Prefill of many rows with more than 128 query heads to a KV head, which the kernel for few
    rows takes, and decode."""
    hk, d, page = 2, 64, 32
    lens, rows = [300, 1, 45, 1200], [40, 1, 45, 9]
    kv = filled(pkg, dev, lens, hk=hk, d=d, page=page, max_pages=40, dtype=dtype)
    cu = [0, 40, 41, 86, 95]
    q = torch.randn(95, hk * group, d, generator=torch.Generator().manual_seed(2)).half().to(dev)
    out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, None, i32(cu, dev), want_lse=True)
    for i in range(4):
        last = min(rows[i], 2)
        a = slice(cu[i + 1] - last, cu[i + 1])
        ref.check_attention(kv, 0, q[a], out[a], [i], [0, last], d ** -0.5, lse=lse[a])
    one, lse = pkg.ops.attention_paged_decode(kv, 0, q[:4], want_lse=True)
    ref.check_attention(kv, 0, q[:4], one, [0, 1, 2, 3], [0, 1, 2, 3, 4], d ** -0.5, lse=lse)
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("one_by_one", [False, True])
def test_the_cache_against_the_rows_that_were_written(pkg, dev, dtype, one_by_one):
    """Stored values and attention against the FP16 keys and values, in 64 bits; rows that come at
    once, and one at a time with magnitudes that grow, so that pages are rounded again and again.

    A rounding to a code of scale s is off by at most s / 2 (int8), or 2^-4 of the value or
    s 2^-10 where that is more (e4m3: half a step, half of the smallest one); a page that grows is
    rounded once more at its new scale, on top of what it was off by.  (x / s itself has three FP32
    roundings.)  With |dk_j|, |dv_j| so bounded, a score is off by at most
    e = max_j scale sum |q||dk_j|, a softmax weight by a factor within exp(+-2 e), so that
      |err| <= (exp(2 e) - 1) sum p |v| + exp(2 e) sum p |dv|
    beside the kernel's own error on the stored codes (attend64's bound)."""
    page, d, hk, heads, n = 32, 128, 2, 8, 75
    kv = pkg.ops.PagedKV.empty(1, 8, hk, page, d, 2, 4, dtype, dev)
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(2, n, hk, d, generator=g) * (1 + torch.arange(n)[:, None, None] / 25)
    rows = rows.half()
    on = rows.to(dev).flatten(2)
    slot = i32([1], dev)
    off = torch.zeros(2, n, hk, d, dtype=torch.float64)  # what each stored value may be off by
    x = rows.double()
    scale = np.zeros((2, 4, hk))
    grown = 0
    steps = [(i, i + 1) for i in range(n)] if one_by_one else [(0, n)]
    for a, b in steps:
        assert int(pkg.ops.kv_pages_extend(kv, slot, i32([b - a], dev))) == 0
        pkg.ops.kv_pages_write(kv, 0, on[0, a:b], on[1, a:b], slot, None if one_by_one else i32([0, n], dev))
        table = kv.table[1].tolist()
        for e in range(a // page, (b - 1) // page + 1):
            lo, hi = max(a, e * page), min(b, (e + 1) * page)
            for i, t in enumerate((kv.k_scale, kv.v_scale)):
                s = t[0, table[e]].double().cpu()[:, None]
                again = torch.from_numpy(scale[i, e])[:, None] < s

                def rounded(y, o, s=s):
                    return o + (s / 2 if dtype == I8 else torch.maximum(2.0 ** -4 * (y.abs() + o), s * 2.0 ** -10))

                if lo > e * page and again.any():
                    grown += 1
                    old = slice(e * page, lo)
                    off[i, old] = torch.where(again, rounded(x[i, old], off[i, old]), off[i, old])
                off[i, lo:hi] = rounded(x[i, lo:hi], off[i, lo:hi])
                scale[i, e] = s[:, 0].numpy()
    assert (grown > 10) == one_by_one
    off += 2.0 ** -20 * x.abs()
    ids = kv.table[1, :3].long()
    stored = torch.stack([(c[0][ids].double() * sc[0][ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:n]
                          for c, sc in ((kv.k, kv.k_scale), (kv.v, kv.v_scale))]).cpu()
    assert ((stored - x).abs() <= off).all(), ((stored - x).abs() / off).max()
    q = torch.randn(1, heads, d, generator=g).half()
    out = pkg.ops.attention_paged_decode(kv, 0, q.to(dev), slot).double().cpu().numpy()[0]
    _, _, own = ref.attend64(kv, 0, q, 1, [n - 1], d ** -0.5)
    for h in range(heads):
        k, v = x[0, :, h // 4].numpy(), x[1, :, h // 4].numpy()
        qh = q[0, h].double().numpy()
        w = k @ qh * d ** -0.5
        p = np.exp(w - w.max())
        p /= p.sum()
        e = (off[0, :, h // 4].numpy() @ np.abs(qh)).max() * d ** -0.5
        bound = np.expm1(2 * e) * (p @ np.abs(v)) + np.exp(2 * e) * (p @ off[1, :, h // 4].numpy()) + own[0, h]
        assert (np.abs(out[h] - p @ v) <= bound).all(), (h, (np.abs(out[h] - p @ v) / bound).max())
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (64, 128)])
def test_the_smallest_pool(pkg, dev, dtype, d, page):
    """One page, one KV head, one slot: both attention kernels, with fewer rows in the pool than a
    tile has, and a fork and an extend that it cannot meet."""
    kv = filled(pkg, dev, [page - 3], hk=1, d=d, page=page, max_pages=1, dtype=dtype, spare=1)
    kv.ref[1:] = 1  # (`filled` leaves a page free)
    for rows in (1, 3, 40):
        q = torch.randn(rows, 2, d, generator=torch.Generator().manual_seed(rows)).half().to(dev)
        out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, i32([0], dev), i32([0, rows], dev), want_lse=True)
        ref.check_attention(kv, 0, q, out, [0], [0, rows], d ** -0.5, lse=lse)
    assert int(pkg.ops.kv_pages_fork(kv, i32([0], dev), i32([1], dev))) == 1
    assert int(pkg.ops.kv_pages_extend(kv, i32([0, 1], dev), i32([3, 1], dev))) == 1
    assert int(pkg.ops.kv_pages_extend(kv, i32([0], dev), i32([3], dev))) == 0
    assert kv.length.tolist() == [page, 0] and kv.table.tolist() == [[0], [-1]]
    assert pkg.device_status() == 0


def test_host_threads_at_once(pkg, dev):
    """Eight host threads, each with a stream and a cache of its own, step at once."""
    import threading

    wrong = []

    def work(i):
        try:
            torch.cuda.set_device(dev)
            with torch.cuda.stream(torch.cuda.Stream()):
                lens = [40 + 300 * i, 1 + i]
                kv = filled(pkg, dev, lens, hk=2, d=64 if i % 2 else 128, page=32, max_pages=80, dtype=I8 if i % 3 else E4M3)
                d = kv.head_dim
                q = torch.randn(30, 8, d, generator=torch.Generator().manual_seed(i)).half().to(dev)
                for _ in range(5):
                    one = pkg.ops.attention_paged_decode(kv, 0, q[:2])
                    many = pkg.ops.attention_paged_prefill(kv, 0, q, None, i32([0, 29, 30], dev))
                torch.cuda.current_stream().synchronize()
                ref.check_attention(kv, 0, q[:2], one, [0, 1], [0, 1, 2], d ** -0.5)
                ref.check_attention(kv, 0, q, many, [0, 1], [0, 29, 30], d ** -0.5)
        except BaseException as e:  # noqa: BLE001 (told to the main thread)
            wrong.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    assert pkg.device_status() == 0
