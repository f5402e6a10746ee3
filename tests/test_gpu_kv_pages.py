"""GPU: the paged 8-bit KV cache and its attention through the public calls.

The bookkeeping and the codes are compared bit for bit with tests/paged_ref.py's
restatement, attention with 64-bit arithmetic under its derived bound."""
from __future__ import annotations

import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

I8, E4M3 = torch.int8, torch.float8_e4m3fn


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def make(pkg, dev, *, layers=1, n_pages=24, hk=2, page=16, d=64, slots=6, max_pages=12, dtype=I8):
    m = ref.Model(layers, n_pages, hk, page, d, slots, max_pages, dtype)
    kv = pkg.ops.PagedKV.empty(layers, n_pages, hk, page, d, slots, max_pages, dtype, dev)
    for t in (kv.k, kv.v):  # what a page held before is of no account
        t.view(torch.uint8).random_(0, 256)
    return m, kv


def grow(pkg, m, kv, slots, n_new, dev, seed=0, amp=1.0, layers=None):
    """extend, then new rows written to every layer, on both sides."""
    g = torch.Generator().manual_seed(seed)
    st = pkg.ops.kv_pages_extend(kv, i32(slots, dev), i32(n_new, dev))
    want = m.extend(slots, n_new)
    assert int(st) == want
    if want:
        return want
    cu = [0]
    for n in n_new:
        cu.append(cu[-1] + n)
    width = kv.n_kv_heads * kv.head_dim
    for layer in range(kv.k.shape[0]) if layers is None else layers:
        rows = (torch.randn(cu[-1], 2 * width + 8, generator=g) * amp).half()
        on = rows.to(dev)
        pkg.ops.kv_pages_write(kv, layer, on[:, :width], on[:, width:2 * width], i32(slots, dev), i32(cu, dev))
        m.write(layer, rows[:, :width], rows[:, width:2 * width], slots, cu)
    return 0


# ------------------------------------------------------------------ write


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("page,d,hk", [(16, 64, 2), (32, 128, 1), (64, 64, 3), (128, 128, 2), (64, 128, 8)])
def test_write_codes_and_scales(pkg, dev, dtype, page, d, hk):
    """Prompts of odd lengths, then appends of one and several rows, into scattered
    pages: codes and scales bit for bit."""
    m, kv = make(pkg, dev, page=page, d=d, hk=hk, dtype=dtype, n_pages=26, layers=2)
    slots = [4, 0, 2, 5]
    grow(pkg, m, kv, slots, [1, page, 3 * page - 1, page + 5], dev, 1)
    m.same_books(kv)
    m.same_data(kv)
    grow(pkg, m, kv, [2, 4], [1, 1], dev, 2, amp=3.0)      # larger rows: the pages are rounded again
    grow(pkg, m, kv, [5, 0, 4], [page - 4, 0, 2], dev, 3)  # across a page's end; no rows; two
    grow(pkg, m, kv, [4, 5], [1, 2 * page], dev, 4, amp=0.01)  # smaller: the scales stay
    m.same_books(kv)
    m.same_data(kv)


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_write_one_row_each(pkg, dev, dtype):
    """cu_new None: a generated token per sequence; every row within half a step."""
    m, kv = make(pkg, dev, page=16, d=128, hk=3, dtype=dtype, slots=40, n_pages=90)
    grow(pkg, m, kv, list(range(40)), [1 + (i * 7) % 20 for i in range(40)], dev, 5)
    slots = list(range(39, -1, -2))
    rows = torch.randn(len(slots), 2, 3 * 128, generator=torch.Generator().manual_seed(6)).half()
    pkg.ops.kv_pages_extend(kv, i32(slots, dev), i32([1] * len(slots), dev))
    m.extend(slots, [1] * len(slots))
    on = rows.to(dev)
    pkg.ops.kv_pages_write(kv, 0, on[:, 0], on[:, 1], i32(slots, dev))
    m.write(0, rows[:, 0], rows[:, 1], slots, list(range(len(slots) + 1)))
    m.same_books(kv)
    m.same_data(kv)
    for i, s in enumerate(slots):  # in 64 bits: the stored value is the nearest code
        e, r = divmod(m.length[s] - 1, 16)
        w = m.rows[s][e]
        for t, sc, x in ((kv.k, kv.k_scale, rows[i, 0]), (kv.v, kv.v_scale, rows[i, 1])):
            a = sc[0, w].double().cpu()[:, None]
            got = t[0, w, :, r].cpu().float().double() * a
            x = x.double().view(3, 128)
            # half a step of the type, and the FP32 roundings of x / scale (3 of 2^-24)
            step = a * 0.5 if dtype == I8 else torch.maximum(2.0 ** -4 * x.abs(), a * 2.0 ** -10)
            assert ((got - x).abs() <= step * (1 + 2.0 ** -20) + x.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_write_zeros_extremes_and_non_finite(pkg, dev, dtype):
    m, kv = make(pkg, dev, page=16, d=64, hk=2, dtype=dtype, slots=5)
    slots, n = [0, 1, 2, 3, 4], [5] * 5
    pkg.ops.kv_pages_extend(kv, i32(slots, dev), i32(n, dev))
    m.extend(slots, n)
    rows = torch.randn(25, 128, generator=torch.Generator().manual_seed(1)).half()
    rows[0:5] = 0                      # an all-zero page: scale 0
    rows[5:10] = 6e-8                  # FP16's smallest number
    rows[10, 3] = 65504
    rows[16, 7] = float("inf")         # one head only
    rows[21, 70] = float("nan")
    cu = [0, 5, 10, 15, 20, 25]
    on = rows.to(dev)
    pkg.ops.kv_pages_write(kv, 0, on, on, i32(slots, dev), i32(cu, dev))
    m.write(0, rows, rows, slots, cu)
    m.same_data(kv)
    assert kv.k_scale[0, m.rows[0][0]].eq(0).all()
    assert kv.k_scale[0, m.rows[3][0]].isnan().tolist() == [True, False]
    assert kv.k_scale[0, m.rows[4][0]].isnan().tolist() == [False, True]
    grow(pkg, m, kv, slots, [1] * 5, dev, 9)  # a zero page takes real rows; a NaN scale stays
    m.same_data(kv)


def test_write_leaves_the_rest_alone(pkg, dev):
    """Rows past cu_new[-1], other pages, other layers and rows past the length stay."""
    m, kv = make(pkg, dev, layers=3, page=32, d=64, hk=2)
    grow(pkg, m, kv, [1, 3], [40, 10], dev, 1, layers=[])
    before = [t.clone() for t in (kv.k, kv.v)]
    sc = [t.clone() for t in (kv.k_scale, kv.v_scale)]
    rows = torch.randn(60, 128).half()
    on = rows.to(dev)
    pkg.ops.kv_pages_write(kv, 1, on, on, i32([1, 3], dev), i32([0, 40, 50], dev))  # ten rows of padding
    m.write(1, rows, rows, [1, 3], [0, 40, 50])
    for t, b in zip((kv.k, kv.v), before):
        assert torch.equal(t[0].view(torch.uint8), b[0].view(torch.uint8))
        assert torch.equal(t[2].view(torch.uint8), b[2].view(torch.uint8))
        used = [m.rows[1][0], m.rows[1][1], m.rows[3][0]]
        rest = [i for i in range(kv.n_pages) if i not in used]
        assert torch.equal(t[1, rest].view(torch.uint8), b[1, rest].view(torch.uint8))
        assert torch.equal(t[1, used[1], :, 8:].view(torch.uint8), b[1, used[1], :, 8:].view(torch.uint8))
        assert torch.equal(t[1, used[2], :, 10:].view(torch.uint8), b[1, used[2], :, 10:].view(torch.uint8))
    for t, b in zip((kv.k_scale, kv.v_scale), sc):
        assert torch.equal(t[0], b[0]) and torch.equal(t[2], b[2])


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_write_leaves_shared_pages_alone(pkg, dev, dtype):
    """Rows of a slot that was forked at a page's end and not extended: the page has two users and
    stays; the batch's other rows, and the slot's rows in pages of its own, are written."""
    page, d, hk = 16, 64, 2
    m, kv = make(pkg, dev, page=page, d=d, hk=hk, dtype=dtype)
    grow(pkg, m, kv, [0, 1], [2 * page, 7], dev, 1)
    assert int(pkg.ops.kv_pages_fork(kv, i32([0, 0], dev), i32([3, 4], dev))) == m.fork([0, 0], [3, 4]) == 0
    pkg.ops.kv_pages_extend(kv, i32([1], dev), i32([1], dev))
    m.extend([1], [1])
    rows = 5 * torch.randn(4, hk * d, generator=torch.Generator().manual_seed(2)).half()
    on = rows.to(dev)
    for slots in ([3, 1], [4, 1], [0, 1]):  # one row each; slot 1's row is rewritten
        pkg.ops.kv_pages_write(kv, 0, on[:2], on[2:], i32(slots, dev))
        assert pkg.device_status() == 2
    m.write(0, rows[1:2], rows[3:4], [1], [0, 1])
    m.write(0, rows[1:2], rows[3:4], [1], [0, 1])
    m.write(0, rows[1:2], rows[3:4], [1], [0, 1])
    m.same_books(kv)
    m.same_data(kv)
    # ragged: five rows of slot 3, of which three fall into the shared page; slot 1 as it is
    assert int(pkg.ops.kv_pages_extend(kv, i32([3], dev), i32([2], dev))) == m.extend([3], [2]) == 0
    rows = 5 * torch.randn(6, hk * d, generator=torch.Generator().manual_seed(3)).half()
    on = rows.to(dev)
    pkg.ops.kv_pages_write(kv, 0, on, on, i32([3, 1], dev), i32([0, 5, 6], dev))
    assert pkg.device_status() == 2
    m.write(0, rows[3:], rows[3:], [3, 1], [0, 2, 3])
    m.same_books(kv)
    m.same_data(kv)
    # with its own pages alone, nothing is left out
    pkg.ops.kv_pages_free(kv, i32([0, 4], dev))
    m.free([0, 4])
    pkg.ops.kv_pages_write(kv, 0, on, on, i32([3, 1], dev), i32([0, 5, 6], dev))
    m.write(0, rows, rows, [3, 1], [0, 5, 6])
    assert pkg.device_status() == 0
    m.same_data(kv)


def test_one_row_has_any_pitch(pkg, dev):
    """A single row's pitch is no part of it: views whose rows are 8 n + 3 elements apart, of K and
    V in tensors of different widths."""
    d, hk, heads = 64, 2, 8
    m, kv = make(pkg, dev, d=d, hk=hk)
    grow(pkg, m, kv, [2], [20], dev, 1)
    assert int(pkg.ops.kv_pages_extend(kv, i32([2], dev), i32([1], dev))) == m.extend([2], [1]) == 0
    k, v, q = (torch.randn(1, n, generator=torch.Generator().manual_seed(n)).half() for n in (395, 261, 1027))
    on = [t.to(dev) for t in (k, v, q)]
    pkg.ops.kv_pages_write(kv, 0, on[0][:, 128:256], on[1][:, :128], i32([2], dev))
    m.write(0, k[:, 128:256], v[:, :128], [2], [0, 1])
    m.same_data(kv)
    one = on[2][:, 8:8 + heads * d].view(1, heads, d)
    got = pkg.ops.attention_paged_decode(kv, 0, one, i32([2], dev))
    ref.check_attention(kv, 0, one, got, [2], [0, 1], d ** -0.5)
    assert torch.equal(got, pkg.ops.attention_paged_prefill(kv, 0, one, i32([2], dev), i32([0, 1], dev)))


# ------------------------------------------------------------ bookkeeping


@pytest.mark.parametrize("page,seed", [(16, 0), (32, 1), (128, 2)])
def test_random_operations(pkg, dev, page, seed):
    """A few hundred random extends (with writes), forks, frees and compactions, some of
    them impossible: books and data as the restatement's after each."""
    rng = random.Random(seed)
    m, kv = make(pkg, dev, layers=2, n_pages=24, hk=1, page=page, d=64, slots=12, max_pages=9)
    seen = set()
    for step in range(200):
        what = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        if what == "extend":
            slots = rng.sample(range(12), rng.randint(1, 5))
            st = grow(pkg, m, kv, slots, [rng.choice([0, 1, 1, page, rng.randint(1, 3 * page)]) for _ in slots], dev, step)
            seen.add(("extend", min(st, 1)))
        elif what == "fork":
            n = rng.randint(1, 4)
            parents = [rng.randrange(12) for _ in range(n)]
            children = [rng.randrange(12) for _ in range(n)]
            st = pkg.ops.kv_pages_fork(kv, i32(parents, dev), i32(children, dev))
            want = m.fork(parents, children)
            assert int(st) == want
            seen.add(("fork", min(want, 1)))
        elif what == "free":
            slots = [rng.randrange(12) for _ in range(rng.randint(1, 4))]  # the same slot twice, at times
            pkg.ops.kv_pages_free(kv, i32(slots, dev))
            m.free(slots)
        else:
            remap = pkg.ops.kv_pages_compact(kv)
            assert remap.tolist() == m.compact()
        m.same_books(kv)
        if step % 10 == 9:
            m.same_data(kv)
    m.same_data(kv)
    pkg.device_status()  # refused calls set bit 2
    assert {("extend", 0), ("extend", 1), ("fork", 0), ("fork", -1)} <= seen


def test_refused_calls_change_nothing(pkg, dev):
    m, kv = make(pkg, dev, n_pages=10, page=16, slots=6, max_pages=4)
    grow(pkg, m, kv, [0, 1], [20, 33], dev)
    ops = pkg.ops
    for slots, n in (([0, 0], [1, 1]), ([0, 6], [1, 1]), ([-1], [1]), ([0], [-1]), ([0], [45]),
                     ([2, 3, 4], [64, 64, 64])):
        st = ops.kv_pages_extend(kv, i32(slots, dev), i32(n, dev))
        assert int(st) == m.extend(slots, n) != 0
        m.same_books(kv)
    for par, chi in (([0], [1]), ([0, 0], [2, 2]), ([0, 2], [2, 3]), ([0], [6]), ([7], [2]),
                     ([0, 1, 0, 1, 0, 1], [2, 3, 4, 5, 2, 3])):
        st = ops.kv_pages_fork(kv, i32(par, dev), i32(chi, dev))
        assert int(st) == m.fork(par, chi) != 0
        m.same_books(kv)
    assert pkg.device_status() & 2
    assert int(ops.kv_pages_extend(kv, None, i32([1, 2, 3], dev))) == m.extend([0, 1, 2], [1, 2, 3]) == 0
    m.same_books(kv)
    assert int(ops.kv_pages_extend(kv, i32([], dev), i32([], dev))) == 0
    assert int(ops.kv_pages_fork(kv, i32([], dev), i32([], dev))) == 0
    ops.kv_pages_free(kv, i32([], dev))
    m.same_books(kv)
    assert pkg.device_status() == 0


def test_extend_by_more_pages_than_32_bits_count(pkg, dev):
    """2048 slots that want 2^20 pages each: refused, with the number that is missing."""
    n, per = 2048, 2 ** 20
    kv = pkg.ops.PagedKV.empty(1, 40, 1, 16, 64, n, per, I8, dev)  # 8.6 GB of table
    st = pkg.ops.kv_pages_extend(kv, None, i32([per * 16] * n, dev))
    assert int(st) == 2 ** 31 - 40 and kv.length.eq(0).all() and kv.ref.eq(0).all()
    st = pkg.ops.kv_pages_extend(kv, i32([3, 9], dev), i32([17, 600], dev))
    assert int(st) == 0 and kv.ref.sum() == 40
    st = pkg.ops.kv_pages_extend(kv, None, i32([16] * n, dev))
    assert int(st) == n
    assert kv.table[9, :38].tolist() == list(range(2, 40)) and kv.length.sum() == 617
    assert pkg.device_status() == 0


def test_many_slots_and_pages(pkg, dev):
    """The most slots of a call, and pools of several thousand pages."""
    n = 2048
    m, kv = make(pkg, dev, n_pages=9000, hk=1, page=16, d=64, slots=2 * n, max_pages=6)
    a, b = list(range(0, 2 * n, 2)), list(range(1, 2 * n, 2))
    lens = [1 + (i * 37) % 50 for i in range(n)]
    assert int(pkg.ops.kv_pages_extend(kv, i32(a, dev), i32(lens, dev))) == m.extend(a, lens) == 0
    m.same_books(kv)
    assert int(pkg.ops.kv_pages_fork(kv, i32(a, dev), i32(b, dev))) == m.fork(a, b) == 0
    m.same_books(kv)
    pkg.ops.kv_pages_free(kv, i32(a[::3], dev))
    m.free(a[::3])
    m.same_books(kv)
    assert pkg.ops.kv_pages_compact(kv).tolist() == m.compact()
    m.same_books(kv)


# -------------------------------------------------------------- attention


HEADS = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (32, 1, 64), (40, 2, 128), (6, 2, 64), (20, 4, 128)]


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("heads,hk,d", HEADS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_decode(pkg, dev, dtype, heads, hk, d, page):
    lens = [1, 0, page, page + 1, 3 * page - 7, 300]
    m, kv = make(pkg, dev, layers=2, hk=hk, d=d, page=page, dtype=dtype, slots=8, n_pages=60, max_pages=24)
    slots = [5, 0, 3, 7, 1, 2]
    grow(pkg, m, kv, slots, lens, dev, 3)
    q = torch.randn(6, heads + 1, d, generator=torch.Generator().manual_seed(2)).half().to(dev)[:, :heads]  # strided rows
    out, lse = pkg.ops.attention_paged_decode(kv, 1, q, i32(slots, dev), want_lse=True)
    ref.check_attention(kv, 1, q, out, slots, list(range(7)), d ** -0.5, lse=lse)
    assert out[1].eq(0).all() and lse[1].isneginf().all()
    assert torch.equal(out, pkg.ops.attention_paged_decode(kv, 1, q, i32(slots, dev)))  # deterministic
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("n", [2049, 5000])
def test_decode_long(pkg, dev, dtype, n):
    """Split over many CTAs; scales that differ by orders of magnitude from page to page."""
    m, kv = make(pkg, dev, hk=2, d=128, page=64, dtype=dtype, slots=3, n_pages=170, max_pages=100)
    grow(pkg, m, kv, [0, 2], [n, 77], dev, 3)
    kv.v_scale.mul_(10 ** torch.linspace(-4, 3, 170, device=dev)[torch.randperm(170)][:, None])
    q = (2 * torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(2))).half().to(dev)
    out, lse = pkg.ops.attention_paged_decode(kv, 0, q, i32([0, 2], dev), want_lse=True)
    ref.check_attention(kv, 0, q, out, [0, 2], [0, 1, 2], 128 ** -0.5, lse=lse)


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("heads,hk,d", HEADS)
@pytest.mark.parametrize("page,causal", [(16, True), (32, False), (128, True)])
def test_prefill(pkg, dev, dtype, heads, hk, d, page, causal):
    """Whole prompts, chunks on a cached part, single rows, no rows and empty sequences in
    one ragged batch; the rows behind the last sequence stay."""
    lens = [150, 37, 0, 290, 1, 64, 131]
    new = [150, 5, 0, 140, 1, 0, 3]
    m, kv = make(pkg, dev, hk=hk, d=d, page=page, dtype=dtype, slots=8, n_pages=64, max_pages=20)
    slots = [6, 0, 3, 7, 1, 2, 5]
    grow(pkg, m, kv, slots, lens, dev, 4)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    q = torch.randn(cu[-1] + 9, heads + 2, d, generator=torch.Generator().manual_seed(3)).half().to(dev)[:, :heads]
    out = torch.full(q.shape, 7.0, device=dev, dtype=torch.float16)
    got, lse = pkg.ops.attention_paged_prefill(kv, 0, q, i32(slots, dev), i32(cu, dev), out=out,
                                               is_causal=causal, want_lse=True)
    assert got is out
    ref.check_attention(kv, 0, q, out, slots, cu, d ** -0.5, causal, lse)
    assert out[cu[-1]:].eq(7).all()
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_pages_of_zeros_beside_small_values(pkg, dev, dtype, new):
    """A key in a page whose V is all zeros takes most of the weight, beside values of about
    1e-3: the others' weights keep their precision."""
    hk, d, page = 2, 64, 16
    m, kv = make(pkg, dev, hk=hk, d=d, page=page, dtype=dtype)
    n = 5 * page
    assert int(pkg.ops.kv_pages_extend(kv, i32([0], dev), i32([n], dev))) == m.extend([0], [n]) == 0
    g = torch.Generator().manual_seed(8)
    q = (1 + 0.1 * torch.randn(new, 4, d, generator=g)).half().to(dev)
    k = 0.05 * torch.randn(n, hk * d, generator=g)
    k[0] = 0.52  # a score 4.2 above the others'
    v = 1e-3 * torch.randn(n, hk * d, generator=g)
    v[:page] = 0
    v[2 * page:3 * page] = 0
    pkg.ops.kv_pages_write(kv, 0, k.half().to(dev), v.half().to(dev), i32([0], dev), i32([0, n], dev))
    if new == 1:
        out, lse = pkg.ops.attention_paged_decode(kv, 0, q, i32([0], dev), want_lse=True)
    else:
        out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, i32([0], dev), i32([0, new], dev), want_lse=True)
    ref.check_attention(kv, 0, q, out, [0], [0, new], d ** -0.5, True, lse)


@pytest.mark.parametrize("rows", [[1], [4, 0, 2], [7, 9, 1, 1, 3], [33], [70, 40, 0, 150], [9] * 12])
def test_prefill_cut_items(pkg, dev, rows):
    """Rows over a few thousand keys: items cut into many parts, few items or many, both kernels."""
    n = len(rows)
    lens = [1400 + 331 * i for i in range(n)]
    lens[-1] = 40
    m, kv = make(pkg, dev, hk=2, d=64, page=64, slots=n, n_pages=700, max_pages=100)
    grow(pkg, m, kv, list(range(n)), lens, dev, 3)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], 8, 64, generator=torch.Generator().manual_seed(2)).half().to(dev)
    out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, None, i32(cu, dev), want_lse=True)
    ref.check_attention(kv, 0, q, out, list(range(n)), cu, 0.125, True, lse)
    assert torch.equal(out, pkg.ops.attention_paged_prefill(kv, 0, q, None, i32(cu, dev)))
    assert pkg.device_status() == 0


@pytest.mark.parametrize("heads,hk,d", [(192, 3, 64), (32, 2, 64), (32, 8, 128)])
def test_prefill_items_without_a_second_side(pkg, dev, heads, hk, d):
    """Short sequences with odd tails, so that items of one tile with and without rows in the
    second half follow each other: every call answers the same, no wait runs out."""
    rnd = random.Random(4)
    n = 17
    lens = [rnd.choice([0, 1, 3, rnd.randint(1, 200), 128, 130]) for _ in range(n)]
    rows = [rnd.choice([1, 33, 65, rnd.randint(30, 300), 128]) for _ in range(n)]
    m, kv = make(pkg, dev, hk=hk, d=d, page=32, slots=n, n_pages=120, max_pages=9, dtype=E4M3)
    grow(pkg, m, kv, list(range(n)), lens, dev, 3)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], heads, d, generator=torch.Generator().manual_seed(2)).half().to(dev)
    first = None
    for _ in range(25):
        out = torch.full_like(q, 7)
        pkg.ops.attention_paged_prefill(kv, 0, q, None, i32(cu, dev), out=out)
        first = out if first is None else first
        assert torch.equal(out, first)
    assert pkg.device_status() == 0
    for b in (2, 7, 11, 16):  # the last rows of some
        at = slice(cu[b + 1] - min(rows[b], 3), cu[b + 1])
        ref.check_attention(kv, 0, q[at], first[at], [b], [0, min(rows[b], 3)], d ** -0.5)


def test_prefill_rows_that_see_nothing(pkg, dev):
    """More query rows than positions: the first rows see no key."""
    m, kv = make(pkg, dev, hk=2, d=128, page=16)
    grow(pkg, m, kv, [0, 1], [5, 40], dev, 4)
    q = torch.randn(70, 8, 128).half().to(dev)
    out, lse = pkg.ops.attention_paged_prefill(kv, 0, q, i32([0, 1], dev), i32([0, 30, 70], dev), want_lse=True)
    ref.check_attention(kv, 0, q, out, [0, 1], [0, 30, 70], 128 ** -0.5, True, lse)
    assert out[:25].eq(0).all() and lse[:25].isneginf().all()


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_attention_ignores_what_is_not_the_sequences(pkg, dev, dtype):
    """NaN codes and scales past the lengths, in unused pages and in pages that a row
    does not see, do not reach it; a NaN that it sees does."""
    m, kv = make(pkg, dev, hk=2, d=64, page=16, dtype=dtype, slots=4, n_pages=20)
    grow(pkg, m, kv, [0, 1, 2], [21, 40, 90], dev, 4)
    nan = 0x7f if dtype == E4M3 else 0x80
    for t in (kv.k, kv.v):
        u = t.view(torch.uint8)
        free = [i for i, r in enumerate(m.ref) if r == 0]
        u[0, free] = nan
        u[0, m.rows[0][1], :, 5:] = nan
        u[0, m.rows[1][2], :, 8:] = nan
    kv.k_scale[0, free] = kv.v_scale[0, free] = float("nan")
    kv.v_scale[0, m.rows[2][5]] = kv.k_scale[0, m.rows[2][5]] = float("nan")  # positions 80..89
    q = torch.randn(3, 4, 64).half().to(dev)
    out = pkg.ops.attention_paged_decode(kv, 0, q, i32([0, 1, 2], dev))
    assert out[2].isnan().all() and out[:2].isfinite().all()
    ref.check_attention(kv, 0, q, out[:2], [0, 1], [0, 1, 2], 0.125)
    qs = torch.randn(40, 4, 64).half().to(dev)
    out = pkg.ops.attention_paged_prefill(kv, 0, qs, i32([2], dev), i32([0, 40], dev))
    assert out[30:].isnan().all() and out[:30].isfinite().all()
    kv.length[2] = 80
    ref.check_attention(kv, 0, qs[:30], out[:30], [2], [0, 30], 0.125)


def test_bad_entries_are_left_out(pkg, dev):
    """Page ids, slots, lengths and row counts out of range: flagged, skipped, nothing faults."""
    m, kv = make(pkg, dev, hk=2, d=64, page=16, slots=4, max_pages=5)
    grow(pkg, m, kv, [0, 1], [48, 30], dev, 4)
    ops = pkg.ops
    q = torch.randn(2, 4, 64).half().to(dev)
    q2 = torch.randn(20, 4, 64).half().to(dev)
    good = ops.attention_paged_decode(kv, 0, q, i32([1, 1], dev))
    for bad in (-1, kv.n_pages, 2 ** 31 - 1):
        kv.table[0, 1] = bad
        out = ops.attention_paged_decode(kv, 0, q, i32([0, 1], dev))
        out2 = ops.attention_paged_prefill(kv, 0, q2, i32([0], dev), i32([0, 20], dev))
        assert pkg.device_status() & 2
        assert torch.equal(out[1], good[1]) and out.isfinite().all() and out2.isfinite().all()
    # the bad page's keys are left out: as the sequence without them
    row = kv.table[0].clone()
    kv.table[0, 1], kv.length[0] = row[2], 32
    short = ops.attention_paged_decode(kv, 0, q, i32([0, 1], dev))
    kv.table[0], kv.length[0] = row, 48
    assert (short[0].float() - out[0].float()).abs().max() < 2e-3  # the same sums in another split
    for slots in ([7, 1], [-3, 1]):
        out = ops.attention_paged_decode(kv, 0, q, i32(slots, dev))
        assert pkg.device_status() & 2
        assert out[0].eq(0).all() and torch.equal(out[1], good[1])
    kv.length[0] = 1000
    ops.attention_paged_decode(kv, 0, q, i32([0, 1], dev))
    assert pkg.device_status() & 2
    kv.length[0] = 48
    rows = torch.randn(20, 128).half().to(dev)
    before = kv.k.clone()
    for slots, cu in (([9], [0, 20]), ([1], [0, 40]), ([1], [20, 0]), ([1], [-5, 5])):
        ops.kv_pages_write(kv, 0, rows, rows, i32(slots, dev), i32(cu, dev))
        if cu != [0, 20]:
            ops.attention_paged_prefill(kv, 0, q2, i32(slots, dev), i32(cu, dev))
        assert pkg.device_status() & 2
    assert torch.equal(kv.k, before)


@pytest.mark.parametrize("length", [65, 2 ** 31 - 1, -1, -2 ** 31])
def test_lengths_that_a_row_cannot_hold_are_left_out(pkg, dev, length):
    """A slot whose length is beyond its table row, every entry of which is in use: its rows are not
    written and its attention is that of an empty slot; the batch's other slot is as it was."""
    m, kv = make(pkg, dev, page=16, d=64, hk=2, slots=3, max_pages=4)
    grow(pkg, m, kv, [0, 1], [64, 20], dev, 1)
    q = torch.randn(60, 8, 64, generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = pkg.ops.attention_paged_decode(kv, 0, q[:2])[1]
    rows = 5 * torch.randn(41, 128, generator=torch.Generator().manual_seed(2)).half()
    on = rows.to(dev)
    kv.length[0] = length
    pkg.ops.kv_pages_write(kv, 0, on[:1], on[:1], i32([0], dev))
    assert pkg.device_status() == 2
    pkg.ops.kv_pages_write(kv, 0, on, on, i32([0, 1], dev), i32([0, 40, 41], dev))
    assert pkg.device_status() == 2
    out, lse = pkg.ops.attention_paged_decode(kv, 0, q[:2], want_lse=True)
    assert pkg.device_status() == 2
    assert out[0].eq(0).all() and lse[0].isneginf().all()
    for r in (3, 50):  # both kernels
        pre, lse = pkg.ops.attention_paged_prefill(kv, 0, q[:r + 1], None, i32([0, r, r + 1], dev), want_lse=True)
        assert pkg.device_status() == 2
        assert pre[:r].eq(0).all() and lse[:r].isneginf().all() and pre[r].isfinite().all()
    kv.length[0] = 64
    assert not torch.equal(out[1], want)  # its last row is another one now
    m.write(0, rows[40:], rows[40:], [1], [0, 1])
    m.same_books(kv)
    m.same_data(kv)


@pytest.mark.parametrize("n_tokens", [4095, 16384])
def test_rows_that_overlap_without_end(pkg, dev, n_tokens):
    """Row counts that go back and forth, so that 512 sequences have all of the rows: more work
    than 32 bits count (both attention kernels).  Flagged, nothing done."""
    hk, group, d, page = 8, 8, 64, 128
    kv = pkg.ops.PagedKV.empty(1, 2, hk, page, d, 1, 1024, I8, dev)
    kv.table.zero_()
    kv.length.fill_(1024 * page)
    q = torch.zeros(n_tokens, hk * group, d, dtype=torch.float16, device=dev)
    cu = i32([0, n_tokens] * 512 + [0], dev)
    out = torch.full_like(q, 3)
    pkg.ops.attention_paged_prefill(kv, 0, q, torch.zeros(1024, dtype=torch.int32, device=dev), cu, is_causal=False,
                                    out=out)
    assert pkg.device_status() & 2
    assert out.eq(3).all()


def test_codes_past_4_gib(pkg, dev):
    """A pool whose byte offsets pass 32 bits: the last pages."""
    n_pages = 70000  # 8 heads x 64 x 128 bytes each: 4.6 GB a side
    kv = pkg.ops.PagedKV.empty(1, n_pages, 8, 64, 128, 2, 4, I8, dev)
    m = ref.Model(1, 4, 8, 64, 128, 2, 4, I8)
    m.extend([1, 0], [150, 9])
    rows = torch.randn(159, 2, 1024).half()
    m.write(0, rows[:, 0], rows[:, 1], [1, 0], [0, 150, 159])
    kv.ref.fill_(1)
    kv.ref[n_pages - 4:] = 0
    on = rows.to(dev)
    assert int(pkg.ops.kv_pages_extend(kv, i32([1, 0], dev), i32([150, 9], dev))) == 0
    assert kv.table[1].tolist() == [n_pages - 4, n_pages - 3, n_pages - 2, -1]
    pkg.ops.kv_pages_write(kv, 0, on[:, 0], on[:, 1], i32([1, 0], dev), i32([0, 150, 159], dev))
    small = pkg.ops.PagedKV.empty(1, 4, 8, 64, 128, 2, 4, I8, dev)
    m.load(small)
    for e in range(3):
        n = min(64, 150 - 64 * e)
        assert torch.equal(kv.k[0, n_pages - 4 + e, :, :n], small.k[0, e, :, :n])
    q = torch.randn(2, 32, 128).half().to(dev)
    want = pkg.ops.attention_paged_decode(small, 0, q)
    assert torch.equal(pkg.ops.attention_paged_decode(kv, 0, q), want)
    qs = torch.randn(100, 32, 128).half().to(dev)
    cu = i32([0, 100], dev)
    want = pkg.ops.attention_paged_prefill(small, 0, qs, i32([1], dev), cu)
    assert torch.equal(pkg.ops.attention_paged_prefill(kv, 0, qs, i32([1], dev), cu), want)


# ---------------------------------------------------------- used together


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_serving_run(pkg, dev, dtype):
    """Prompts enter, tokens are generated, sequences fork, grow apart, end, the pool is
    compacted, more tokens: attention right and the books as the restatement's throughout."""
    heads, hk, d, page = 8, 2, 128, 32
    m, kv = make(pkg, dev, layers=2, hk=hk, d=d, page=page, dtype=dtype, slots=8, n_pages=40, max_pages=10)
    g = torch.Generator().manual_seed(1)

    def step(slots, n_new, seed):
        assert grow(pkg, m, kv, slots, n_new, dev, seed) == 0
        cu = [0]
        for n in n_new:
            cu.append(cu[-1] + n)
        q = torch.randn(cu[-1], heads, d, generator=g).half().to(dev)
        for layer in range(2):
            out = pkg.ops.attention_paged_prefill(kv, layer, q, i32(slots, dev), i32(cu, dev))
            ref.check_attention(kv, layer, q, out, slots, cu, d ** -0.5)
            if max(n_new) == 1:
                one = pkg.ops.attention_paged_decode(kv, layer, q, i32(slots, dev))
                ref.check_attention(kv, layer, q, one, slots, cu, d ** -0.5)
        m.same_books(kv)

    step([0, 1, 2], [70, 33, 5], 1)
    for i in range(3):
        step([0, 1, 2], [1, 1, 1], 10 + i)
    assert int(pkg.ops.kv_pages_fork(kv, i32([0, 0, 1], dev), i32([5, 6, 7], dev))) == m.fork([0, 0, 1], [5, 6, 7])
    step([0, 5, 6, 7, 1], [1, 1, 1, 1, 1], 20)
    step([6, 7], [4, 40], 21)  # draft tokens; a second turn's prompt
    pkg.ops.kv_pages_free(kv, i32([0, 2], dev))
    m.free([0, 2])
    assert pkg.ops.kv_pages_compact(kv).tolist() == m.compact()
    m.same_books(kv)
    m.same_data(kv)
    step([5, 1, 7], [1, 1, 1], 30)
    m.same_data(kv)
    assert pkg.device_status() == 0


def test_captured_decode_step(pkg, dev):
    """extend, write and decode captured once, replayed as the sequences grow across
    pages; two graphs of one cache, replayed on two streams that wait for each other."""
    heads, hk, d, page = 8, 2, 64, 16
    m, kv = make(pkg, dev, hk=hk, d=d, page=page, slots=4, n_pages=30, max_pages=8)
    grow(pkg, m, kv, [0, 1, 2, 3], [14, 30, 1, 60], dev, 1)
    groups = ([0, 3], [1, 2])
    rows = [torch.zeros(2, 2, hk * d, device=dev, dtype=torch.float16) for _ in groups]
    qs = [torch.zeros(2, heads, d, device=dev, dtype=torch.float16) for _ in groups]
    slots = [i32(s, dev) for s in groups]
    ones = i32([1, 1], dev)
    outs, graphs = [], []
    for r, q, s in zip(rows, qs, slots):
        pkg.ops.attention_paged_decode(kv, 0, q, s)  # warm
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st = pkg.ops.kv_pages_extend(kv, s, ones)
            pkg.ops.kv_pages_write(kv, 0, r[:, 0], r[:, 1], s)
            outs.append((pkg.ops.attention_paged_decode(kv, 0, q, s), st))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in groups]
    m.same_books(kv)
    for step in range(6):
        for i, grp in enumerate(groups):
            new = torch.randn(2, 2, hk * d, generator=torch.Generator().manual_seed(10 * step + i)).half()
            rows[i].copy_(new)
            qs[i].copy_(torch.randn(2, heads, d, generator=torch.Generator().manual_seed(100 * step + i)))
            with torch.cuda.stream(streams[i]):
                streams[i].wait_stream(torch.cuda.current_stream() if i == 0 else streams[0])
                streams[i].wait_stream(torch.cuda.default_stream())
                graphs[i].replay()
            assert m.extend(grp, [1, 1]) == 0
            m.write(0, new[:, 0], new[:, 1], grp, [0, 1, 2])
        torch.cuda.synchronize()
        m.same_books(kv)
        for i, grp in enumerate(groups):
            assert int(outs[i][1]) == 0
            ref.check_attention(kv, 0, qs[i], outs[i][0], grp, [0, 1, 2], d ** -0.5)
    m.same_data(kv)


@pytest.mark.parametrize("ragged", [False, True])
def test_a_step_whose_extend_is_refused_leaves_the_cache(pkg, dev, ragged):
    """extend, write and decode captured once, the write with the extend's status: a replay that
    lacks pages changes nothing, and the next one after a free goes on as if it had not been."""
    heads, hk, d, page = 8, 2, 64, 16
    m, kv = make(pkg, dev, layers=2, hk=hk, d=d, page=page, slots=5, n_pages=7, max_pages=4)
    grow(pkg, m, kv, [0, 1, 4], [30, 32, 17], dev, 1)  # 2 + 2 + 2 pages; slot 1 is at a page's end
    assert int(pkg.ops.kv_pages_fork(kv, i32([1], dev), i32([3], dev))) == m.fork([1], [3]) == 0
    slots, n = i32([0, 1, 3], dev), i32([1, 1, 1], dev)
    cu = i32([0, 1, 2, 3], dev) if ragged else None
    rows = torch.zeros(3, 2, hk * d, device=dev, dtype=torch.float16)
    q = torch.randn(3, heads, d, generator=torch.Generator().manual_seed(2)).half().to(dev)

    def step():
        st = pkg.ops.kv_pages_extend(kv, slots, n)
        for layer in range(2):
            pkg.ops.kv_pages_write(kv, layer, rows[:, 0], rows[:, 1], slots, cu, status=st)
        return st, pkg.ops.attention_paged_decode(kv, 1, q, slots)

    pkg.ops.attention_paged_decode(kv, 0, q, slots)  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st, out = step()
    for i in range(3):  # two pages are wanted, one is free; the third time two more are
        new = torch.randn(3, 2, hk * d, generator=torch.Generator().manual_seed(10 + i)).half()
        rows.copy_(9 * new)
        if i == 2:
            pkg.ops.kv_pages_free(kv, i32([4], dev))
            m.free([4])
        graph.replay()
        want = m.extend([0, 1, 3], [1, 1, 1])
        assert int(st) == want == (0 if i == 2 else 1)
        if want == 0:
            for layer in range(2):
                m.write(layer, 9 * new[:, 0], 9 * new[:, 1], [0, 1, 3], [0, 1, 2, 3])
        m.same_books(kv)
        m.same_data(kv)
    assert pkg.device_status() == 0
    ref.check_attention(kv, 1, q, out, [0, 1, 3], [0, 1, 2, 3], d ** -0.5)
    with pytest.raises(ValueError, match="status must be the one word"):
        pkg.ops.kv_pages_write(kv, 0, rows[:, 0], rows[:, 1], slots, cu, status=n)


def test_two_attentions_at_once(pkg, dev):
    """Calls on two streams that run together do not share anything."""
    m, kv = make(pkg, dev, hk=2, d=128, page=64, slots=3, n_pages=150, max_pages=70)
    grow(pkg, m, kv, [0, 1, 2], [4000, 2500, 700], dev, 3)
    q = torch.randn(3, 16, 128).half().to(dev)
    qs = torch.randn(300, 16, 128).half().to(dev)
    cu = i32([0, 200, 300], dev)
    want = pkg.ops.attention_paged_decode(kv, 0, q)
    want2 = pkg.ops.attention_paged_prefill(kv, 0, qs, i32([2, 0], dev), cu)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(a):
            got.append((pkg.ops.attention_paged_decode(kv, 0, q), want))
        with torch.cuda.stream(b):
            got.append((pkg.ops.attention_paged_prefill(kv, 0, qs, i32([2, 0], dev), cu), want2))
    torch.cuda.synchronize()
    for x, w in got:
        assert torch.equal(x, w)
