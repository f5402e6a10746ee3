"""GPU: the bounded waits of attention over the paged cache."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

# Every eighth sequence has rows in the second half of its items; a CTA has some 50 items, and goes
# through those of seven sequences, about 6 ms, before side B has rows again.
_CHILD = r"""
import sys
sys.path.insert(0, {root!r})
import torch
from tests.conftest import load_package
pkg = load_package()
ops, dev = pkg.ops, torch.device("cuda:0")
torch.cuda.set_device(dev)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
n, keys, hk, d, page = 1000, 8192, 8, 128, 128
kv = ops.PagedKV.empty(1, keys // page, hk, page, d, n, keys // page, torch.int8, dev)
assert int(ops.kv_pages_extend(kv, i32([0]), i32([keys]))) == 0
x = torch.randn(keys, 2, hk * d, generator=torch.Generator().manual_seed(1)).half().to(dev)
ops.kv_pages_write(kv, 0, x[:, 0], x[:, 1], i32([0]), i32([0, keys]))
assert int(ops.kv_pages_fork(kv, i32([0] * (n - 1)), i32(list(range(1, n))))) == 0
cu = [0]
for i in range(n):
    cu.append(cu[-1] + (64 if i % 8 == 7 else 32))
q = torch.randn(64, 32, d, generator=torch.Generator().manual_seed(2)).half().to(dev)
out = torch.full((cu[-1], 32, d), 7.0, device=dev, dtype=torch.float16)
rows = torch.cat([torch.arange(64 if i % 8 == 7 else 32) for i in range(n)]).to(dev)
ops.attention_paged_prefill(kv, 0, q[rows], None, i32(cu), out=out, is_causal=False)
flags = pkg.device_status()
# each token of q over the same keys, whatever its sequence: in small calls of their own
want = torch.cat([ops.attention_paged_prefill(kv, 0, q[a:a + 32], i32([0]), i32([0, 32]), is_causal=False) for a in (0, 32)])
left = out.eq(7).all(-1)
err = (out.float() - want[rows].float()).abs().amax(-1)
assert pkg.device_status() == 0
# rows are as they were or right (another split of the keys: roundings of 16 bits)
assert (left | (err < 2.0 ** -8)).all(), (err * ~left).max()
print("FLAGS", flags, "LEFT", int(left.sum()))
"""


@pytest.mark.parametrize("limit", ["1", None])
def test_a_side_without_rows_waits_as_long_as_the_other_works(dev, limit):
    """Side B's wait for its next item lasts as long as the items in between take, which may be
    any multiple of the limit for one tile."""
    env = dict(os.environ)
    env.pop("ENGINE_WAIT_TIMEOUT_MS", None)
    if limit:
        env["ENGINE_WAIT_TIMEOUT_MS"] = limit
    r = subprocess.run([sys.executable, "-c", _CHILD.format(root=str(ROOT))], env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split() == ["FLAGS", "0", "LEFT", "0"], r.stdout
