"""CPU: the paged cache's calls refuse bad arguments before any device work, and the
tests' restatement of the operators holds its own definitions."""
from __future__ import annotations

import pytest
import torch

from tests import paged_ref as ref

P = 4096  # a non-null, aligned pointer value; never dereferenced by a rejected call


def desc(pkg, **over):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, table=P, length=P, ref=P, n_layers=2, n_pages=100,
             n_kv_heads=8, page_size=64, head_dim=128, n_slots=10, max_pages=20, type=pkg.cuda.KV_I8)
    f.update(over)
    return pkg.KvPages(*(f[n] for n, _ in pkg.KvPages._fields_))


def _throws(pkg, fn, *args, substr, code=1):
    with pytest.raises(pkg.EngineError) as e:
        fn(*args)
    assert substr in str(e.value), str(e.value)
    assert e.value.code == code


BAD = [({"k": 0}, "k/v is null"), ({"v_scale": 0}, "k_scale/v_scale is null"),
       ({"table": 0}, "table/length/ref is null"), ({"ref": 0}, "is null"), ({"type": 0}, "type must be"),
       ({"page_size": 48}, "page_size must be"), ({"head_dim": 96}, "head_dim must be 64 or 128"),
       ({"n_pages": 0}, "must be positive"), ({"n_slots": -1}, "must be positive"),
       ({"k": P + 8}, "16-byte aligned")]


@pytest.mark.parametrize("over,msg", BAD)
def test_every_call_checks_the_cache(pkg, over, msg):
    c, kv = pkg.cuda, desc(pkg, **over)
    _throws(pkg, c.kv_pages_extend, kv, P, P, P, 1, substr=msg)
    _throws(pkg, c.kv_pages_fork, kv, P, P, P, 1, substr=msg)
    _throws(pkg, c.kv_pages_free, kv, P, 1, substr=msg)
    _throws(pkg, c.kv_pages_compact, kv, substr=msg)
    _throws(pkg, c.kv_pages_write, kv, 0, P, P, 1024, P, P, 1, 1, substr=msg)
    _throws(pkg, c.attention_paged_decode, kv, 0, P, 4096, P, P, 0, 1, 32, 0.1, substr=msg)
    _throws(pkg, c.attention_paged_prefill, kv, 0, P, 4096, P, P, P, 0, 1, 1, 32, 0.1, substr=msg)


def test_dimensions_too_large(pkg):
    c = pkg.cuda
    for over in ({"n_pages": 2 ** 26}, {"max_pages": 2 ** 26}, {"n_kv_heads": 70000}, {"n_layers": 70000}):
        _throws(pkg, c.kv_pages_free, desc(pkg, **over), P, 1, substr="too large", code=3)


def test_arguments(pkg):
    c, kv = pkg.cuda, desc(pkg)
    ex, fo, fr, wr = c.kv_pages_extend, c.kv_pages_fork, c.kv_pages_free, c.kv_pages_write
    de, pr = c.attention_paged_decode, c.attention_paged_prefill
    _throws(pkg, ex, 0, P, P, P, 1, substr="kv is null")
    _throws(pkg, ex, kv, P, P, P, -1, substr="non-negative")
    _throws(pkg, ex, kv, P, P, P, c.KV_MAX_SLOTS + 1, substr="ENGINE_KV_MAX_SLOTS")
    _throws(pkg, ex, kv, 0, P, P, 11, substr="n > n_slots")
    _throws(pkg, ex, kv, P, P, 0, 1, substr="status is null")
    _throws(pkg, ex, kv, P, 0, P, 1, substr="n_new is null")
    _throws(pkg, fo, kv, P, P, P, -1, substr="non-negative")
    _throws(pkg, fo, kv, P, P, P, c.KV_MAX_SLOTS + 1, substr="ENGINE_KV_MAX_SLOTS")
    _throws(pkg, fo, kv, P, 0, P, 1, substr="parents/children is null")
    _throws(pkg, fo, kv, P, P, 0, 1, substr="status is null")
    _throws(pkg, fr, kv, P, -1, substr="non-negative")
    _throws(pkg, fr, kv, 0, 11, substr="n > n_slots")
    fr(kv, 0, 0)  # nothing to do
    _throws(pkg, wr, kv, 2, P, P, 1024, P, P, 1, 1, substr="layer out of range")
    _throws(pkg, wr, kv, -1, P, P, 1024, P, P, 1, 1, substr="layer out of range")
    _throws(pkg, wr, kv, 0, P, P, 1023, P, P, 1, 1, substr="row_pitch <")
    _throws(pkg, wr, kv, 0, P, P, 1024, P, P, -1, 1, substr="non-negative")
    _throws(pkg, wr, kv, 0, P, P, 1024, P, 0, 2, 3, substr="cu_new is null")
    _throws(pkg, wr, kv, 0, P, P, 1024, 0, P, 11, 20, substr="n_seq > n_slots")
    _throws(pkg, wr, kv, 0, 0, P, 1024, P, P, 1, 1, substr="k_new/v_new is null")
    _throws(pkg, wr, kv, 0, P + 2, P, 1024, P, P, 1, 1, substr="16-byte aligned", code=3)
    _throws(pkg, wr, kv, 0, P, P, 1028, P, P, 1, 1, substr="multiple of 8", code=3)
    wr(kv, 0, 0, 0, 1024, 0, 0, 0, 0)
    for f, mid in ((de, (P,)), (pr, (P, P))):
        tail = (1,) if f is de else (1, 1)
        _throws(pkg, f, kv, 5, P, 4096, *mid, P, 0, *tail, 32, 0.1, substr="layer out of range")
        _throws(pkg, f, kv, 0, P, 4096, *mid, P, 0, *tail, 30, 0.1, substr="divisible by n_kv_heads")
        _throws(pkg, f, kv, 0, P, 4096, *mid, P, 0, *tail, 0, 0.1, substr="n_heads must be positive")
        _throws(pkg, f, kv, 0, P, 4000, *mid, P, 0, *tail, 32, 0.1, substr="q_pitch <")
        _throws(pkg, f, kv, 0, P, 4096, *mid, P, 0, *tail, 32, float("nan"), substr="scale must be")
        _throws(pkg, f, kv, 0, P, 4096, *mid, P, 0, *tail, 32, -0.1, substr="scale must be")
        _throws(pkg, f, kv, 0, 0, 4096, *mid, P, 0, *tail, 32, 0.1, substr="q is null")
        _throws(pkg, f, kv, 0, P, 4096, *mid, 0, 0, *tail, 32, 0.1, substr="out is null")
        _throws(pkg, f, kv, 0, P + 2, 4096, *mid, P, 0, *tail, 32, 0.1, substr="16-byte", code=3)
        _throws(pkg, f, kv, 0, P, 4100, *mid, P, 0, *tail, 32, 0.1, substr="multiple of 8", code=3)
    _throws(pkg, de, kv, 0, P, 4096, 0, P, 0, 11, 32, 0.1, substr="n_seq > n_slots")
    _throws(pkg, pr, kv, 0, P, 4096, P, 0, P, 0, 1, 1, 32, 0.1, substr="cu_q is null")
    _throws(pkg, pr, kv, 0, P, 4096, P, P, P, 0, 1, 2 ** 27, 32, 0.1, substr="too large", code=3)
    de(kv, 0, 0, 4096, 0, 0, 0, 0, 32, 0.1)          # no sequences
    pr(kv, 0, 0, 4096, 0, 0, 0, 0, 3, 0, 32, 0.1)    # no rows


def test_paged_kv_checks_its_tensors(pkg):
    """Tensors that are not on a GPU, of another type or of other shapes."""
    z = torch.zeros
    good = dict(k=z(1, 4, 2, 16, 64, dtype=torch.int8), v=z(1, 4, 2, 16, 64, dtype=torch.int8), k_scale=z(1, 4, 2),
                v_scale=z(1, 4, 2), table=z(3, 5, dtype=torch.int32), length=z(3, dtype=torch.int32), ref=z(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.ops.PagedKV(**good)
    with pytest.raises(TypeError, match="int8 or float8"):
        pkg.ops.PagedKV(**{**good, "k": good["k"].half()})
    with pytest.raises(ValueError, match="of one shape"):
        pkg.ops.PagedKV(**{**good, "v": good["v"][:, :3]})
    with pytest.raises(ValueError, match="of one shape"):
        pkg.ops.PagedKV(**{**good, "k": good["k"][0], "v": good["v"][0]})


def test_cpp_adapter(pkg, tmp_path):
    """engine::cuda::kv_pages_* / attention_paged_* of kernels_b200.hpp: they compile, link,
    and throw EngineError with the library's message before any device work."""
    import subprocess

    src = r"""
#include <cstdio>
#include <engine/kernels_b200.hpp>
namespace ec = engine::cuda;
template <typename F> static int throws(F f, const char* part) {
  try { f(); } catch (const engine::EngineError& e) {
    if (std::string(e.what()).find(part) != std::string::npos) return 0;
    std::printf("%s\n", e.what());
  }
  return 1;
}
int main() {
  ec::KvPages kv = {};
  auto* p = reinterpret_cast<void*>(4096);
  auto* i = reinterpret_cast<std::int32_t*>(4096);
  auto* h = reinterpret_cast<__half*>(4096);
  int bad = throws([&] { ec::kv_pages_compact(kv); }, "k/v is null");
  kv.k = kv.v = p;
  kv.k_scale = kv.v_scale = reinterpret_cast<float*>(p);
  kv.table = kv.length = kv.ref = i;
  kv.n_layers = 1; kv.n_pages = 4; kv.n_kv_heads = 2; kv.page_size = 16; kv.head_dim = 64;
  kv.n_slots = 2; kv.max_pages = 2; kv.type = ENGINE_KV_E4M3;
  bad += throws([&] { ec::kv_pages_extend(kv, i, i, nullptr, 1); }, "status is null");
  bad += throws([&] { ec::kv_pages_fork(kv, i, nullptr, i, 1); }, "children is null");
  bad += throws([&] { ec::kv_pages_free(kv, i, -1); }, "non-negative");
  bad += throws([&] { ec::kv_pages_write(kv, 1, h, h, 128, i, i, 1, 1); }, "layer out of range");
  bad += throws([&] { ec::attention_paged_decode(kv, 0, h, 256, i, h, 1, 3, 0.125f); }, "divisible");
  bad += throws([&] { ec::attention_paged_prefill(kv, 0, h, 256, i, nullptr, h, 1, 1, 4, 0.125f); }, "cu_q is null");
  return bad;
}
"""
    from tests.conftest import ROOT

    exe = tmp_path / "kv_pages"
    (tmp_path / "kv_pages.cpp").write_text(src)
    r = subprocess.run(["g++", "-std=c++17", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include",
                        str(tmp_path / "kv_pages.cpp"), "-o", str(exe), str(pkg.LIB_PATH),
                        f"-Wl,-rpath,{pkg.LIB_PATH.parent}"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


def test_calls_check_their_tensors(pkg, monkeypatch):
    """Another current device, other types, shapes and strides: refused in Python, with a
    stand-in for the cache (nothing reaches the library)."""
    from types import SimpleNamespace

    ops = pkg.ops
    kv = SimpleNamespace(device_index=1, handle=0, width=128, head_dim=64, n_pages=4)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    i = torch.zeros(2, dtype=torch.int32)
    h = torch.zeros(2, 128).half()
    for call in (lambda: ops.kv_pages_extend(kv, i, i), lambda: ops.kv_pages_fork(kv, i, i),
                 lambda: ops.kv_pages_free(kv, i), lambda: ops.kv_pages_compact(kv),
                 lambda: ops.kv_pages_write(kv, 0, h, h), lambda: ops.attention_paged_decode(kv, 0, h),
                 lambda: ops.attention_paged_prefill(kv, 0, h, None, i)):
        with pytest.raises(ValueError, match="not the current device"):
            call()
    kv.device_index = 0
    with pytest.raises(ValueError, match="n_new must be a CUDA tensor"):
        ops.kv_pages_extend(kv, None, i)
    with pytest.raises(ValueError, match="slots must be a CUDA tensor"):
        ops.kv_pages_free(kv, i)
    with pytest.raises(TypeError, match="k_rows must be a CUDA float16"):
        ops.kv_pages_write(kv, 0, h, h)
    with pytest.raises(TypeError, match="q must be a CUDA float16"):
        ops.attention_paged_decode(kv, 0, h)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_restatement_rounds_to_the_nearest(dtype):
    """The Model's codes: each value within half a step of what was written, also after
    a page grew (one more half step for each growth)."""
    m = ref.Model(1, 8, 2, 16, 64, 2, 4, dtype)
    g = torch.Generator().manual_seed(0)
    assert m.extend([1], [21]) == 0
    k, v = (torch.randn(21, 128, generator=g).half() for _ in range(2))
    m.write(0, k, v, [1], [0, 21])
    for i, x in ((0, k), (1, v)):
        for e, w in enumerate(m.rows[1]):
            n = min(16, 21 - 16 * e)
            a = m.scale[i, 0, w].double()[:, None, None]
            got = m.code[i, 0, w, :, :n].double() * a
            want = x[16 * e:16 * e + n].double().view(n, 2, 64).transpose(0, 1)
            step = a * 0.5 if dtype == torch.int8 else torch.maximum(2.0 ** -4 * want.abs(), a * 2.0 ** -10)
            assert ((got - want).abs() <= step * (1 + 2.0 ** -20) + want.abs() * 2.0 ** -22).all()
    assert m.fork([1], [0]) == 0 and m.ref == [2, 1, 1, 0, 0, 0, 0, 0]
    m.free([1])
    assert m.compact() == [0, -1, 1, -1, -1, -1, -1, -1] and m.rows[0] == [0, 1]


def test_write_with_a_status_checks_its_arguments(pkg):
    """The call with the word of an extend refuses what the call without it does."""
    w, kv = pkg.lib().engine_cuda_kv_pages_write_if, desc(pkg)
    import ctypes

    def bad(*args, code=1, substr=""):
        assert w(ctypes.addressof(kv), *args) == code
        assert substr in pkg.lib().engine_last_error().decode()

    bad(2, P, P, 1024, P, P, 1, 1, P, 0, substr="layer out of range")
    bad(0, P, P, 1023, P, P, 1, 1, P, 0, substr="row_pitch <")
    bad(0, 0, P, 1024, P, P, 1, 1, P, 0, substr="k_new/v_new is null")
    bad(0, P, P, 1028, P, P, 1, 1, P, 0, code=3, substr="multiple of 8")
    assert w(ctypes.addressof(kv), 0, 0, 0, 1024, 0, 0, 0, 0, P, 0) == 0  # nothing to write
