"""Paged-cache and sampling entry points on the CPU: what the C ABI refuses before any HIP call, and the device
helpers that turn positions into pages, compiled for the host."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from autokernel_amd import _lib
    return _lib.load()


def test_paged_attention_refusals(lib):
    from autokernel_amd import _lib
    x, s = ctypes.c_void_p(4096), _lib.i64_array([64, 64, 64])
    base = dict(dtype=1, q=x, kc=x, vc=x, o=x, table=x, starts=x, lens=x, T=4, B=2, Hq=4, Hkv=2, D=64, pages=8, page=16,
                width=4, stride=4, qs=s, ks=s, vs=s, os=s, scale=1.0, ws=None, wsb=0, stream=None)

    def call(**kw):
        return lib.ak_paged_attn(*{**base, **kw}.values())
    for bad in (dict(dtype=7), dict(T=-1), dict(B=-1), dict(Hq=5), dict(Hkv=0), dict(D=0), dict(pages=-1), dict(page=0),
                dict(width=-1), dict(stride=3), dict(q=None), dict(kc=None), dict(vc=None), dict(o=None), dict(table=None),
                dict(starts=None), dict(lens=None), dict(qs=None), dict(os=None), dict(ks=None), dict(vs=None),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(T=1 << 31),
                dict(pages=1 << 31), dict(page=1 << 20, width=1 << 12, stride=1 << 12), dict(Hq=1 << 20, Hkv=1),
                dict(scale=2.1e38), dict(ks=_lib.i64_array([64, -64, 64])), dict(vs=_lib.i64_array([-1, 64, 64])),
                dict(width=400, stride=400),                                # needs a workspace
                dict(width=400, stride=400, ws=ctypes.c_void_p(8), wsb=1 << 40)):  # misaligned
        assert call(**bad) == _lib.AK_EINVAL, bad
    assert call(D=257) == _lib.AK_EUNSUPPORTED
    for empty in (dict(T=0), dict(B=0, starts=None, lens=None, table=None), dict(Hq=0)):
        assert call(**empty) == _lib.AK_OK, empty
    need = lib.ak_paged_attn_workspace_bytes
    assert need(1, 4, 2, 4, 2, 64, 16, 4) == 0          # 64 positions: one slice
    assert need(1, 4, 2, 4, 2, 64, 16, 400) > 0
    assert need(1, 0, 2, 4, 2, 64, 16, 400) == 0 and need(9, 4, 2, 4, 2, 64, 16, 400) == 0
    assert need(1, 4, 2, 4, 3, 64, 16, 400) == 0 and need(1, 4, 2, 4, 2, 64, -16, 400) == 0


def test_kv_append_refusals(lib):
    from autokernel_amd import _lib
    x, s = ctypes.c_void_p(4096), _lib.i64_array([64, 64, 64])
    base = dict(dtype=1, q=x, k=x, v=x, qo=x, kc=x, vc=x, cos=x, sin=x, table=x, starts=x, lens=x, T=4, B=2, Hq=4, Hkv=2,
                D=64, rot=64, rows=100, pages=8, page=16, width=4, stride=4, qs=s, ks=s, vs=s, os=s, kcs=s, vcs=s, inter=1,
                stream=None)

    def call(**kw):
        return lib.ak_kv_append(*{**base, **kw}.values())
    for bad in (dict(dtype=7), dict(T=-1), dict(B=-1), dict(Hq=-1), dict(D=0), dict(rot=63), dict(rot=66), dict(rot=-2),
                dict(rows=-1), dict(page=0), dict(stride=3), dict(q=None), dict(k=None), dict(v=None), dict(qo=None),
                dict(kc=None), dict(vc=None), dict(cos=None), dict(sin=None), dict(rot=0), dict(qs=None), dict(kcs=None),
                dict(kcs=_lib.i64_array([64, 64, -64])), dict(vcs=_lib.i64_array([-64, 64, 64])),
                dict(table=None), dict(starts=None), dict(lens=None), dict(T=1 << 31), dict(Hkv=1 << 20)):
        assert call(**bad) == _lib.AK_EINVAL, bad
    assert call(D=258) == _lib.AK_EUNSUPPORTED
    for empty in (dict(T=0), dict(B=0, starts=None, lens=None, table=None), dict(Hq=0, Hkv=0, rot=0)):
        assert call(**empty) == _lib.AK_OK, empty


PAGE_PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_common.h"
using namespace ak;
// every position of several page sizes, tables with every kind of wrong entry: the page, or -1, never an access
// outside the table
int main() {
  srand(1);
  for (int page : {1, 3, 8, 16, 24, 100, 1024, 65536, 1 << 30}) {
    const int width = page > 60000 ? 1 : 37, B = 3;
    const int64_t stride = width + 2, pages = 50;
    std::vector<int32_t> table(2 * stride + width);  // the last row ends with the table
    for (auto& e : table) {
      const int r = rand() % 8;
      e = r == 0 ? -1 : r == 1 ? 50 : r == 2 ? INT32_MIN : r == 3 ? INT32_MAX : rand() % 50;
    }
    if (!paged_args_ok(table.data(), table.data(), table.data(), 4, B, pages, page, width, stride)) return 1;
    const PagedSeqs s = make_paged(table.data(), nullptr, nullptr, 4, B, pages, page, width, stride);
    for (int b = 0; b < B; ++b)
      for (int64_t pos = 0; pos < (int64_t)width * page + 3 * (int64_t)page; pos += page > 60000 ? 9973 : 1) {
        const int64_t in = pos / page;
        const int64_t want = in >= width || table.at(b * stride + in) < 0 || table.at(b * stride + in) >= pages
                                 ? -1 : table.at(b * stride + in);
        if (paged_page_of(s, b, pos) != want) return printf("page %d b %d pos %lld\n", page, b, (long long)pos), 1;
      }
    for (int64_t pos : {(int64_t)INT32_MAX, (int64_t)1 << 31, (int64_t)1 << 32, (int64_t)1 << 40})
      if (pos >= (int64_t)width * page && paged_page_of(s, 0, pos) != -1) return 1;
  }
  const PagedSeqs none = make_paged(nullptr, nullptr, nullptr, 1, 1, 0, 16, 0, 0);  // an empty table and cache
  if (paged_page_of(none, 0, 0) != -1) return 1;
  puts("ok");
}
"""


def test_pages_of_positions_on_the_host(tmp_path):
    from autokernel_amd import build
    src, exe = tmp_path / "pages.hip", tmp_path / "pages"
    src.write_text(PAGE_PROGRAM)
    flags = [f for f in build.HIP_FLAGS if f != "-O3"]
    subprocess.run([build.hipcc(), *flags, "-O1", f"-I{build.CSRC}", str(src), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_sample_refusals(lib):
    from autokernel_amd import _lib
    x = ctypes.c_void_p(4096)
    base = dict(dtype=1, x=x, u=x, out=x, rows=4, vocab=100, stride=100, tp=None, t=1.0, kp=None, k=0, pp=None, p=1.0,
                mp=None, m=0.0, stream=None)

    def call(**kw):
        return lib.ak_sample(*{**base, **kw}.values())
    nan = float("nan")
    for bad in (dict(dtype=7), dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(stride=99), dict(stride=-1), dict(x=None),
                dict(u=None), dict(out=None), dict(t=-1.0), dict(t=nan), dict(t=float("inf")), dict(p=nan), dict(m=nan),
                dict(rows=1 << 31), dict(rows=1 << 30)):
        assert call(**bad) == _lib.AK_EINVAL, bad
    assert call(vocab=(1 << 20) + 1, stride=1 << 21) == _lib.AK_EUNSUPPORTED
    assert call(rows=0) == _lib.AK_OK
