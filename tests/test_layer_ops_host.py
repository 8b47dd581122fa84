"""Host side of the operators around the expert block, on the CPU: refusals before
any device work, the paged cache's index arithmetic for every entry a device array
can hold, the rotary frequencies."""
import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from moe_stream_amd import _lib, ops
from oracle import layer as O

ROOT = Path(__file__).resolve().parent.parent
FAKE = 0x30_0000_0000   # an aligned address that no refused call touches


def _refused(rc, text, code=_lib.MOE_ERR_INVALID):
    assert rc == code, rc
    assert text in _lib.lib().moe_last_error().decode(), _lib.lib().moe_last_error()


def test_norm_refusals():
    f = _lib.lib().moe_add_rms_norm

    def call(x=FAKE, xs=64, r=FAKE, rs=64, w=FAKE, dt=0, T=2, D=64, eps=1e-6, y=FAKE, q=None,
             s=None, h=FAKE):
        return f(x, xs, r, rs, w, dt, T, D, eps, y, q, s, h, None)

    _refused(call(dt=2), "dtype")
    _refused(call(T=-1), "T=-1")
    _refused(call(D=0), "width=0")
    _refused(call(D=16385, xs=20000, rs=20000), "width=16385")
    _refused(call(eps=-1.0), "eps")
    _refused(call(eps=float("nan")), "eps")
    _refused(call(y=None), "give y, or q")
    _refused(call(q=FAKE, s=FAKE), "give y, or q")
    _refused(call(y=None, q=FAKE), "give y, or q")
    _refused(call(s=FAKE), "give y, or q")
    _refused(call(r=None), "without residual")
    _refused(call(x=None), "NULL")
    _refused(call(w=None), "NULL")
    _refused(call(xs=63), "strides")
    _refused(call(rs=63), "strides")
    assert call(T=0) == _lib.MOE_OK


def test_linear_refusals():
    L = _lib.lib()

    def call(x=FAKE, xd=2, st=256, xs=FAKE, w=FAKE, ws=FAKE, b=None, T=3, K=256, N=128, od=0,
             y=FAKE, work=FAKE, n=1 << 30):
        return L.moe_linear_fp8(x, xd, st, xs, w, ws, b, T, K, N, od, y, work, n, None)

    _refused(call(xd=3), "x dtype")
    _refused(call(od=2), "output dtype")
    _refused(call(T=-1), "T=-1")
    _refused(call(K=250), "K=250")
    _refused(call(K=0), "K=0")
    _refused(call(N=0), "N=0")
    _refused(call(xs=None), "x_scales")
    _refused(call(xd=0), "x_scales")
    _refused(call(w=None), "NULL")
    _refused(call(st=240), "stride")
    _refused(call(w=FAKE + 8), "aligned")
    _refused(call(x=FAKE + 8), "aligned")
    _refused(call(st=264), "aligned")
    # a tile's rows lie within 32-bit offsets, a product in one launch
    _refused(call(st=(1 << 23) + 16), "2^23")
    _refused(call(T=(1 << 24) - 1, K=16, N=1 << 22), "one launch")
    # 16-bit rows beyond the few that are quantised on the way need room for their codes
    _refused(call(xd=0, xs=None, T=50, work=None), "workspace")
    _refused(call(xd=0, xs=None, T=50, work=FAKE + 16), "workspace")
    _refused(call(xd=0, xs=None, T=50, n=100), "workspace 100")
    assert call(T=0) == _lib.MOE_OK
    assert L.moe_linear_fp8_workspace(0, 256, 128, 0) == 0
    assert L.moe_linear_fp8_workspace(50, 256, 128, 0) >= 50 * 256 + 50 * 2 * 4


def _view(**kw):
    v = _lib.KvView(FAKE, FAKE, FAKE, FAKE, FAKE, 100, 2, 16, 64, 0, 4, 8)
    for k, x in kw.items():
        setattr(v, k, x)
    return v


BAD_VIEWS = [(dict(k=None), "NULL"), (dict(lens=None), "NULL"), (dict(dtype=2), "dtype"),
             (dict(n_pages=0), "positive"), (dict(kv_heads=-1), "positive"),
             (dict(n_seqs=0), "positive"), (dict(table_width=0), "positive"),
             (dict(page_size=8), "page_size=8"), (dict(page_size=48), "page_size=48"),
             (dict(page_size=512), "page_size=512"), (dict(head_dim=63), "head_dim=63"),
             (dict(head_dim=514), "head_dim=514"),
             (dict(table_width=1 << 23, page_size=256), "2^30")]


@pytest.mark.parametrize("bad,text", BAD_VIEWS)
def test_kv_view_refusals(bad, text):
    L, v = _lib.lib(), _view(**bad)
    _refused(_rope(v), text)
    _refused(_attn(v), text)
    assert L.moe_attn_paged_workspace(C.byref(v), 3, 8, 0) == 0


def _rope(v, q=FAKE, T=3, H=8, f=FAKE, rot=64, eps=1e-6, out=FAKE):
    return _lib.lib().moe_rope_cache(C.byref(v), q, 512, 64, FAKE, 128, 64, FAKE, 128, 64, T, H, f,
                                     rot, 0, 1.0, None, None, eps, out, None)


def _attn(v, q=FAKE, qt=512, qh=64, T=3, H=8, window=0, out=FAKE, work=FAKE, n=1 << 40,
          scale=0.125):
    return _lib.lib().moe_attn_paged(C.byref(v), q, qt, qh, T, H, scale, window, None, out, work,
                                     n, None)


def test_rope_refusals():
    v = _view()
    _refused(_lib.lib().moe_rope_cache(None, *([FAKE, 1, 1] * 3), 1, 1, FAKE, 64, 0, 1.0, None, None,
                                       0.0, FAKE, None), "view is NULL")
    _refused(_rope(v, T=-1), "T=-1")
    _refused(_rope(v, H=0), "heads=0")
    _refused(_rope(v, rot=66), "rot=66")
    _refused(_rope(v, rot=3), "rot=3")
    _refused(_rope(v, eps=-1.0), "eps")
    _refused(_rope(v, q=None), "NULL")
    _refused(_rope(v, f=None), "NULL")
    _refused(_rope(v, out=None), "NULL")
    assert _rope(v, T=0) == _lib.MOE_OK


def test_attn_refusals():
    v = _view()
    _refused(_attn(v, T=(1 << 24) + 1), "T=16777217")
    _refused(_attn(v, H=7), "heads=7")
    _refused(_attn(v, H=0), "heads=0")
    _refused(_attn(v, H=130), "65 heads", _lib.MOE_ERR_UNSUPPORTED)
    _refused(_attn(_view(head_dim=80)), "head_dim=80", _lib.MOE_ERR_UNSUPPORTED)
    _refused(_attn(v, window=-1), "window=-1")
    for scale in (-0.125, float("nan"), float("inf")):
        _refused(_attn(v, scale=scale), "scale")
    _refused(_attn(v, q=None), "NULL")
    _refused(_attn(v, out=None), "NULL")
    _refused(_attn(v, q=FAKE + 8), "aligned")
    _refused(_attn(v, qt=516), "aligned")
    _refused(_attn(v, qh=65), "aligned")
    _refused(_attn(_view(k=FAKE + 2)), "aligned")
    _refused(_attn(v, out=FAKE + 4), "aligned")
    need = _lib.lib().moe_attn_paged_workspace(C.byref(v), 3, 8, 0)
    if need:
        _refused(_attn(v, work=None), "workspace")
        _refused(_attn(v, n=need - 1), "workspace")
    assert _attn(v, T=0) == _lib.MOE_OK


def test_operators_refuse_host_tensors_and_wrong_types():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="device"):
        ops.add_rms_norm(x, w)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.add_rms_norm(x.float(), w)
    f8 = x.to(torch.float8_e4m3fn)
    with pytest.raises(TypeError, match="device"):
        ops.linear_fp8(f8, f8, torch.zeros(1, 1), x_scales=torch.zeros(2, 1))
    with pytest.raises(TypeError, match="device"):
        ops.linear_fp8(x, f8, torch.zeros(1, 1))
    q = torch.zeros(2, 4, 64, dtype=torch.float32)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.attn_paged(q, q, q, q, q, q)
    with pytest.raises(TypeError, match="device"):
        ops.rope_cache(q.half(), q, q, q, q, q, q, q, q)


CHECK = r"""
#include "paged.h"
#include <cstdio>
#include <cstdlib>
#include <climits>
#include <initializer_list>
using namespace moe;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); std::exit(1); } } while (0)
int main() {
  const int v[] = {INT_MIN, INT_MIN + 1, -1000, -1, 0, 1, 5, 15, 16, 17, 100, 1000, INT_MAX - 1, INT_MAX};
  const int caps[] = {16, 64, 4096, INT_MAX - 15};
  for (int a : v) for (int b : v) for (int n : v) for (int total : {1, 16, 100, 1 << 24}) for (int cap : caps) {
    const SeqSpan s = seq_span(a, b, n, total, cap);
    CHECK(s.first >= 0 && s.rows >= 0 && s.first <= total && s.rows <= total - s.first);
    CHECK(s.len >= 0 && s.len <= cap && s.base == s.len - s.rows);
    const bool in = a >= 0 && a <= b && b <= total && n >= 0 && n <= cap && n >= b - a;
    CHECK(s.ok == in);
    if (in) CHECK(s.first == a && s.rows == b - a && s.len == n);
    for (int w : {0, 1, 7, 128, INT_MAX}) for (int pos : {s.base, s.base + s.rows / 2, s.base + s.rows - 1}) {
      int lo, hi;
      seen_keys(pos, s.len, w, &lo, &hi);
      CHECK(lo >= 0 && hi >= 0 && hi <= s.len);
      if (pos < 0) CHECK(lo >= hi);
      if (pos >= 0 && pos < s.len) {
        CHECK(hi == pos + 1);
        CHECK(hi - lo == (w > 0 && w < hi ? w : hi));
      }
    }
  }
  for (int pages : {1, 3, 1 << 20}) for (int e : v) for (int heads : {1, 8}) for (int sh = 4; sh <= 8; ++sh)
    for (int pos : {0, 1, 15, 16, 255, 100000}) for (int h = 0; h < heads; ++h) {
      const long long at = page_row(e, pages, heads, h, sh, pos, 128);
      if (e < 0 || e >= pages) { CHECK(at == -1); continue; }
      const long long want = (((long long)e * heads + h) * (1 << sh) + pos % (1 << sh)) * 128;
      CHECK(at == want);
      CHECK(at >= 0 && at + 128 <= (long long)pages * heads * (1 << sh) * 128);
    }
  std::puts("ok");
}
"""


def test_paged_index_arithmetic(tmp_path):
    """Every entry that a batch's device arrays can hold maps inside the batch, the
    table and the pages, or is refused."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    src = tmp_path / "check.cpp"
    src.write_text(CHECK)
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(ROOT / "moe_stream_amd" / "csrc"), str(src), "-o", str(exe)],
                   check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout.strip() == "ok"


def test_rope_freqs():
    f, m = ops.rope_freqs(128, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    want = [10000.0 ** (-2 * i / 128) for i in range(64)]
    np.testing.assert_allclose(f.numpy(), want, rtol=1e-14)
    f2, m = ops.rope_freqs(128, 10000.0, 8.0, "linear", device="cpu")
    np.testing.assert_allclose(f2.numpy(), np.array(want) / 8, rtol=1e-14)
    # yarn, the gpt-oss setting: a pair's turns within the original length decide
    f3, m = ops.rope_freqs(64, 150000.0, 32.0, "yarn", original=4096, device="cpu")
    assert m == pytest.approx(0.1 * math.log(32) + 1, rel=1e-14)
    base = np.array([150000.0 ** (-2 * i / 64) for i in range(32)])
    turns = 4096 * base / (2 * math.pi)
    ratio = f3.numpy() / base
    assert np.allclose(ratio[turns > 32 * 1.5], 1.0) and np.allclose(ratio[turns < 0.6], 1 / 32)
    assert (np.diff(ratio) <= 1e-15).all()
    lo, hi = 8, 18   # floor and ceil of 32 ln(4096 / (32, 1) / 2 pi) / ln 150000
    assert math.floor(32 * math.log(4096 / 32 / 2 / math.pi) / math.log(150000)) == lo
    assert math.ceil(32 * math.log(4096 / 2 / math.pi) / math.log(150000)) == hi
    for i in range(32):
        r = min(max((i - lo) / (hi - lo), 0), 1)
        assert ratio[i] == pytest.approx((1 - r) + r / 32, rel=1e-13)
    f4, m = ops.rope_freqs(128, 500000.0, 8.0, "llama3", original=8192, device="cpu")
    base = np.array([500000.0 ** (-2 * i / 128) for i in range(64)])
    for i in range(64):
        wl = 2 * math.pi / base[i]
        if wl < 8192 / 4:
            want = base[i]
        elif wl > 8192 / 1:
            want = base[i] / 8
        else:
            k = (8192 / wl - 1) / (4 - 1)
            want = (1 - k) * base[i] / 8 + k * base[i]
        assert float(f4[i]) == pytest.approx(want, rel=1e-12)
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, base=1.0), dict(rot=8, factor=0.5),
                dict(rot=8, kind="other"), dict(rot=8, kind="llama3", low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            ops.rope_freqs(device="cpu", **bad)


def test_oracle_codes():
    """The oracle's e4m3 rounding against torch's conversion, on every code, halfway
    between neighbours and beside it."""
    codes = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert (O.e4m3(codes) == codes).all() and codes[-1] == 448
    mid = (codes[1:] + codes[:-1]) / 2
    for x in (mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9), -mid):
        x32 = x.astype(np.float32)
        want = torch.tensor(x32).to(torch.float8_e4m3fn).double().numpy()
        assert (O.e4m3(x32.astype(np.float64)) == want).all()
