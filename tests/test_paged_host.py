"""The operators over many sessions without a GPU: what their calls refuse
(arguments are checked before the context is used), the frequencies that
c2h_rope_init fills, and the index arithmetic of the kernels compiled as
plain C++."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from c2slm_amd import _lib as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -3
A = 0x10000  # an aligned address; nothing here reads or writes it


def kv(**over):
    d = dict(k=A, v=2 * A, type=H.BF16, n_pages=100, page_size=16, n_kv_heads=2, head_dim=64, reserved=0,
             page_stride=16 * 128, token_stride=128, head_stride=64, k_scale=None, v_scale=None)
    d.update(over)
    return H.PagedKV(*[d[n] for n, _ in H.PagedKV._fields_])


def batch(**over):
    d = dict(block_table=A, table_stride=8, seq_lens=A, n_seqs=3, max_len=128)
    d.update(over)
    return H.PagedBatch(*[d[n] for n, _ in H.PagedBatch._fields_])


def heads(data=A, token_stride=1024, head_stride=64):
    return H.Heads(data, token_stride, head_stride)


def refused(rc, code, word):
    assert rc == code, (rc, H.lib().c2h_last_error(None))
    assert word in H.lib().c2h_last_error(None).decode()


BAD_CACHE = [
    (dict(type=12), UNSUPPORTED, "type"), (dict(page_size=4), UNSUPPORTED, "page_size"),
    (dict(page_size=24), UNSUPPORTED, "page_size"), (dict(page_size=2048), UNSUPPORTED, "page_size"),
    (dict(head_dim=72), UNSUPPORTED, "head_dim"), (dict(head_dim=272), UNSUPPORTED, "head_dim"),
    (dict(head_dim=0), UNSUPPORTED, "head_dim"), (dict(n_pages=0), INVALID, "pages"),
    (dict(n_kv_heads=0), INVALID, "KV heads"), (dict(k=None), INVALID, "memory"), (dict(v=None), INVALID, "memory"),
    (dict(v=A), INVALID, "memory of their own"), (dict(k=A + 8), INVALID, "16 bytes"),
    (dict(token_stride=132), INVALID, "16 bytes"), (dict(token_stride=-128), INVALID, "strides"),
    (dict(head_stride=32), INVALID, "overlap"), (dict(token_stride=64), INVALID, "overlap"),
    (dict(page_stride=15 * 128), INVALID, "overlap"), (dict(page_stride=0), INVALID, "overlap"),
    (dict(page_stride=1 << 50), INVALID, "strides"),
]
BAD_BATCH = [
    (dict(n_seqs=-1), "sessions"), (dict(max_len=-1), "max_len"), (dict(max_len=(1 << 23) + 1, table_stride=1 << 30), "max_len"),
    (dict(block_table=None), "table"), (dict(seq_lens=None), "lengths"), (dict(max_len=129), "does not cover"),
    (dict(table_stride=-1), "does not cover"),
]


@pytest.mark.parametrize("over,code,word", BAD_CACHE, ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_cache_descriptions_refused(over, code, word):
    L, n, q = H.lib(), C.c_size_t(7), heads()
    refused(L.c2h_paged_attn_workspace(kv(**over), batch(), 4, 0, C.byref(n)), code, word)
    assert n.value == 0
    refused(L.c2h_paged_attn_dev(None, kv(**over), batch(), H.F32, 4, 0.125, 0, q, q), code, word)
    refused(L.c2h_paged_append_dev(None, kv(**over), batch(), None, 3, None, H.F32, q, q, 0, None, None), code, word)


@pytest.mark.parametrize("over,word", BAD_BATCH, ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_batch_descriptions_refused(over, word):
    L, n, q = H.lib(), C.c_size_t(7), heads()
    refused(L.c2h_paged_attn_workspace(kv(), batch(**over), 4, 0, C.byref(n)), INVALID, word)
    refused(L.c2h_paged_attn_dev(None, kv(), batch(**over), H.F32, 4, 0.125, 0, q, q), INVALID, word)
    refused(L.c2h_paged_append_dev(None, kv(), batch(**over), None, 3, None, H.F32, q, q, 0, None, None), INVALID, word)


def test_attention_arguments_refused():
    L, q = H.lib(), heads()

    def call(kv_=None, type=H.F32, n_heads=4, scale=0.125, window=0, q=q, out=q):
        return L.c2h_paged_attn_dev(None, kv_ or kv(), batch(), type, n_heads, scale, window, q, out)

    refused(call(type=H.F8_E4M3), UNSUPPORTED, "type")
    refused(call(type=12), UNSUPPORTED, "type")
    refused(call(n_heads=3), INVALID, "query heads")
    refused(call(n_heads=0), INVALID, "query heads")
    refused(call(window=-1), INVALID, "window")
    refused(call(scale=float("nan")), INVALID, "scale")
    refused(call(scale=float("inf")), INVALID, "scale")
    refused(call(q=None), INVALID, "q: no data")
    refused(call(q=heads(data=None)), INVALID, "q: no data")
    refused(call(out=heads(data=A + 4)), INVALID, "out: data and strides")
    refused(call(q=heads(token_stride=1026)), INVALID, "q: data and strides")
    refused(call(q=heads(head_stride=-64)), INVALID, "q: strides")
    refused(call(out=heads(token_stride=0)), INVALID, "out: vectors overlap")
    refused(call(out=heads(head_stride=32)), INVALID, "out: vectors overlap")
    refused(call(out=heads(token_stride=192)), INVALID, "out: vectors overlap")
    refused(call(q=heads(token_stride=0)), INVALID, "no context")  # one query for all sessions is fine


def test_append_and_rope_arguments_refused():
    L, x, r = H.lib(), heads(), H.rope(64, 1e6)

    def app(n=3, start=None, rope=None, type=H.F32, k=x, v=x, n_heads=0, q=None, q_out=None):
        return L.c2h_paged_append_dev(None, kv(), batch(), start, n, rope, type, k, v, n_heads, q, q_out)

    refused(app(n=4), INVALID, "4 tokens for 3 sessions")
    refused(app(n=-1, start=A), INVALID, "tokens")
    refused(app(type=H.F8_E4M3), UNSUPPORTED, "type")
    refused(app(rope=H.Rope()), INVALID, "did not fill")
    refused(app(rope=H.rope(128, 1e6)), INVALID, "rot_dim 128 exceeds head_dim 64")
    refused(app(k=None), INVALID, "k: no data")
    refused(app(v=heads(data=A + 2)), INVALID, "v: data")
    refused(app(q=x, n_heads=4), INVALID, "q_out: no data")
    refused(app(q_out=x, n_heads=4), INVALID, "q: no data")
    refused(app(q=x, q_out=x), INVALID, "query heads")
    refused(app(q=x, q_out=heads(token_stride=128), n_heads=4), INVALID, "q_out: vectors overlap")
    refused(app(rope=r, q=x, q_out=x, n_heads=4), INVALID, "no context")
    refused(app(n=9, start=A), INVALID, "no context")

    def rope(rope=r, type=H.F32, x=x, pos=A, n=3, n_heads=4, hd=64, y=x):
        return L.c2h_rope_dev(None, rope, type, x, pos, n, n_heads, hd, y)

    refused(rope(rope=None), INVALID, "no rotation")
    refused(rope(pos=None), INVALID, "positions")
    refused(rope(type=H.F8_E4M3), UNSUPPORTED, "type")
    refused(rope(n=-1), INVALID, "tokens")
    refused(rope(n_heads=0), INVALID, "heads")
    refused(rope(hd=60), UNSUPPORTED, "head_dim")
    refused(rope(hd=264), UNSUPPORTED, "head_dim")
    refused(rope(hd=56), INVALID, "exceeds")
    refused(rope(y=heads(head_stride=32)), INVALID, "y: vectors overlap")
    refused(rope(x=None), INVALID, "x: no data")
    refused(rope(), INVALID, "no context")


def test_more_than_a_launch_refused():
    """Work-items of a launch are counted in 32 bits."""
    L, r, row = H.lib(), H.rope(64, 1e6), heads(token_stride=1024, head_stride=64)
    # one row of all sessions' queries; outputs of 2^18 elements a session
    q, out = heads(token_stride=0), heads(token_stride=1 << 18)

    def rope(n):
        return L.c2h_rope_dev(None, r, H.F32, row, A, n, 4, 64, row)

    def app(n):
        return L.c2h_paged_append_dev(None, kv(), batch(), A, n, None, H.F32, row, row, 0, None, None)

    def attn(n_seqs, n_heads):
        return L.c2h_paged_attn_dev(None, kv(), batch(n_seqs=n_seqs), H.F32, n_heads, 0.1, 0, q, out)

    def norm(n):
        return L.c2h_rmsnorm_q8k_dev(None, H.F32, A, 256, None, 0, A, 1e-6, n, 256, None, 0, A, None, 0)

    for call, most in ((rope, 2 ** 24 - 1), (app, 2 ** 24 - 1), (norm, 2 ** 22 - 1)):
        refused(call(most), INVALID, "no context")
        for n in (most + 1, 2 ** 31 - 1):
            refused(call(n), UNSUPPORTED, "up to %d" % most)
    refused(attn(65535, 256), INVALID, "no context")
    refused(attn(65535, 258), UNSUPPORTED, "65535 sessions of 258 heads")
    refused(attn(4096, 4096), UNSUPPORTED, "4096 sessions of 4096 heads")
    n = C.c_size_t(7)
    refused(L.c2h_paged_attn_workspace(kv(), batch(n_seqs=65535), 4096, 0, C.byref(n)), UNSUPPORTED, "sessions")
    assert n.value == 0


def test_norm_arguments_refused():
    L = H.lib()

    def norm(type=H.F32, x=A, xs=1024, r=None, rs=0, w=A, eps=1e-6, n=2, cols=896, s=None, ss=0, q=A, y=None, ys=0):
        return L.c2h_rmsnorm_q8k_dev(None, type, x, xs, r, rs, w, eps, n, cols, s, ss, q, y, ys)

    refused(norm(type=H.F8_E4M3), UNSUPPORTED, "type")
    for cols in (255, 0, -256, 16385):
        refused(norm(cols=cols), UNSUPPORTED, "columns")
    refused(norm(n=-1), INVALID, "rows")
    refused(norm(x=None), INVALID, "required")
    refused(norm(w=None), INVALID, "required")
    refused(norm(q=None), INVALID, "required")
    refused(norm(r=A, rs=1024), INVALID, "come together")
    refused(norm(s=A, ss=1024), INVALID, "come together")
    refused(norm(eps=-1.0), INVALID, "eps")
    refused(norm(eps=float("nan")), INVALID, "eps")
    refused(norm(x=A + 2), INVALID, "whole elements")
    refused(norm(type=H.BF16, x=A + 1), INVALID, "whole elements")
    refused(norm(y=A + 2, ys=1024), INVALID, "whole elements")
    refused(norm(q=A + 2), INVALID, "q8k_out must be")
    refused(norm(w=A + 1), INVALID, "4 bytes")
    refused(norm(type=H.BF16, x=A + 2, xs=897, cols=897), INVALID, "no context")
    refused(norm(y=A, ys=512), INVALID, "row stride")
    refused(norm(r=A, rs=1024, s=A, ss=0), INVALID, "row stride")
    refused(norm(xs=-1024), INVALID, "row stride")
    refused(norm(), INVALID, "no context")


def test_workspace_follows_the_split():
    # sessions that one step of a workgroup holds need none; longer ones meet
    # in head_dim + 2 floats per query head and chunk, and two integers each
    one = batch(n_seqs=1, max_len=8192, table_stride=512)
    assert H.paged_attn_workspace(kv(), batch(n_seqs=512, max_len=100), 14) == 0
    got = H.paged_attn_workspace(kv(), one, 14) - 8
    assert got > 0 and got % (14 * (64 + 2) * 4) == 0
    # a window bounds it
    assert H.paged_attn_workspace(kv(), one, 14, window=100) == 0
    assert H.paged_attn_workspace(kv(), batch(n_seqs=0), 14) == 0


@pytest.mark.parametrize("over,code,word", [
    (dict(rot_dim=4), UNSUPPORTED, "rot_dim"), (dict(rot_dim=60), UNSUPPORTED, "rot_dim"),
    (dict(rot_dim=264), UNSUPPORTED, "rot_dim"), (dict(base=1.0), INVALID, "base"), (dict(base=float("inf")), INVALID, "base"),
    (dict(base=float("nan")), INVALID, "base"), (dict(factor=0.5), INVALID, "factor"),
    (dict(factor=float("nan")), INVALID, "factor"), (dict(mscale=float("inf")), INVALID, "mscale"),
    (dict(orig_ctx=-1), INVALID, "orig_ctx"), (dict(factor=4.0, orig_ctx=4096, beta_fast=0.0), INVALID, "beta"),
    (dict(freq_factors=np.zeros(32)), INVALID, "freq_factors"),
], ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_rope_descriptions_refused(over, code, word):
    args = dict(rot_dim=64, base=1e6)
    args.update(over)
    with pytest.raises(H.C2hError) as e:
        H.rope(**args)
    assert e.value.code == code and word in str(e.value)


def test_rope_frequencies():
    n = np.arange(32)
    f = 1e6 ** (-n / 32.0)
    got = lambda r: np.array(r.turns[:r.rot_dim // 2]) * 2 * math.pi  # noqa: E731
    # a few roundings of 64 bits each
    np.testing.assert_allclose(got(H.rope(64, 1e6)), f, rtol=2e-15)
    np.testing.assert_allclose(got(H.rope(64, 1e6, factor=4.0)), f / 4, rtol=2e-15)
    c = np.linspace(1, 8, 32).astype(np.float32)
    np.testing.assert_allclose(got(H.rope(64, 1e6, freq_factors=c)), f / c.astype(np.float64), rtol=2e-15)
    # YaRN: pairs that turn often keep their frequency, slow ones are divided
    corner = lambda t: 64 * math.log(4096 / (2 * math.pi * t)) / (2 * math.log(1e6))  # noqa: E731
    lo, hi = math.floor(corner(32.0)), math.ceil(corner(1.0))
    assert 0 < lo < hi < 32
    r = np.clip((n - lo) / (hi - lo), 0, 1)
    y = got(H.rope(64, 1e6, factor=8.0, orig_ctx=4096))
    np.testing.assert_allclose(y, f * (1 - r) + f / 8 * r, rtol=4e-15)
    assert np.allclose(y[:lo + 1], f[:lo + 1], rtol=2e-15) and np.allclose(y[hi:], f[hi:] / 8, rtol=2e-15)
    r = H.rope(8, 1e4, layout="interleaved", mscale=1.25)
    assert r.layout == 1 and r.rot_dim == 8 and r.mscale == 1.25 and r.turns[0] * 2 * math.pi == 1.0
    assert not any(r.turns[4:])


HARNESS = r"""
#include <cassert>
#include <climits>
#include <cstdio>
#include <initializer_list>
#include "c2h_paged.h"
using namespace c2h;
int main() {
  // pages: an index is used only inside the pool
  assert(page_ok(0, 1) && page_ok(99, 100) && !page_ok(100, 100) && !page_ok(-1, 100) && !page_ok(INT_MIN, 100) &&
         !page_ok(INT_MAX, 100));
  assert(length_ok(0, 0) && length_ok(5, 5) && !length_ok(6, 5) && !length_ok(-1, 5) && !length_ok(INT_MIN, 1 << 30));
  // windows and chunks cover the span once, in order, without overflow, and
  // a wave holds the pages of its steps
  const int lens[] = {0, 1, 2, 127, 128, 129, 4095, 4096, 100001, PAGED_MAX_LEN};
  const int wins[] = {0, 1, 127, 128, 1000, 1 << 30};
  for (int len : lens)
    for (int w : wins)
      for (int unit : {64, 128, 256})
        for (int cu : {1, 2, 3, 7, 30, 1000}) {
          const int chunk = cu * unit, step = unit / 4;
          const Span s = attended(len, w);
          assert(s.hi == len && s.lo >= 0 && s.hi - s.lo == (w > 0 && w < len ? w : len));
          const int units = units_of(s, unit), n = chunks_of(units, cu);
          const int longest = w > 0 && w < PAGED_MAX_LEN ? w + SPAN_ALIGN - 1 : PAGED_MAX_LEN;
          assert(n >= 1 && (units == 0) == (len == 0) && units <= units_of(Span{0, longest}, unit));
          int64_t at = s.lo;
          for (int i = 0; len > 0 && i < n; i = i == 2 && n > 6 ? n - 3 : i + 1) {  // the first and last three
            const int64_t b = chunk_base(s, chunk, i), c0 = b > s.lo ? b : s.lo, c1 = b + chunk < s.hi ? b + chunk : s.hi;
            assert(b % SPAN_ALIGN == 0 && c1 > c0 && c1 - c0 <= chunk && (i < 3 ? c0 == at : c0 > s.lo));
            at = c1;
            for (int sh = 3; sh <= 10; ++sh)
              for (int wave = 0; wave < 4; ++wave) {
                int p0 = (int)c0 >> sh, first = (int)b + wave * step, beyond = first_step_beyond(p0, sh, first, step, unit);
                int turns = 0;
                for (int base = first; base < c1 && turns < 5; base += unit) {
                  if (base == beyond) {
                    p0 = base >> sh;
                    beyond = first_step_beyond(p0, sh, base, step, unit);
                    ++turns;
                  }
                  assert(base < beyond && (beyond - first) % unit == 0);
                  for (int pos : {base, base + step - 1}) {
                    const int p = pos < c0 ? (int)c0 : pos < c1 ? pos : (int)c1 - 1;
                    assert((p >> sh) - p0 >= 0 && (p >> sh) - p0 < 64);
                  }
                }
              }
          }
          assert(at == s.hi);
        }
  // the bound of a batch's chunks holds for even and uneven batches
  for (int n_seqs : {1, 2, 63, 64, 65, 700})
    for (int rows : {1, 2, 8, 600})
      for (int shape = 0; shape < 4; ++shape) {
        int64_t units = 0, chunks = 0;
        auto u = [&](int i) { return shape == 0 ? 0 : shape == 1 ? 50 : shape == 2 ? (i * 7919) % 51 : i ? 1 : 50; };
        for (int i = 0; i < n_seqs; ++i) units += u(i);
        const int cu = chunk_units(units, rows);
        for (int i = 0; i < n_seqs; ++i) chunks += chunks_of(u(i), cu);
        assert(cu >= 1 && chunks <= chunks_bound(n_seqs, rows, 50));
      }
  // the tokens of a session are its last ones
  assert(token_pos(10, 5, 6) == 9 && token_pos(10, 0, 6) == 4 && token_pos(3, 0, 6) == -3 && token_pos(0, 0, 1) == -1);
  assert(token_pos(1 << 30, INT_MAX - 1, INT_MAX) == (1 << 30) - 1);
  puts("ok");
}
"""


def test_index_arithmetic(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "c2slm_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stderr


def test_python_views_refused():
    class T:
        def __init__(self, shape, stride):
            self.shape, self._s, self.ndim = shape, stride, len(shape)

        def stride(self, i=None):
            return self._s if i is None else self._s[i]

        def data_ptr(self):
            return A

    with pytest.raises(ValueError):
        H.heads(T((2, 3, 64), (384, 128, 2)))
    with pytest.raises(ValueError):
        H.heads(T((2, 64), (64, 1)))
    with pytest.raises(ValueError):
        H.paged_kv(T((4, 16, 2, 64), (2048, 128, 64, 1)), T((4, 16, 2, 64), (4096, 128, 64, 1)), H.BF16)
    with pytest.raises(ValueError):
        H.paged_batch(T((3, 4), (4, 1)), T((2,), (1,)), 64)
    with pytest.raises(ValueError):
        H.rope(64, 1e6, freq_factors=np.ones(31))
    p = H.paged_kv(T((4, 2, 16, 64), (2048, 1024, 64, 1)), T((4, 2, 16, 64), (2048, 1024, 64, 1)), H.BF16, order="hnd")
    assert (p.page_size, p.n_kv_heads, p.token_stride, p.head_stride) == (16, 2, 64, 1024)


def test_python_tensors_of_other_shapes_and_types_refused():
    """What Python's calls take by address they check first: 64-bit indexes
    (torch's default) or a column of a tensor would be read as other numbers,
    rows of another shape beyond their end."""
    torch = pytest.importorskip("torch")
    ctx = object.__new__(H.Ctx)
    ctx.h = None
    lens, table = torch.ones(2, dtype=torch.int32), torch.ones(2, 4, dtype=torch.int32)
    assert H.paged_batch(table, lens, 64).n_seqs == 2
    for t, n in ((table.long(), lens), (table, lens.long()), (table, table[:, 0])):
        with pytest.raises(ValueError):
            H.paged_batch(t, n, 64)
    pool = torch.ones(4, 16, 2, 64, dtype=torch.uint8)
    assert H.paged_kv(pool, pool, H.F8_E4M3, k_scale=torch.ones(2)).k_scale
    for bad in (torch.ones(2, dtype=torch.bfloat16), torch.ones(1), torch.ones(16), torch.ones(2, 2)[:, 0]):
        with pytest.raises(ValueError):
            H.paged_kv(pool, pool, H.F8_E4M3, k_scale=bad)
        with pytest.raises(ValueError):
            H.paged_kv(pool, pool, H.F8_E4M3, v_scale=bad)
    rope, x = H.rope(64, 1e6), heads()
    kv_, batch_ = kv(), batch()
    for bad in (torch.arange(3), torch.ones(3, 2, dtype=torch.int32)[:, 0]):
        with pytest.raises(ValueError):
            ctx.rope_dev(rope, H.F32, x, bad, 3, 4, 64, x)
        with pytest.raises(ValueError):
            ctx.paged_append_dev(kv_, batch_, H.F32, 3, x, x, token_start=bad)
    r, w, q8k = torch.ones(3, 512), torch.ones(512), torch.ones(3, 2, 292, dtype=torch.uint8)

    def norm(x=r, w=w, q8k=q8k, **more):
        with pytest.raises(ValueError):
            ctx.rmsnorm_q8k_dev(H.F32, x, w, 1e-6, q8k, **more)

    norm(x=torch.ones(512, 3).T)
    norm(w=w[:256])
    norm(w=torch.ones(1024)[::2])
    norm(q8k=q8k[:2])
    norm(q8k=torch.ones(3, 2, 584, dtype=torch.uint8)[:, :, :292])
    for bad in (r[:2], r[:, :256], torch.ones(512, 3).T, torch.ones(3, 1024)[:, ::2]):
        norm(residual=bad, sum_out=r)
        norm(residual=r, sum_out=bad)
        norm(y=bad)


def host_ctx():
    """A context that no call reaches: every call here is refused before.  The
    tensors' device, the CPU's -1, stands for the context's GPU."""
    ctx = object.__new__(H.Ctx)
    ctx.h, ctx.device = None, -1
    return ctx


def test_norm_tensors_of_other_element_types_refused():
    """A weight, row or output of fewer bytes an element than the kernel takes
    would be read or written beyond its end."""
    torch = pytest.importorskip("torch")
    ctx, q8k = host_ctx(), torch.ones(3, 2, 292, dtype=torch.uint8)
    types = {H.F32: torch.float32, H.F16: torch.float16, H.BF16: torch.bfloat16}
    H.lib()
    for ty, own in types.items():
        good = dict(x=torch.ones(3, 512, dtype=own), w=torch.ones(512), residual=torch.ones(3, 512, dtype=own),
                    sum_out=torch.ones(3, 512, dtype=own), y=torch.ones(3, 512))
        for name in good:
            mine = torch.float32 if name in ("w", "y") else own
            for other in (torch.float32, torch.float16, torch.bfloat16, torch.float64, torch.int32):
                if other != mine:
                    with pytest.raises(ValueError):
                        ctx.rmsnorm_q8k_dev(ty, eps=1e-6, q8k=q8k, **dict(good, **{name: good[name].to(other)}))
    with pytest.raises(ValueError):
        ctx.rmsnorm_q8k_dev(H.F8_E4M3, torch.ones(3, 512), torch.ones(512), 1e-6, q8k)


def test_fewer_indexes_than_the_call_reads_refused():
    """Positions one per token, starts one more than sessions, integers of 32
    bits: floats would be read as their bit patterns, and with the last start
    missing the last session's tokens would go to another one's slots."""
    torch = pytest.importorskip("torch")
    ctx, rope, x = host_ctx(), H.rope(64, 1e6), heads()
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    for bad in (i32(1), i32(0), torch.zeros(3), i32(3).view(torch.float32), torch.zeros(6, dtype=torch.int16)):
        with pytest.raises(ValueError):
            ctx.rope_dev(rope, H.F32, x, bad, 3, 4, 64, x)
    for bad in (i32(3), i32(1), torch.zeros(4), torch.zeros(8, dtype=torch.int16)):
        with pytest.raises(ValueError):
            ctx.paged_append_dev(kv(), batch(), H.F32, 3, x, x, token_start=bad)
    table, lens = torch.ones(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for t, n in ((table.float(), lens), (table, lens.float()), (table.view(torch.float32), lens)):
        with pytest.raises(ValueError):
            H.paged_batch(t, n, 64)
    # more than the call reads is fine; without a context the library refuses it
    for call in (lambda: ctx.rope_dev(rope, H.F32, x, i32(9), 3, 4, 64, x),
                 lambda: ctx.paged_append_dev(kv(), batch(), H.F32, 3, x, x, token_start=i32(9))):
        with pytest.raises(H.C2hError, match="no context"):
            call()


def test_pools_of_another_element_type_or_order_refused():
    """A 16-bit pool read as 32-bit ends halfway; an order that is not one of
    the two was taken for the second."""
    torch = pytest.importorskip("torch")
    H.lib()
    types = {H.F32: torch.float32, H.F16: torch.float16, H.BF16: torch.bfloat16, H.F8_E4M3: torch.float8_e4m3fn}
    pools = [torch.zeros(4, 16, 2, 64, dtype=torch.uint8).to(t) for t in types.values()]
    pools += [torch.zeros(4, 16, 2, 64).to(t) for t in (torch.float64, torch.int32, torch.int16, torch.float8_e5m2,
                                                        torch.float8_e4m3fnuz)]
    for ty, own in types.items():
        good = torch.zeros(4, 16, 2, 64, dtype=own)
        assert H.paged_kv(good, good, ty).type == ty
        for other in pools:
            if other.dtype != own:
                for k, v in ((other, other), (good, other), (other, good)):
                    with pytest.raises(ValueError):
                        H.paged_kv(k, v, ty)
    for bits in (torch.uint8, torch.int8):
        pool = torch.zeros(4, 16, 2, 64, dtype=bits)
        assert H.paged_kv(pool, pool, H.F8_E4M3).type == H.F8_E4M3
    with pytest.raises(ValueError):
        H.paged_kv(good, good, 12)
    for order in ("NHD", "HND", "", "hdn", None):
        with pytest.raises(ValueError):
            H.paged_kv(good, good, H.F8_E4M3, order=order)
    for scale in (torch.ones(2, dtype=torch.int32), torch.ones(2, dtype=torch.float64), torch.ones(4, dtype=torch.float16)):
        with pytest.raises(ValueError):
            H.paged_kv(good, good, H.F8_E4M3, k_scale=scale)
        with pytest.raises(ValueError):
            H.paged_kv(good, good, H.F8_E4M3, v_scale=scale)


def test_tables_of_fewer_columns_than_max_len_takes_refused():
    """A view of some columns of a wider table covers what its columns cover:
    pages are not taken from the table's other columns or from behind it."""
    torch = pytest.importorskip("torch")
    ctx, x = host_ctx(), heads()
    wide, lens = torch.ones(3, 8, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for view in (wide[:, :4], wide[:, 4:], wide[:, 2:6]):
        good, bad = H.paged_batch(view, lens, 64), H.paged_batch(view, lens, 65)
        assert (good.table_stride, good.n_seqs) == (8, 3)
        assert H.paged_attn_workspace(kv(), good, 4) == 0
        calls = (lambda b: ctx.paged_attn_dev(kv(), b, H.F32, 4, 0.125, x, x),
                 lambda b: ctx.paged_append_dev(kv(), b, H.F32, 3, x, x))
        for call in calls:
            with pytest.raises(H.C2hError, match="no context"):
                call(good)
            with pytest.raises(ValueError, match="cover"):
                call(bad)
        with pytest.raises(ValueError, match="cover"):
            H.paged_attn_workspace(kv(), bad, 4)
    # a single row's stride is its columns; a whole table is the library's to check
    assert H.paged_batch(wide[:1, :4], lens[:1], 64).table_stride == 4
    with pytest.raises(H.C2hError, match="cover"):
        H.paged_attn_workspace(kv(), H.paged_batch(wide[:1, :4], lens[:1], 65), 4)
    with pytest.raises(H.C2hError, match="cover"):
        H.paged_attn_workspace(kv(), H.paged_batch(wide, lens, 129), 4)


def test_calls_beyond_the_tensor_that_heads_took_refused():
    """The type, tokens, heads and width that a call names have to lie within
    the tensor; what heads() did not make is taken as it is described."""
    torch = pytest.importorskip("torch")
    ctx, rope, at = host_ctx(), H.rope(64, 1e6), torch.zeros(3, dtype=torch.int32)
    t = lambda *shape, dtype=torch.float32: H.heads(torch.zeros(*shape, dtype=dtype))  # noqa: E731
    small = [t(2, 4, 64), t(3, 1, 64), t(3, 4, 48), t(3, 4, 64, dtype=torch.bfloat16), t(3, 4, 64, dtype=torch.float16),
             t(3, 4, 64, dtype=torch.int32), t(3, 4, 64, dtype=torch.float64)]
    kv2 = kv()

    def calls(h):
        """Each place of each call with h there, the rest fitting."""
        x = lambda: t(3, 4, 64)  # noqa: E731
        return [lambda: ctx.rope_dev(rope, H.F32, h, at, 3, 4, 64, x()), lambda: ctx.rope_dev(rope, H.F32, x(), at, 3, 4, 64, h),
                lambda: ctx.paged_append_dev(kv2, batch(), H.F32, 3, h, x()),
                lambda: ctx.paged_append_dev(kv2, batch(), H.F32, 3, x(), h),
                lambda: ctx.paged_append_dev(kv2, batch(), H.F32, 3, x(), x(), q=h, q_out=x(), n_heads=4),
                lambda: ctx.paged_append_dev(kv2, batch(), H.F32, 3, x(), x(), q=x(), q_out=h, n_heads=4),
                lambda: ctx.paged_attn_dev(kv2, batch(), H.F32, 4, 0.125, h, x()),
                lambda: ctx.paged_attn_dev(kv2, batch(), H.F32, 4, 0.125, x(), h)]

    for bad in small:
        for call in calls(bad):
            with pytest.raises(ValueError):
                call()
    for good in (t(3, 4, 64), t(5, 6, 80), heads()):
        for call in calls(good):
            with pytest.raises(H.C2hError, match="no context"):
                call()
    # found to fit one call does not answer for another
    good = t(3, 4, 64)
    for _ in range(2):
        for n, n_heads, dim, ty in ((3, 4, 64, H.F32), (4, 4, 64, H.F32), (3, 5, 64, H.F32), (3, 4, 72, H.F32),
                                    (3, 4, 64, H.BF16), (3, 4, 64, H.F16)):
            fits = (n, n_heads, dim, ty) == (3, 4, 64, H.F32)
            with pytest.raises(H.C2hError if fits else ValueError):
                ctx.rope_dev(rope, ty, good, torch.zeros(9, dtype=torch.int32), n, n_heads, dim, heads())


def test_tensors_that_are_not_on_the_contexts_gpu_refused():
    """A CPU tensor, or one of another GPU, would fault in the kernel."""
    torch = pytest.importorskip("torch")
    ctx, rope = host_ctx(), H.rope(64, 1e6)
    f, i = (lambda *s: torch.zeros(*s)), (lambda *s: torch.zeros(*s, dtype=torch.int32))
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.uint8)
    norm = dict(x=f(3, 512), w=f(512), q8k=torch.zeros(3, 2, 292, dtype=torch.uint8), residual=f(3, 512), sum_out=f(3, 512), y=f(3, 512))

    class Elsewhere:
        """t, on GPU 1."""

        def __init__(self, t):
            self.t = t

        def get_device(self):
            return 1

        def __getattr__(self, name):
            return getattr(self.t, name)

    def calls(x=heads(), y=heads(), pos=i(3), start=i(4), kv_=kv(), batch_=batch(), **more):
        return [lambda: ctx.rope_dev(rope, H.F32, x, pos, 3, 4, 64, y),
                lambda: ctx.paged_append_dev(kv_, batch_, H.F32, 3, x, y, token_start=start, q=y, q_out=x, n_heads=4),
                lambda: ctx.paged_attn_dev(kv_, batch_, H.F32, 4, 0.125, x, y),
                lambda: ctx.rmsnorm_q8k_dev(H.F32, eps=1e-6, **dict(norm, **more))]

    def said(call):
        with pytest.raises((ValueError, H.C2hError)) as e:
            call()
        return "GPU" if "GPU" in str(e.value) else "context" if "no context" in str(e.value) else str(e.value)

    own = dict(x=H.heads(f(3, 4, 64)), kv_=H.paged_kv(pool, pool.clone(), H.F8_E4M3, k_scale=f(2)), batch_=H.paged_batch(i(3, 8), i(3), 128))
    assert [said(c) for c in calls(**{**own, "x": heads()})] == ["context"] * 4
    assert said(calls(x=own["x"])[0]) == "context"
    far = dict(x=H.heads(Elsewhere(f(3, 4, 64))), y=H.heads(Elsewhere(f(3, 4, 64))),
               kv_=H.paged_kv(Elsewhere(pool), Elsewhere(pool.clone()), H.F8_E4M3), batch_=H.paged_batch(Elsewhere(i(3, 8)), Elsewhere(i(3)), 128))
    for name, which in (("x", (0, 1, 2)), ("y", (0, 1, 2)), ("kv_", (1, 2)), ("batch_", (1, 2))):
        got = [said(c) for c in calls(**{name: far[name]})[:3]]
        assert got == ["GPU" if n in which else "context" for n in range(3)], (name, got)
    assert said(calls(pos=Elsewhere(i(3)))[0]) == "GPU" and said(calls(start=Elsewhere(i(4)))[1]) == "GPU"
    for name in norm:
        x = norm[name]
        assert said(lambda: ctx.rmsnorm_q8k_dev(H.F32, eps=1e-6, **dict(norm, **{name: Elsewhere(x)}))) == "GPU", name
    for bad in (dict(k=Elsewhere(pool), v=pool), dict(k=pool, v=pool, k_scale=Elsewhere(f(2))), dict(k=pool, v=pool, v_scale=Elsewhere(f(2)))):
        with pytest.raises(ValueError, match="GPU"):
            H.paged_kv(ggml_type=H.F8_E4M3, **bad)
    with pytest.raises(ValueError, match="GPU"):
        H.paged_batch(i(3, 8), Elsewhere(i(3)), 128)
    # a context of a GPU takes nothing of the CPU's
    ctx.device = 0
    assert [said(c) for c in calls(**own)] == ["GPU"] * 4


LARGEST = r"""
#include <initializer_list>
#include <cassert>
#include <cstdio>
#include "c2h_paged.h"
using namespace c2h;
int main() {
  // batches up to the largest that a call accepts: a chunk's positions, and
  // the positions that a session's chunks begin and end at, fit 32 bits, and
  // the chunks cover the session
  for (int unit : {64, 128, 256})
    for (int n_seqs : {1, 64, 1000, 16383, 65535})
      for (int n_rows : {1, 16, 256, 1024, 4096})
        for (int len : {1, 5000, 131072, 140000, 1 << 20, PAGED_MAX_LEN - 1, PAGED_MAX_LEN}) {
          if ((int64_t)n_seqs * n_rows > MAX_SESSION_HEADS) continue;
          const Span s = attended(len, 0);
          const int units = units_of(s, unit), cu = chunk_units((int64_t)units * n_seqs, n_rows);
          const int chunk = cu * unit, n = chunks_of(units, cu);  // as the kernel computes it
          assert(cu >= 1 && chunk >= unit && n >= 1 && (int64_t)n * n_seqs <= chunks_bound(n_seqs, n_rows, units));
          int at = 0;
          for (int i = 0; i < n; ++i) {
            const int b = chunk_base(s, chunk, i), e = b + chunk < s.hi ? b + chunk : s.hi;
            assert(b == at && e > b);
            at = e;
          }
          assert(at == len);
        }
  puts("ok");
}
"""


def test_chunks_of_the_largest_batches(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(LARGEST)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "c2slm_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stderr


def test_batch_of_empty_sessions_without_pages():
    """max_len 0: no session holds a position, and the table may be empty."""
    L, n, q = H.lib(), C.c_size_t(7), heads()
    none = batch(block_table=None, table_stride=0, max_len=0)
    assert L.c2h_paged_attn_workspace(kv(), none, 4, 0, C.byref(n)) == 0 and n.value == 0
    refused(L.c2h_paged_attn_dev(None, kv(), none, H.F32, 4, 0.125, 0, q, q), INVALID, "no context")
    refused(L.c2h_paged_append_dev(None, kv(), none, None, 3, None, H.F32, q, q, 0, None, None), INVALID, "no context")
    refused(L.c2h_paged_attn_dev(None, kv(), batch(block_table=None, table_stride=0, max_len=0, seq_lens=None), H.F32, 4, 0.125, 0,
                                 q, q), INVALID, "lengths")
