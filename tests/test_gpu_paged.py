"""The operators over many sessions on the GPU against their formulas in 64
bits on the CPU: paged attention, append with rotation, rotation alone,
RMSNorm to Q8_K rows, and a layer's run of them.

Tolerances count roundings.  A value rounded to a type is off by at most half
a step: |x| U[type], at least half the least subnormal.  Attention's scores
are 32-bit sums over head_dim of products, (head_dim + 8) 2^-24 sum |q k|
each; a probability is off by twice that (its own score and the maximum's),
by 2^-22 of its exponent's size, and by what its split into 16-bit parts
leaves; the weighted sum adds at most 256 roundings of 2^-24 along its
longest chain of matrix instructions, waves and chunks."""
import math

import numpy as np
import pytest
import torch

from c2slm_amd import _lib as H
from c2slm_amd import gguf as G
from oracle import oracle as O

pytestmark = pytest.mark.gpu

TORCH = {H.F32: torch.float32, H.F16: torch.float16, H.BF16: torch.bfloat16, H.F8_E4M3: torch.float8_e4m3fn}
U = {H.F32: 2.0 ** -24, H.F16: 2.0 ** -11, H.BF16: 2.0 ** -8, H.F8_E4M3: 2.0 ** -4}
TINY = {H.F32: 2.0 ** -150, H.F16: 2.0 ** -25, H.BF16: 2.0 ** -134, H.F8_E4M3: 2.0 ** -10}
NAMES = {H.F32: "f32", H.F16: "f16", H.BF16: "bf16", H.F8_E4M3: "e4m3"}
RANGE = -5


@pytest.fixture(scope="module")
def ctx():
    c = H.Ctx(None)
    yield c
    c.close()


def rounding(want, ty):
    return want.abs() * U[ty] + TINY[ty]


def nan_pool(shape, ty):
    """A pool whose every element is NaN: what a kernel must not use."""
    if ty == H.F8_E4M3:
        return torch.full(shape, 0x7F, dtype=torch.uint8).view(TORCH[ty])
    return torch.full(shape, float("nan"), dtype=torch.float32).to(TORCH[ty])


class Sessions:
    """A batch over a pool: only held positions hold numbers, pages are
    handed out in random order, unused table entries point outside."""

    def __init__(self, lens, kv, dim, page, order, cache, seed, scaled=True, max_len=None, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kv, self.dim, self.page, self.cache, self.order = lens, kv, dim, page, cache, order
        need = [-(-max(n, 0) // page) for n in lens]
        self.width = max(max(need), 1) + 1
        self.n_pages = sum(need) + spare
        perm = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(lens), self.width), -7, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = perm[at:at + n]
            at += n
        shape = (self.n_pages, page, kv, dim) if order == "nhd" else (self.n_pages, kv, page, dim)
        self.pools = [nan_pool(shape, cache), nan_pool(shape, cache)]
        self.rows = []  # per session [2][len, kv, dim] in 64 bits, as stored
        e4 = cache == H.F8_E4M3
        self.scale = (torch.rand(2, kv, generator=g) + 0.5) / 16 if e4 and scaled else None
        for s, n in enumerate(lens):
            pair = []
            for i in range(2):
                x = (torch.randn(max(n, 0), kv, dim, generator=g) * (16 if e4 else 1)).to(TORCH[cache])
                pos = torch.arange(max(n, 0))
                self.view(i, bits=True)[self.table[s].long()[pos // page], pos % page] = self.bits(x)
                x = x.double()
                pair.append(x if self.scale is None else x * self.scale[i].double().view(1, -1, 1))
            self.rows.append(pair)
        self.max_len = max(max(lens), 0) if max_len is None else max_len

    @staticmethod
    def bits(x):
        return x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])

    def view(self, i, bits=False):
        p = self.bits(self.pools[i]) if bits else self.pools[i]
        return p if self.order == "nhd" else p.transpose(1, 2)

    def cuda(self):
        self.dev = [p.cuda() for p in self.pools]
        self.table_d, self.lens_d = self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.scale_d = None if self.scale is None else self.scale.cuda()
        sc = self.scale_d if self.scale_d is not None else [None, None]
        kv = H.paged_kv(self.dev[0], self.dev[1], self.cache, self.order, sc[0], sc[1])
        return kv, H.paged_batch(self.table_d, self.lens_d, self.max_len)


def attention64(sess, q, scale, window, ty):
    """(out, tolerance) [sessions, heads, dim] in 64 bits."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // sess.kv
    split = 2.0 ** -21 if ty == H.F32 else 2.0 ** -15
    for s, n in enumerate(sess.lens):
        lo = max(0, n - window) if window else 0
        if n <= 0:
            continue
        for h in range(q.shape[1]):
            k, v = (r[lo:n, h // group] for r in sess.rows[s])
            qk = k * q[s, h].double()
            sc = qk.sum(-1) * scale
            p = torch.softmax(sc, -1)
            out[s, h] = p @ v
            ds = abs(scale) * (sess.dim + 8) * 2.0 ** -24 * qk.abs().sum(-1).max() + sc.abs().max() * 2.0 ** -22
            tol[s, h] = (p @ v.abs()) * (4 * ds + split + 256 * 2.0 ** -24)
    return out, tol + rounding(out, ty)


def run_attention(ctx, sess, q, scale, window=0, extra_rows=2):
    """The kernel's rows on a strided q and an out with rows beyond the batch."""
    kv, batch = sess.cuda()
    n, heads, dim = q.shape
    ty = {v: k for k, v in TORCH.items()}[q.dtype]
    fused = torch.full((n, heads + 2, dim + 16), 7.0, dtype=q.dtype, device="cuda")
    fused[:, 1:heads + 1, :dim] = q.cuda()
    buf = torch.full((n + extra_rows, heads + 1, dim), 5.0, dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_attn_dev(kv, batch, ty, heads, scale, H.heads(fused[:, 1:heads + 1, :dim]), H.heads(buf[:n, :heads]),
                       window=window)
    ctx.sync()
    got = buf.cpu()
    assert (got[n:] == 5.0).all() and (got[:n, heads:] == 5.0).all(), "rows behind the batch changed"
    return got[:n, :heads].double()


def check_attention(ctx, lens, heads, kv, dim, page, order, cache, ty, window=0, seed=1, q_scale=1.0, max_len=None):
    sess = Sessions(lens, kv, dim, page, order, cache, seed, max_len=max_len)
    g = torch.Generator().manual_seed(seed + 100)
    q = (torch.randn(len(lens), heads, dim, generator=g) * q_scale).to(TORCH[ty])
    scale = dim ** -0.5
    want, tol = attention64(sess, q, scale, window, ty)
    got = run_attention(ctx, sess, q, scale, window)
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


TYPES = [(c, t) for c in (H.F32, H.F16, H.BF16, H.F8_E4M3) for t in (H.F32, H.F16, H.BF16)]
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 200]


@pytest.mark.parametrize("cache,ty", TYPES, ids=lambda t: NAMES[t])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (16, 8, 128), (3, 1, 256)])
def test_attention_types_and_lengths(ctx, cache, ty, heads, kv, dim):
    check_attention(ctx, LENS, heads, kv, dim, 16, "nhd", cache, ty)


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 240, 256])
@pytest.mark.parametrize("cache", [H.F32, H.BF16, H.F8_E4M3], ids=lambda t: NAMES[t])
def test_attention_head_dims(ctx, dim, cache):
    check_attention(ctx, [5, 70, 300], 6, 2, dim, 8, "hnd", cache, H.F32, seed=dim)


@pytest.mark.parametrize("heads,kv", [(1, 1), (7, 7), (16, 1), (17, 1), (24, 1), (40, 2), (64, 2), (71, 1)])
@pytest.mark.parametrize("cache", [H.F16, H.F32], ids=lambda t: NAMES[t])
def test_attention_head_groups(ctx, heads, kv, cache):
    check_attention(ctx, [3, 50, 0, 129], heads, kv, 64, 32, "nhd", cache, H.F16, seed=heads)


@pytest.mark.parametrize("page", [8, 32, 128, 1024])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
def test_attention_pages(ctx, page, order):
    check_attention(ctx, [1, 7, 8, 9, 1023, 1024, 1025, 2500], 4, 2, 128, page, order, H.BF16, H.BF16, seed=page)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 100, 129, 1000, 5000])
@pytest.mark.parametrize("cache", [H.BF16, H.F8_E4M3], ids=lambda t: NAMES[t])
def test_attention_windows(ctx, window, cache):
    check_attention(ctx, [0, 1, 16, 99, 128, 130, 1500, 4097], 8, 2, 64, 16, "nhd", cache, H.F32, window=window)


@pytest.mark.parametrize("cache,ty", [(H.F32, H.F32), (H.F16, H.F32), (H.BF16, H.BF16), (H.F8_E4M3, H.F16)],
                         ids=lambda t: NAMES[t])
@pytest.mark.parametrize("n", [4095, 9000, 33001])
def test_attention_split_sessions(ctx, cache, ty, n):
    # one long session beside short ones: chunks that are whole, ragged, absent
    check_attention(ctx, [n, 1, 0, 700, n // 2], 14, 2, 64, 16, "hnd", cache, ty, seed=n)


@pytest.mark.parametrize("n", [63, 64, 65, 129, 513, 1500])
@pytest.mark.parametrize("window", [0, 200])
def test_attention_many_sessions(ctx, n, window):
    # each lane of a wave looks after one session, a few, more than eight;
    # some are split, some empty
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 40, n)
    lens[rng.integers(0, n, 8)] = rng.integers(300, 2500, 8)
    check_attention(ctx, lens.tolist(), 2, 1, 16, 16, "nhd", H.F32, H.F32, window=window, seed=n)


@pytest.mark.parametrize("dim,cache,ty", [(64, H.F16, H.F16), (80, H.F32, H.BF16), (128, H.BF16, H.F32), (144, H.F16, H.F32),
                                          (256, H.F8_E4M3, H.BF16)], ids=str)
def test_attention_join_of_many_rows(ctx, dim, cache, ty):
    # 2,200 rows: most of one chunk, some of several, empty ones and a bad page
    rng = np.random.default_rng(dim)
    lens = rng.integers(0, 30, 1100)
    lens[[0, 7, 500, 1099]] = [3000, 700, 1111, 2000]
    check_attention(ctx, lens.tolist(), 2, 1, dim, 16, "hnd", cache, ty, seed=dim)
    sess = Sessions([int(n) for n in lens], 1, dim, 16, "hnd", cache, dim)
    sess.table[500, 40] = -1
    kv, batch = sess.cuda()
    q = torch.ones(1100, 2, dim).to(TORCH[ty]).cuda()
    out = torch.full_like(q, 5.0)
    torch.cuda.synchronize()
    ctx.paged_attn_dev(kv, batch, ty, 2, 0.01, H.heads(q), H.heads(out))
    with pytest.raises(H.C2hError):
        ctx.sync()
    got = out.cpu()
    assert torch.isnan(got[500]).all() and torch.isfinite(got[torch.arange(1100) != 500]).all()


def strided_pool(sess, how):
    """The session's pools laid out otherwise on the GPU: (k, v) views."""
    k, v = sess.pools
    if how == "side by side":  # a page's keys, then its values
        both = torch.stack([k.view(torch.int8) if sess.cache == H.F8_E4M3 else k, v.view(torch.int8) if sess.cache == H.F8_E4M3 else v], 1).cuda()
        if sess.cache == H.F8_E4M3:
            both = both.view(TORCH[sess.cache])
        return both, both[:, 0], both[:, 1]
    if how == "heads outermost":
        out = [p.permute(2, 0, 1, 3).contiguous().cuda().permute(1, 2, 0, 3) for p in sess.pools]
        return out, out[0], out[1]
    wide = [torch.zeros((p.shape[0], p.shape[1] + 1, p.shape[2] + 2, p.shape[3] + 16), dtype=p.dtype) for p in sess.pools]
    for w, p in zip(wide, sess.pools):  # gaps after elements, heads, tokens
        w[:, :-1, :-2, :-16] = p
    wide = [w.cuda() for w in wide]
    return wide, *(w[:, :-1, :-2, :-16] for w in wide)


@pytest.mark.parametrize("how", ["side by side", "heads outermost", "gaps"])
@pytest.mark.parametrize("cache", [H.F32, H.BF16], ids=lambda t: NAMES[t])
def test_pools_of_other_strides(ctx, how, cache):
    # append three tokens a session, then attend with one query for all sessions
    lens = [3, 40, 300, 17]
    sess = Sessions(lens, 2, 64, 16, "nhd", cache, 3)
    g = torch.Generator().manual_seed(4)
    kn, vn = torch.randn(12, 2, 64, generator=g), torch.randn(12, 2, 64, generator=g)
    keep, k, v = strided_pool(sess, how)
    sess.cuda()
    kv, batch = H.paged_kv(k, v, cache), H.paged_batch(sess.table_d, sess.lens_d, max(lens))
    start = torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32).cuda()
    kd, vd = kn.cuda(), vn.cuda()
    q = torch.randn(1, 4, 64, generator=g).cuda()
    out = torch.zeros(4, 4, 64, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_append_dev(kv, batch, H.F32, 12, H.heads(kd), H.heads(vd), token_start=start)
    ctx.paged_attn_dev(kv, batch, H.F32, 4, 0.125, H.Heads(q.data_ptr(), 0, 64), H.heads(out))
    ctx.sync()
    for s, n in enumerate(lens):
        for i, x in enumerate((kn, vn)):
            sess.rows[s][i][n - 3:] = x[3 * s:3 * s + 3].to(TORCH[cache]).double()
    want, tol = attention64(sess, q.cpu().expand(4, 4, 64), 0.125, 0, H.F32)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    if how == "gaps":
        assert all((w[:, -1:] == 0).all() and (w[:, :, -2:] == 0).all() and (w[..., -16:] == 0).all() for w in keep)


def test_offsets_beyond_32_bits(ctx):
    # a pool of 6 GiB each of keys and values: pages at its start and its end
    pages = (6 << 30) // (16 * 8 * 128 * 2)
    pool = [torch.empty((pages, 16, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    used = [pages - 1, 0, pages - 2, pages // 2, pages // 3 * 2]
    lens = [70]
    sess = Sessions(lens, 8, 128, 16, "nhd", H.BF16, 8, spare=0)
    rank = {int(p): u for p, u in zip(sess.table[0, :5], used)}
    for i in range(2):
        for p, u in rank.items():
            pool[i][u] = sess.pools[i][p].cuda()
    table = torch.tensor([used], dtype=torch.int32).cuda()
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    kv, batch = H.paged_kv(pool[0], pool[1], H.BF16), H.paged_batch(table, lens_d, 80)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(1, 16, 128, generator=g).bfloat16()
    x = torch.randn(1, 16, 128, generator=g).bfloat16().cuda()  # the 70th token: page 4, slot 5
    qd, out = q.cuda(), torch.zeros(1, 16, 128, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_append_dev(kv, batch, H.BF16, 1, H.heads(x[:, :8]), H.heads(x[:, 8:]))
    ctx.paged_attn_dev(kv, batch, H.BF16, 16, 0.1, H.heads(qd), H.heads(out))
    ctx.sync()
    for i in range(2):
        sess.rows[0][i][69] = x[0, 8 * i:8 * i + 8].cpu().double()
        assert torch.equal(pool[i][used[4], 5], x[0, 8 * i:8 * i + 8])
    want, tol = attention64(sess, q, 0.1, 0, H.BF16)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("cache,ty", [(H.F32, H.F32), (H.BF16, H.BF16), (H.F8_E4M3, H.F16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("window", [0, 1111])
def test_attention_chunks_of_more_pages_than_lanes(ctx, cache, ty, window):
    # 1,024 rows of up to 163 pages each, whole sessions by one workgroup: a
    # wave's lanes hold 64 pages at a time
    lens = [1300 - 7 * (i % 19) for i in range(62)] + [513, 1]
    check_attention(ctx, lens, 16, 16, 16, 8, "nhd", cache, ty, window=window)


def test_attention_bad_page_past_the_first_64(ctx):
    lens = [1300] * 64
    sess = Sessions(lens, 16, 16, 8, "nhd", H.F16, 9)
    held = sess.table.clone()
    sess.table[3, 100] = sess.n_pages
    sess.table[9, 162] = -5
    q = torch.randn(64, 16, 16, generator=torch.Generator().manual_seed(7)).half()
    kv, batch = sess.cuda()
    out, qd = torch.zeros_like(q, device="cuda"), q.cuda()
    torch.cuda.synchronize()
    ctx.paged_attn_dev(kv, batch, H.F16, 16, 0.25, H.heads(qd), H.heads(out))
    with pytest.raises(H.C2hError) as e:
        ctx.sync()
    assert e.value.code == RANGE and "page" in str(e.value) and "length" not in str(e.value)
    got = out.cpu().double()
    assert torch.isnan(got[[3, 9]]).all()
    sess.table = held
    want, tol = attention64(sess, q, 0.25, 0, H.F16)
    rest = [i for i in range(64) if i not in (3, 9)]
    assert ((got - want).abs()[rest] <= tol[rest]).all()


def test_attention_max_len_beyond_the_lengths(ctx):
    # the launch is sized by a bound far above the lengths: most chunks are empty
    sess = Sessions([5, 0, 300], 2, 64, 16, "nhd", H.F16, 3)
    sess.table = torch.nn.functional.pad(sess.table, (0, 2000), value=-9)
    sess.max_len = 16 * 2000
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(5)).half()
    want, tol = attention64(sess, q, 0.125, 0, H.F16)
    assert ((run_attention(ctx, sess, q, 0.125) - want).abs() <= tol).all()


@pytest.mark.parametrize("q_scale", [2.0 ** -30, 2.0 ** -12, 64.0, 300.0])
@pytest.mark.parametrize("cache,ty", [(H.F16, H.F32), (H.F8_E4M3, H.BF16), (H.BF16, H.F32), (H.F32, H.F32)],
                         ids=lambda t: NAMES[t])
def test_attention_query_sizes(ctx, q_scale, cache, ty):
    # even probabilities, and ones that all but a position or two lose
    check_attention(ctx, [1, 40, 500], 4, 2, 64, 16, "nhd", cache, ty, q_scale=q_scale)


@pytest.mark.parametrize("cache", [H.F32, H.F16, H.BF16, H.F8_E4M3], ids=lambda t: NAMES[t])
def test_attention_late_maximum(ctx, cache):
    # the largest score comes last, then first: what was summed before it is
    # brought down, in a wave, between waves and between chunks
    for where in (0, 1, 37, 130, 2999):
        sess = Sessions([3000], 1, 64, 16, "nhd", cache, 11, scaled=False)
        k = torch.full((64,), 0.5)
        page, at = sess.table[0, where // 16].item(), where % 16
        sess.view(0, bits=True)[page, at, 0] = Sessions.bits((k * 12).to(TORCH[cache]))
        sess.rows[0][0][where, 0] = (k * 12).to(TORCH[cache]).double()
        q = torch.full((1, 2, 64), 1.0)
        q[:, 1] = -1.0
        want, tol = attention64(sess, q, 0.25, 0, H.F32)
        got = run_attention(ctx, sess, q, 0.25)
        assert ((got - want).abs() <= tol).all(), where


def test_attention_nan_and_infinity_of_held_positions(ctx):
    # a NaN key makes its head's row NaN and no other's; an infinite value
    # with weight stays infinite
    sess = Sessions([100, 100], 2, 64, 16, "nhd", H.F32, 4)
    sess.view(0)[sess.table[0, 2].item(), 3, 1] = float("nan")
    sess.view(1)[sess.table[1, 1].item(), 5, 0, 7] = float("inf")
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(6))
    want, tol = attention64(sess, q, 0.125, 0, H.F32)
    got = run_attention(ctx, sess, q, 0.125)
    assert torch.isnan(got[0, 2:]).all()
    assert (got[1, :2, 7] == float("inf")).all()
    got[1, :2, 7] = want[1, :2, 7]
    assert ((got - want).abs()[0, :2] <= tol[0, :2]).all() and ((got - want).abs()[1] <= tol[1]).all()


@pytest.mark.parametrize("n", [40, 5000])
def test_attention_bad_tables_and_lengths_are_reported(ctx, n):
    # a page outside the pool, a length above max_len, a negative one: their
    # rows are NaN, the others right, and the next sync says so, once
    sess = Sessions([n] * 6, 2, 64, 16, "nhd", H.F16, 9)
    held = sess.table.clone()
    sess.table[1, 1] = sess.n_pages
    sess.table[2, (n - 1) // 16] = -1
    sess.max_len = n
    sess.lens = [n, n, n, n + 1, -3, n]
    q = torch.randn(6, 4, 64, generator=torch.Generator().manual_seed(7)).half()
    kv, batch = sess.cuda()
    out, qd = torch.zeros(6, 4, 64, dtype=torch.float16, device="cuda"), q.cuda()
    torch.cuda.synchronize()
    ctx.paged_attn_dev(kv, batch, H.F16, 4, 0.125, H.heads(qd), H.heads(out))
    with pytest.raises(H.C2hError) as e:
        ctx.sync()
    assert e.value.code == RANGE and "length" in str(e.value) and "page" in str(e.value)
    ctx.sync()
    got = out.cpu().double()
    assert torch.isnan(got[1:5]).all()
    sess.table, sess.lens = held, [n] * 6
    want, tol = attention64(sess, q, 0.125, 0, H.F16)
    assert ((got - want).abs()[[0, 5]] <= tol[[0, 5]]).all()


def test_attention_repeats_bit_for_bit_and_survives_a_smaller_call(ctx):
    g = torch.Generator().manual_seed(8)
    big = Sessions([9000, 100], 2, 64, 16, "nhd", H.BF16, 21)
    q = torch.randn(2, 14, 64, generator=g).bfloat16()
    first = run_attention(ctx, big, q, 0.125)
    for _ in range(3):
        check_attention(ctx, [700], 4, 2, 64, 16, "nhd", H.F32, H.F32)
        assert torch.equal(run_attention(ctx, big, q, 0.125), first)


def test_two_contexts_at_once():
    a, b = H.Ctx(None), H.Ctx(None)
    try:
        sess = [Sessions([6000 + i, 50], 2, 128, 16, "nhd", H.F16, 31 + i) for i in range(2)]
        q = [torch.randn(2, 12, 128, generator=torch.Generator().manual_seed(40 + i)).half() for i in range(2)]
        want = [attention64(s, x, 0.1, 0, H.F16) for s, x in zip(sess, q)]
        made = [s.cuda() for s in sess]
        qd, out = [x.cuda() for x in q], [torch.zeros_like(x.cuda()) for x in q]
        torch.cuda.synchronize()
        for _ in range(20):
            for c, m, x, o in zip((a, b), made, qd, out):
                c.paged_attn_dev(m[0], m[1], H.F16, 12, 0.1, H.heads(x), H.heads(o))
        a.sync(), b.sync()
        for o, (w, t) in zip(out, want):
            assert ((o.cpu().double() - w).abs() <= t).all()
    finally:
        a.close(), b.close()


# ------------------------------------------------------- rotation and append

def rotate64(x, pos, rot, base, layout, freq=None, mscale=1.0):
    """x [tokens, heads, dim] in 64 bits, and what 32-bit arithmetic may be
    off: cos and sin by 2^-22 (their own error, the angle's fraction and the
    product with mscale), the two products and their sum by a rounding each."""
    f = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot) if freq is None else freq
    a = (pos.double().unsqueeze(1) * f).unsqueeze(1)
    c, s = a.cos() * mscale, a.sin() * mscale
    x = x.double()
    y, tol = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = x[..., one], x[..., two]
    y[..., one], y[..., two] = u * c - v * s, u * s + v * c
    t = (u.abs() + v.abs()) * mscale * (2.0 ** -22 + 2.0 ** -23)
    tol[..., one], tol[..., two] = t, t
    return y, tol


ROPES = [(64, 64, "half"), (64, 32, "half"), (128, 128, "interleaved"), (128, 40, "half"), (80, 8, "interleaved"),
         (256, 256, "half"), (112, 104, "interleaved"), (96, 24, "half")]


@pytest.mark.parametrize("ty", [H.F32, H.F16, H.BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("dim,rot,layout", ROPES)
def test_rope(ctx, ty, dim, rot, layout):
    g = torch.Generator().manual_seed(dim + rot)
    pos = torch.tensor([0, 1, -5, 40, 32767, 1000003, 2 ** 31 - 1, -2 ** 31, 7, 8, 9], dtype=torch.int32)
    x = torch.randn(len(pos), 5, dim, generator=g).to(TORCH[ty])
    want, tol = rotate64(x, pos, rot, 1e6, layout, mscale=1.2)
    # angles reach 2^31 radians: 64 bits leave 2^31 * 2^-52 of one
    tol = tol + x.double().abs().amax() * 2 * 2.0 ** -21 + rounding(want, ty)
    r = H.rope(rot, 1e6, layout=layout, mscale=1.2)
    buf = torch.full((len(pos) + 1, 7, dim), 3.0, dtype=TORCH[ty], device="cuda")
    buf[:len(pos), 1:6] = x.cuda()
    out = torch.full_like(buf, 9.0)
    pd = pos.cuda()
    torch.cuda.synchronize()
    ctx.rope_dev(r, ty, H.heads(buf[:-1, 1:6]), pd, len(pos), 5, dim, H.heads(out[:-1, 1:6]))
    ctx.sync()
    got = out.cpu().double()
    inner = got[:-1, 1:6]
    bad = (inner - want).abs() > tol
    bad[..., rot:] |= inner[..., rot:] != x[..., rot:].double()
    assert not bad.any()
    got[:-1, 1:6] = 9.0
    assert (got == 9.0).all(), "elements beside the heads changed"
    # in place gives the same bits
    ctx.rope_dev(r, ty, H.heads(buf[:-1, 1:6]), pd, len(pos), 5, dim, H.heads(buf[:-1, 1:6]))
    ctx.sync()
    assert torch.equal(buf[:-1, 1:6].cpu(), out[:-1, 1:6].cpu())


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 14), (3, 40), (257, 2), (1000, 3)])
def test_rope_sizes_and_scaled_frequencies(ctx, tokens, heads):
    g = torch.Generator().manual_seed(tokens)
    x, pos = torch.randn(tokens, heads, 64, generator=g), torch.arange(100, 100 + tokens, dtype=torch.int32)
    xd, pd = x.cuda(), pos.cuda()
    for r in (H.rope(64, 1e4, factor=8.0, orig_ctx=2048), H.rope(64, 1e4, freq_factors=np.linspace(1, 4, 32))):
        out = torch.zeros_like(xd)
        torch.cuda.synchronize()
        ctx.rope_dev(r, H.F32, H.heads(xd), pd, tokens, heads, 64, H.heads(out))
        ctx.sync()
        f = torch.tensor(list(r.turns[:32]), dtype=torch.float64) * 2 * math.pi
        want, tol = rotate64(x, pos, 64, 1e4, "half", freq=f)
        assert ((out.cpu().double() - want).abs() <= tol + rounding(want, H.F32)).all()


def expect_append(sess, new, k, v, q, rot, layout, ty, base=1e6):
    """Pools after the append as (64-bit values, tolerance) where written."""
    pools = [sess.view(i).double().clone() for i in range(2)]
    tols = [torch.full(p.shape, -1.0, dtype=torch.float64) for p in pools]
    qw, qt = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape, -1.0, dtype=torch.float64)
    at = 0
    for s, n in enumerate(new):
        if sess.lens[s] == 0:
            at += n
            continue
        pos = torch.arange(sess.lens[s] - n, sess.lens[s])
        rows = slice(at, at + n)
        at += n
        page, off = sess.table[s].long()[pos // sess.page], pos % sess.page
        for i, x in enumerate((k, v)):
            w, t = rotate64(x[rows], pos, rot, base, layout) if i == 0 and rot else (x[rows].double(), torch.zeros(x[rows].shape, dtype=torch.float64))
            if sess.cache == H.F8_E4M3:
                sc = sess.scale[i].double().view(1, -1, 1) if sess.scale is not None else 1.0
                w, t = (w / sc).clamp(-448, 448), t / sc + (w / sc).abs() * 2.0 ** -23
            pools[i][page, off], tols[i][page, off] = w, t + rounding(w + t, sess.cache)
        if rot:
            w, t = rotate64(q[rows], pos, rot, base, layout)
        else:
            w, t = q[rows].double(), torch.zeros(q[rows].shape, dtype=torch.float64)
        qw[rows], qt[rows] = w, t + rounding(w + t, ty)
    return pools, tols, qw, qt


def check_append(ctx, lens, new, heads, kv, dim, page, order, cache, ty, rot, layout, seed=1, decode=False, pad=0,
                 in_place=False, big=False):
    sess = Sessions(lens, kv, dim, page, order, cache, seed)
    if big and cache == H.F8_E4M3:
        sess.scale = sess.scale / 100  # beyond 448 after the division: saturates
    n = sum(new) + pad
    g = torch.Generator().manual_seed(seed + 1)
    fused = torch.randn(n, heads + 2 * kv, dim, generator=g).to(TORCH[ty])
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    pools, tols, qw, qt = expect_append(sess, new, k, v, q, rot, layout, ty)
    before = [sess.bits(sess.view(i)).clone() for i in range(2)]
    kvd, batch = sess.cuda()
    fd = fused.cuda()
    qo = fd[:, :heads] if in_place else torch.full((n, heads, dim), 6.0, dtype=TORCH[ty], device="cuda")
    start = None if decode else torch.tensor(np.cumsum([0] + new), dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    ctx.paged_append_dev(kvd, batch, ty, n, H.heads(fd[:, heads:heads + kv]), H.heads(fd[:, heads + kv:]), token_start=start,
                         rope=H.rope(rot, 1e6, layout=layout) if rot else None, q=H.heads(fd[:, :heads]) if heads else None,
                         q_out=H.heads(qo) if heads else None, n_heads=heads)
    ctx.sync()
    for i in range(2):
        sess.pools[i] = sess.dev[i].cpu()
        got, written = sess.view(i), tols[i] >= 0
        assert torch.equal(sess.bits(got)[~written], before[i][~written]), "a slot that is not the tokens' changed"
        off = (got.double() - pools[i]).abs()[written]
        assert (off <= tols[i][written]).all(), (i, float((off / tols[i][written]).max()))
    if heads:
        got, written = qo.cpu().double(), qt >= 0
        assert ((got - qw).abs()[written] <= qt[written]).all()
        if not in_place:
            assert (got[~written] == 6.0).all(), "q_out rows of no token changed"


@pytest.mark.parametrize("cache,ty", TYPES, ids=lambda t: NAMES[t])
@pytest.mark.parametrize("dim,rot,layout", [(64, 64, "half"), (128, 96, "interleaved"), (96, 40, "half"), (256, 0, "half")])
def test_append_step(ctx, cache, ty, dim, rot, layout):
    check_append(ctx, [1, 16, 17, 300, 0, 33], [1] * 6, 6, 2, dim, 16, "nhd", cache, ty, rot, layout, decode=True)


@pytest.mark.parametrize("cache", [H.F32, H.BF16, H.F8_E4M3], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("order,page", [("nhd", 8), ("hnd", 64)])
def test_append_prompts(ctx, cache, order, page):
    # whole prompts, later turns, a session without new tokens, padding
    # tokens behind the last session, and a row without a session
    check_append(ctx, [5, 100, 64, 0, 129, 200], [5, 37, 0, 3, 129, 1], 4, 2, 64, page, order, cache, H.BF16, 64, "half", pad=4)


def test_append_many_sessions(ctx):
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 60, 700).tolist()
    new = [int(rng.integers(0, n + 1)) for n in lens]
    check_append(ctx, lens, new, 2, 1, 64, 16, "nhd", H.F16, H.F16, 64, "half")


def test_append_in_place_without_queries_and_saturated(ctx):
    check_append(ctx, [9, 70], [9, 2], 4, 2, 64, 16, "hnd", H.BF16, H.BF16, 64, "half", in_place=True)
    check_append(ctx, [9, 70], [9, 2], 0, 2, 64, 16, "hnd", H.F16, H.F32, 64, "interleaved")
    check_append(ctx, [9, 70], [9, 2], 2, 2, 64, 16, "hnd", H.F8_E4M3, H.F32, 0, "half", big=True)


def test_append_e4m3_special_values(ctx):
    sess = Sessions([1], 1, 16, 8, "nhd", H.F8_E4M3, 1, scaled=False)
    vals = torch.tensor([0.0, -0.0, 448.0, 464.0, 1e9, -1e9, float("inf"), -float("inf"), float("nan"), 2.0 ** -9, 2.0 ** -10,
                         1.5 * 2.0 ** -9, 17.0, 18.0, 19.0, -21.0])
    x = vals.view(1, 1, 16).cuda()
    kv, batch = sess.cuda()
    torch.cuda.synchronize()
    ctx.paged_append_dev(kv, batch, H.F32, 1, H.heads(x), H.heads(x))
    ctx.sync()
    want = vals.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    page = sess.table[0, 0].item()
    for d in sess.dev:
        got = d.cpu()[page, 0, 0].float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5))


def test_append_bad_tables_lengths_and_starts_are_reported(ctx):
    sess = Sessions([20, 20, 20, 20, 20], 1, 64, 16, "nhd", H.F32, 2)
    keep = [p.clone() for p in sess.pools]
    sess.table[0, 1] = sess.n_pages + 5
    sess.table[1, 1] = -1
    sess.lens = [20, 20, 21, -1, 3]  # the last: four new tokens in a session of three
    sess.max_len = 20
    x = torch.randn(8, 1, 64, device="cuda")
    q = torch.full_like(x, 2.0)
    kv, batch = sess.cuda()
    start = torch.tensor([0, 1, 2, 3, 4, 8], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    ctx.paged_append_dev(kv, batch, H.F32, 8, H.heads(x), H.heads(x), token_start=start, q=H.heads(x), q_out=H.heads(q),
                         n_heads=1)
    with pytest.raises(H.C2hError) as e:
        ctx.sync()
    assert e.value.code == RANGE and all(w in str(e.value) for w in ("length", "page", "new tokens"))
    ctx.sync()
    assert (q[:5] == 2.0).all() and torch.equal(q[5:], x[5:])
    # the session of three holds its last three tokens, everything else is as it was
    page = sess.table[4, 0].item()
    for got, was in zip(sess.dev, keep):
        was[page, :3] = x[5:8].cpu()
        assert torch.equal(Sessions.bits(got.cpu()), Sessions.bits(was))


# ------------------------------------------------------- norm to Q8_K rows

def norm_expect(x, r, w, eps, ty):
    """(sum, y) as the operator defines them, y in the same 32-bit steps."""
    s = x if r is None else (x.float() + r.float()).to(TORCH[ty])
    f = s.float()
    scale = (1.0 / torch.sqrt(f.double().square().mean(-1, keepdim=True) + float(np.float32(eps)))).float()
    return s, f * scale * w


@pytest.mark.parametrize("ty", [H.F32, H.F16, H.BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("rows,cols", [(1, 256), (3, 264), (2, 896), (5, 1024), (2, 1536), (4, 2048), (2, 2056), (3, 4096),
                                       (2, 4864), (1, 8192), (2, 8960), (1, 16384), (300, 896)])
def test_norm(ctx, ty, rows, cols):
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(rows, cols + 8, generator=g).to(TORCH[ty])
    r = (torch.randn(rows, cols + 16, generator=g) * 3).to(TORCH[ty])
    w = torch.rand(cols, generator=g) + 0.5
    nb = cols // 256
    xd, rd, wd = x.cuda()[:, :cols], r.cuda()[:, :cols], w.cuda()
    for add in (False, True):
        s, y = norm_expect(x[:, :cols], r[:, :cols] if add else None, w, 1e-6, ty)
        for want_y in (False, True):
            q8k = torch.full((rows + 1, nb, 292), 0xAB, dtype=torch.uint8, device="cuda")
            so = torch.full((rows + 1, cols + 24), 4.0, dtype=TORCH[ty], device="cuda")
            yo = torch.full((rows + 1, cols + 4), 4.0, device="cuda")
            torch.cuda.synchronize()
            ctx.rmsnorm_q8k_dev(ty, xd, wd, 1e-6, q8k, residual=rd if add else None, sum_out=so[:, :cols] if add else None,
                                y=yo[:, :cols] if want_y else None)
            ctx.sync()
            got = q8k.cpu().numpy()
            for i in range(rows):
                assert np.array_equal(got[i].ravel(), O.quantize_row_q8k(y[i].numpy())), (add, want_y, i)
            assert (got[rows] == 0xAB).all()
            so, yo = so.cpu(), yo.cpu()
            if add:
                assert torch.equal(so[:rows, :cols], s)
            assert (so[rows:] == 4.0).all() and (so[:, cols:] == 4.0).all() and (add or (so == 4.0).all())
            if want_y:
                assert torch.equal(yo[:rows, :cols], y)
            assert (yo[rows:] == 4.0).all() and (yo[:, cols:] == 4.0).all() and (want_y or (yo == 4.0).all())


@pytest.mark.parametrize("ty", [H.F32, H.F16, H.BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("rows,cols,shift", [(3, 257, 0), (2, 434, 0), (4, 1001, 0), (2, 2047, 0), (1, 5003, 0), (1, 16383, 0),
                                             (3, 896, 1), (2, 1024, 2)])
def test_norm_odd_widths_and_alignments(ctx, ty, rows, cols, shift):
    # packed rows of odd widths; even ones that start between fours
    g = torch.Generator().manual_seed(cols)
    flat = [torch.randn(rows * cols + 8, generator=g).to(TORCH[ty]) for _ in range(2)]
    x, r = (f[shift:shift + rows * cols].view(rows, cols) for f in flat)
    w = torch.rand(cols + 4, generator=g)[shift:shift + cols]
    s, y = norm_expect(x, r, w, 1e-5, ty)
    fd = [f.cuda() for f in flat]
    xd, rd = (f[shift:shift + rows * cols].view(rows, cols) for f in fd)
    wd = torch.nn.functional.pad(w, (shift, 4)).cuda()[shift:shift + cols]
    nb = cols // 256
    q8k = torch.full((rows * nb * 292 + 8,), 0xAB, dtype=torch.uint8, device="cuda")
    so = torch.full((rows * cols + 8,), 4.0, dtype=TORCH[ty], device="cuda")
    yo = torch.full((rows * cols + 8,), 4.0, device="cuda")
    sv, yv = (t[shift:shift + rows * cols].view(rows, cols) for t in (so, yo))
    torch.cuda.synchronize()
    ctx.rmsnorm_q8k_dev(ty, xd, wd, 1e-5, q8k, residual=rd, sum_out=sv, y=yv)
    ctx.sync()
    got = q8k.cpu().numpy()
    for i in range(rows):
        assert np.array_equal(got[i * nb * 292:(i + 1) * nb * 292], O.quantize_row_q8k(y[i].numpy())), i
    assert (got[rows * nb * 292:] == 0xAB).all()
    assert torch.equal(sv.cpu(), s) and torch.equal(yv.cpu(), y)
    for t in (so, yo):
        assert (t[:shift] == 4.0).all() and (t[shift + rows * cols:] == 4.0).all(), "elements beside the rows changed"


def test_norm_in_place_zero_rows_and_special_values(ctx):
    g = torch.Generator().manual_seed(5)
    x, r, w = torch.randn(4, 896, generator=g), torch.randn(4, 896, generator=g), torch.ones(896)
    x[1] = r[1] = 0.0      # scale 1/sqrt(eps), zero blocks
    x[2, 300] = float("inf")   # every finite element becomes 0, this one NaN
    x[3, 700] = float("nan")
    s, y = norm_expect(x, r, w, 1e-6, H.F32)
    for target in ("x", "residual"):
        xd, rd, wd = x.cuda(), r.cuda(), w.cuda()
        q8k, yo = torch.zeros((4, 3, 292), dtype=torch.uint8, device="cuda"), torch.zeros(4, 896, device="cuda")
        torch.cuda.synchronize()
        so = xd if target == "x" else rd
        ctx.rmsnorm_q8k_dev(H.F32, xd, wd, 1e-6, q8k, residual=rd, sum_out=so, y=yo)
        ctx.sync()
        assert torch.equal(so.cpu().nan_to_num(99.0), s.nan_to_num(99.0))
        assert torch.equal(torch.isnan(yo.cpu()), torch.isnan(y)) and torch.equal(yo.cpu().nan_to_num(), y.nan_to_num())
        for i in range(4):
            assert np.array_equal(q8k[i].cpu().numpy().ravel(), O.quantize_row_q8k(y[i].numpy())), i


def test_empty_calls_do_nothing(ctx):
    sess = Sessions([4], 1, 64, 16, "nhd", H.F32, 1)
    kv, batch = sess.cuda()
    x, no = torch.ones(1, 1, 64, device="cuda"), torch.ones(0, 1, 64, device="cuda")
    none = H.PagedBatch(None, 0, None, 0, 0)
    ctx.paged_attn_dev(kv, none, H.F32, 1, 1.0, H.heads(no), H.heads(no))
    ctx.paged_append_dev(kv, none, H.F32, 0, H.heads(no), H.heads(no), q=H.heads(no), q_out=H.heads(no), n_heads=1)
    ctx.paged_append_dev(kv, batch, H.F32, 0, H.heads(no), H.heads(no), token_start=torch.zeros(2, dtype=torch.int32).cuda())
    ctx.rope_dev(H.rope(64, 1e4), H.F32, H.heads(no), None, 0, 1, 64, H.heads(no))
    ctx.rmsnorm_q8k_dev(H.F32, torch.ones(0, 256, device="cuda"), torch.ones(256, device="cuda"), 1e-6,
                        torch.zeros(16, dtype=torch.uint8, device="cuda"))
    ctx.sync()
    assert (x == 1.0).all()


# ------------------------------------------------------- a layer of them

@pytest.mark.parametrize("cache", [H.F32, H.BF16, H.F8_E4M3], ids=lambda t: NAMES[t])
def test_attention_block_of_a_layer(ctx, cache):
    """Norm, Q4_K projections of each row, append, attention and the output
    projection's quantiser, one after the other without a wait between them,
    over two steps of three sessions; attention against 64 bits on the values
    that the projections gave."""
    E, heads, kv, dim, page = 896, 14, 2, 64, 16
    g = torch.Generator().manual_seed(17)
    lens = [30, 1, 47]
    sess = Sessions(lens, kv, dim, page, "nhd", cache, 5)
    rng = np.random.default_rng(2)
    rows_w = (heads + 2 * kv) * dim
    raw = G.synth_q4_k(rng, rows_w * 3)
    packed = torch.from_numpy(H.pack_weights(H.Q4_K, rows_w, E, raw)).cuda()
    kvd, _ = sess.cuda()
    rope = H.rope(dim, 1e6)
    w = (torch.rand(E, generator=g) + 0.5).cuda()
    resid = torch.randn(3, E, generator=g).cuda()
    L = H.lib()
    for step in range(2):
        if step:
            sess.lens = [n + 1 for n in sess.lens]
            need = [-(-n // page) for n in sess.lens]
            assert max(need) <= sess.width
            spare = sorted(set(range(sess.n_pages)) - {p for s in range(3) for p in sess.table[s].tolist()})
            for s in range(3):  # a new page where the session fills its last one
                if sess.table[s, need[s] - 1] < 0:
                    sess.table[s, need[s] - 1] = spare.pop()
        x = torch.randn(3, E, generator=g)
        xd, table, lens_d = x.cuda(), sess.table.cuda(), torch.tensor(sess.lens, dtype=torch.int32).cuda()
        batch = H.paged_batch(table, lens_d, max(sess.lens))
        q8k = torch.zeros((3, 3, 292), dtype=torch.uint8, device="cuda")
        qkv = torch.zeros((3, heads + 2 * kv, dim), device="cuda")
        qr, att = torch.zeros((3, heads, dim), device="cuda"), torch.zeros((3, heads, dim), device="cuda")
        aq = torch.zeros((3, 3, 292), dtype=torch.uint8, device="cuda")
        before = resid.cpu()
        torch.cuda.synchronize()
        ctx.rmsnorm_q8k_dev(H.F32, xd, w, 1e-6, q8k, residual=resid, sum_out=resid)
        for s in range(3):
            assert L.c2h_gemv_dev(ctx.h, H.Q4_K, packed.data_ptr(), q8k[s].data_ptr(), rows_w, E, qkv[s].data_ptr(), None) == 0
        ctx.paged_append_dev(kvd, batch, H.F32, 3, H.heads(qkv[:, heads:heads + kv]), H.heads(qkv[:, heads + kv:]), rope=rope,
                             q=H.heads(qkv[:, :heads]), q_out=H.heads(qr), n_heads=heads)
        ctx.paged_attn_dev(kvd, batch, H.F32, heads, dim ** -0.5, H.heads(qr), H.heads(att))
        for s in range(3):
            assert L.c2h_quantize_q8k_dev(ctx.h, att[s].data_ptr(), E, aq[s].data_ptr()) == 0
        ctx.sync()
        s64, y = norm_expect(x, before, w.cpu(), 1e-6, H.F32)
        assert torch.equal(resid.cpu(), s64)
        got = qkv.cpu()
        for s in range(3):
            row = O.quantize_row_q8k(y[s].numpy())
            assert np.array_equal(q8k[s].cpu().numpy().ravel(), row)
            want = ctx.gemv(H.Q4_K, raw, row, rows_w, E)
            assert np.array_equal(got[s].numpy().ravel().view(np.uint32), want.view(np.uint32))
        pos = torch.tensor([n - 1 for n in sess.lens])
        # what the cache now holds, by the append's own rule, checked elsewhere
        for i in range(2):
            sess.pools[i] = sess.dev[i].cpu()
        k64, ktol = rotate64(got[:, heads:heads + kv], pos, dim, 1e6, "half")
        for s, n in enumerate(sess.lens):
            at = torch.arange(n)
            for i in range(2):
                c = sess.view(i, bits=True)[sess.table[s].long()[at // page], at % page].contiguous().view(TORCH[cache])
                sc = 1.0 if sess.scale is None else sess.scale[i].double().view(1, -1, 1)
                sess.rows[s][i] = c.double() * sc
            err = (sess.rows[s][0][-1] - k64[s]).abs()
            sc = 1.0 if sess.scale is None else sess.scale[0].double().view(-1, 1)
            if cache != H.F8_E4M3 or (k64[s] / sc).abs().max() < 448:
                assert (err <= ktol[s] * 1.1 + (rounding((k64[s].abs() + ktol[s]) / sc, cache) * sc) * 1.0001).all()
        want, tol = attention64(sess, qr.cpu(), dim ** -0.5, 0, H.F32)
        assert ((att.cpu().double() - want).abs() <= tol).all()
        for s in range(3):
            assert np.array_equal(aq[s].cpu().numpy().ravel(), O.quantize_row_q8k(att[s].cpu().numpy().ravel()))


def test_batch_of_empty_sessions_without_pages(ctx):
    # no session holds a position: a table of no columns, rows of zeros,
    # queries left as they were; a length that is not 0 is reported
    sess = Sessions([4], 2, 64, 16, "nhd", H.BF16, 1)
    kv, _ = sess.cuda()
    before = [d.clone() for d in sess.dev]
    table = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    x = torch.randn(3, 4, 64, device="cuda")
    for lens, bad in (([0, 0, 0], []), ([0, 5, -1], [1, 2])):
        lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
        out, qo = torch.full_like(x, 5.0), torch.full_like(x, 5.0)
        batch = H.paged_batch(table, lens_d, 0)
        torch.cuda.synchronize()
        ctx.paged_append_dev(kv, batch, H.F32, 3, H.heads(x[:, :2]), H.heads(x[:, 2:]), q=H.heads(x), q_out=H.heads(qo), n_heads=4)
        ctx.paged_attn_dev(kv, batch, H.F32, 4, 0.125, H.heads(x), H.heads(out))
        if bad:
            with pytest.raises(H.C2hError, match="length"):
                ctx.sync()
        else:
            ctx.sync()
        assert (qo == 5.0).all()
        for s in range(3):
            assert torch.isnan(out[s]).all() if s in bad else (out[s] == 0.0).all()
    assert all(torch.equal(Sessions.bits(d), Sessions.bits(b)) for d, b in zip(sess.dev, before))
