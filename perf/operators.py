"""What the operators for serving many sessions are measured on: calls of

  c2h_rope_dev          rotary positions of queries or keys
  c2h_paged_append_dev  a step's (or prompts') keys and values into a paged
                        cache, rotated on the way, the queries with them
  c2h_paged_attn_dev    one new token per session over that cache
  c2h_rmsnorm_q8k_dev   residual addition, RMSNorm and Q8_K rows

over the head layouts and widths of the models this package knows (14/2 heads
of 64; 12/2, 16/8 and 16/2 heads of 128; rows of 896, 1,536, 2,048) and
generic ones, from one session's step to batches of long sessions.

run() computes the operators in elementary torch operations in 32 bits
(angles and squared sums in 64) where `own` is false, and calls the package
where it is true.  exact() is each operator's definition in 64 bits.

The package's calls run on the context's stream, which torch's streams do not
wait for.  prepare() returns once the inputs are complete, and run() queues its
call as a layer of a decode step does, without a wait: who uses its outputs
waits first, for the device (torch.cuda.synchronize()) or for the context
(sync(), which also reports a page or length out of range).
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
EPS = 1e-6


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One session's next token: its queries, plain rotation.
        dict(name="rope-1", kind="rope", type="f32", tokens=1, heads=14, dim=64, rot=64, layout="half", base=1e6,
             scaled="none", at=40),
        # A long document's queries far behind the trained context.
        dict(name="rope-prompt-16384", kind="rope", type="bf16", tokens=16384, heads=32, dim=128, rot=128,
             layout="interleaved", base=1e6, scaled="yarn", at=300000),
        # One session's next token into its f32 cache, as a decode step has it.
        dict(name="append-step-1", kind="append", type="f32", cache="f32", heads=14, kv=2, dim=64, page=16,
             order="hnd", seqs=1, lo=40, hi=40, new=1, mix=1, rot=64, layout="half", base=1e6, scaled="none"),
        # A step of a batch of sessions, each at a position of its own.
        dict(name="append-step-256", kind="append", type="bf16", cache="bf16", heads=16, kv=8, dim=128, page=16,
             order="nhd", seqs=256, lo=20, hi=500, new=1, mix=2, rot=128, layout="half", base=1e6, scaled="none"),
        # Prompts of several sessions at once, into an 8-bit cache; only part
        # of the head turns.
        dict(name="append-prompts", kind="append", type="bf16", cache="e4m3", heads=16, kv=2, dim=128, page=64,
             order="hnd", seqs=5, lo=900, hi=4001, new=4001, mix=3, rot=64, layout="half", base=1e6, scaled="linear"),
        # The headline decode workload's attention: one session, short.
        dict(name="attn-1x41", kind="attn", type="f32", cache="f32", heads=14, kv=2, dim=64, page=16, order="hnd",
             seqs=1, lo=41, hi=41, empty=0, window=0, mix=4),
        # One session of a few thousand positions: few rows, a long axis.
        dict(name="attn-1x4096", kind="attn", type="bf16", cache="bf16", heads=16, kv=8, dim=128, page=16,
             order="nhd", seqs=1, lo=4096, hi=4096, empty=0, window=0, mix=5),
        # A serving batch: 64 rows, lengths from tens to thousands, the last
        # rows of the batch without a session.
        dict(name="attn-64-ragged", kind="attn", type="bf16", cache="bf16", heads=12, kv=2, dim=128, page=16,
             order="nhd", seqs=64, lo=30, hi=8000, empty=3, window=0, mix=6),
        # Eight long sessions with f32 activations.
        dict(name="attn-8x32768", kind="attn", type="f32", cache="f16", heads=16, kv=8, dim=128, page=64,
             order="hnd", seqs=8, lo=32000, hi=32768, empty=0, window=0, mix=7),
        # A large batch over an 8-bit cache; attention looks back 4,096.
        dict(name="attn-128-e4m3", kind="attn", type="bf16", cache="e4m3", heads=16, kv=2, dim=128, page=32,
             order="hnd", seqs=128, lo=500, hi=16000, empty=0, window=4096, mix=8),
        # The norm before a decode step's projections.
        dict(name="norm-1x896", kind="norm", type="f32", rows=1, cols=896, add=True, y=False),
        # The same for the rows of a prompt batch, both forms of its output.
        dict(name="norm-8192x2048", kind="norm", type="bf16", rows=8192, cols=2048, add=True, y=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(14, 2, 64), (12, 2, 128), (16, 8, 128), (16, 2, 128), (8, 8, 64), (32, 8, 128), (24, 1, 128), (10, 5, 80),
         (6, 2, 96), (40, 2, 64), (8, 4, 256)]


def _draw_rope(rng, dim):
    return dict(rot=rng.choice([dim, dim, dim // 2, dim - 16]), layout=rng.choice(["half", "interleaved"]),
                base=rng.choice([1e4, 5e5, 1e6]), scaled=rng.choice(["none", "linear", "yarn", "factors"]))


def draw(rng):
    kind = rng.choice(["rope", "append", "attn", "attn", "norm"])
    ty = rng.choice(["f32", "f16", "bf16"])
    heads, kv, dim = rng.choice(HEADS)
    if kind == "rope":
        return dict(kind="rope", type=ty, tokens=_log(rng, 1, min(8192, 32000000 // (heads * dim))), heads=heads, dim=dim,
                    at=_log(rng, 1, 1000000), **_draw_rope(rng, dim))
    if kind == "norm":
        cols = rng.choice([896, 1536, 2048, _log(rng, 256, 8960)])
        return dict(kind="norm", type=ty, rows=_log(rng, 1, min(8192, 8000000 // cols)), cols=cols, add=rng.random() < 0.7,
                    y=rng.random() < 0.5)
    c = dict(kind=kind, type=ty, cache=rng.choice(["f32", "f16", "bf16", "e4m3"]), heads=heads, kv=kv, dim=dim,
             page=rng.choice([8, 16, 16, 32, 64, 128, 256]), order=rng.choice(["nhd", "hnd"]), mix=rng.randrange(1 << 20))
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, 2000)])
        seqs = _log(rng, 1, 256 if new == 1 else max(1, 4000 // new))
        return dict(c, seqs=seqs, lo=new, hi=new + _log(rng, 1, 400), new=new, **_draw_rope(rng, dim))
    hi = _log(rng, 1, 30000)
    most = 500000000 // (hi * kv * dim * 2 * SIZE[c["cache"]])
    return dict(c, seqs=_log(rng, 1, max(1, min(200, most))), lo=max(1, hi // rng.choice([1, 2, 100])), hi=hi,
                empty=rng.choice([0, 0, 1]), window=rng.choice([0, 0, 0, _log(rng, 1, 5000)]))


def _lengths(case):
    """Positions that each session holds (after the append): spread over the
    logarithm of the range, the first the longest."""
    rng = random.Random(case["mix"])
    n = [case["hi"]] + [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]
    e = min(case.get("empty", 0), case["seqs"] - 1)
    return n[:len(n) - e] + [0] * e


def _new(case, lens):
    """New tokens of each session: one in a step, else most of a prompt."""
    rng = random.Random(case["mix"] + 1)
    return [min(n, max(1, round(case["new"] * rng.uniform(0.5, 1.0)))) if case["new"] > 1 else 1 for n in lens]


# ------------------------------------------------------------- rotary positions

FACTOR, ORIG, FAST, SLOW = 8.0, 32768, 32.0, 1.0  # scaled forms: 8 times the trained context


def _mscale(case):
    return 0.1 * math.log(FACTOR) + 1.0 if case["scaled"] == "yarn" else 1.0


def _factors(case):
    """Divisors of the frequencies, as a checkpoint ships them."""
    return np.linspace(1.0, FACTOR, case["rot"] // 2).astype(np.float32)


def _frequencies(case):
    """Radians per position of each pair."""
    i = np.arange(case["rot"] // 2, dtype=np.float64)
    f = case["base"] ** (-2.0 * i / case["rot"])
    if case["scaled"] == "linear":
        return f / FACTOR
    if case["scaled"] == "factors":
        return f / _factors(case).astype(np.float64)
    if case["scaled"] == "yarn":
        def corner(turns):
            return case["rot"] * math.log(ORIG / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))
        lo, hi = max(math.floor(corner(FAST)), 0), min(math.ceil(corner(SLOW)), case["rot"] - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f * (1.0 - ramp) + f / FACTOR * ramp
    return f


def _rotate(x, pos, freq, case):
    """x [tokens, heads, dim] in 32 bits."""
    a = pos.double().unsqueeze(1) * freq
    c = (a.cos() * _mscale(case)).float().unsqueeze(1)
    s = (a.sin() * _mscale(case)).float().unsqueeze(1)
    r, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["layout"] == "half":
        u, v = r.chunk(2, -1)
        return torch.cat([u * c - v * s, u * s + v * c, rest], -1)
    u, v = r[..., 0::2], r[..., 1::2]
    return torch.cat([torch.stack([u * c - v * s, u * s + v * c], -1).flatten(-2), rest], -1)


# ------------------------------------------------------------- prepare

_context = None


def _ctx():
    """The one context such a program keeps."""
    global _context
    from c2slm_amd import _lib as H
    if _context is None:
        _context = H.Ctx()
    return H, _context


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, ty):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[ty])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rope_of(H, case):
    return H.rope(case["rot"], case["base"], layout=case["layout"],
                  factor=FACTOR if case["scaled"] in ("linear", "yarn") else 1.0,
                  orig_ctx=ORIG if case["scaled"] == "yarn" else 0, beta_fast=FAST, beta_slow=SLOW,
                  mscale=_mscale(case), freq_factors=_factors(case) if case["scaled"] == "factors" else None)


def _cache(case, g, pages):
    """One pool, K or V: pages that sessions wrote and left."""
    kv, dim, page = case["kv"], case["dim"], case["page"]
    shape = (pages, page, kv, dim) if case["order"] == "nhd" else (pages, kv, page, dim)
    if case["cache"] != "e4m3":
        return torch.randn(shape, generator=g, device="cuda", dtype=TYPES[case["cache"]])
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * 16).to(TYPES["e4m3"])


def _tokens_first(cache, case):
    """[pages, page, kv, dim] whichever order the pool has."""
    return cache if case["order"] == "nhd" else cache.transpose(1, 2)


def _paged(case, seed, lens):
    g = _gen(seed)
    page = case["page"]
    need = [-(-n // page) for n in lens]
    width, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros((len(lens), width), dtype=torch.int32)
    at = np.cumsum([0] + need)
    order = order.cpu()
    for s, n in enumerate(need):
        table[s, :n] = order[at[s]:at[s + 1]]
    e4 = case["cache"] == "e4m3"
    k, v = _cache(case, g, pages), _cache(case, g, pages)
    # e4m3: values of order one are stored as 16 times themselves, more or less by head
    scale = (torch.rand(2, case["kv"], generator=g, device="cuda") + 0.5) / 16 if e4 else None
    return dict(case=case, g=g, k=k, v=v, ks=scale[0] if e4 else None, vs=scale[1] if e4 else None, table=table.cuda(),
                lens=_ints(lens), longest=max(lens))


def _handles(st):
    """What the package's calls take: the cache and the batch as it describes them."""
    H, ctx = _ctx()
    case = st["case"]
    st.update(ctx=ctx, kv=H.paged_kv(st["k"], st["v"], _code(H, case["cache"]), order=case["order"], k_scale=st["ks"],
                                     v_scale=st["vs"]),
              batch=H.paged_batch(st["table"], st["lens"], st["longest"]), code=_code(H, case["type"]))


def _code(H, ty):
    return {"f32": H.F32, "f16": H.F16, "bf16": H.BF16, "e4m3": H.F8_E4M3}[ty]


def prepare(case, seed):
    st = _prepared(case, seed)
    if own:
        torch.cuda.synchronize()  # the context's stream reads what torch's wrote
    return st


def _prepared(case, seed):
    kind = case["kind"]
    if kind == "rope":
        g, n = _gen(seed), case["tokens"]
        x = _randn(g, (n, case["heads"], case["dim"]), case["type"])
        # a prompt's consecutive positions from `at`; a step's one
        pos = torch.arange(case["at"], case["at"] + n, device="cuda", dtype=torch.int32)
        st = dict(case=case, x=x, pos=pos, out=torch.zeros_like(x), freq=torch.from_numpy(_frequencies(case)).cuda())
        if own:
            H, ctx = _ctx()
            st.update(ctx=ctx, rope=_rope_of(H, case), code=_code(H, case["type"]), xh=H.heads(x), oh=H.heads(st["out"]))
        return st
    if kind == "norm":
        g, n, cols = _gen(seed), case["rows"], case["cols"]
        nb = cols // 256
        x = _randn(g, (n, cols), case["type"])
        r = _randn(g, (n, cols), case["type"]) * 4 if case["add"] else None
        st = dict(case=case, x=x, r=r, w=torch.rand(cols, generator=g, device="cuda") + 0.5,
                  sum=torch.zeros_like(x) if case["add"] else None,
                  y=torch.zeros((n, cols), device="cuda") if case["y"] else None,
                  q8k=torch.zeros((n, nb, 292), dtype=torch.uint8, device="cuda"))
        if own:
            H, ctx = _ctx()
            st.update(ctx=ctx, code=_code(H, case["type"]))
        return st
    lens = _lengths(case)
    st = _paged(case, seed, lens)
    if kind == "append":
        new = _new(case, lens)
        n, start = sum(new), np.cumsum([0] + new)
        # q, k and v are parts of one projection's rows
        rows = _randn(st["g"], (n, case["heads"] + 2 * case["kv"], case["dim"]), case["type"])
        st.update(q=rows[:, :case["heads"]], kn=rows[:, case["heads"]:-case["kv"]], vn=rows[:, -case["kv"]:], n=n,
                  start=_ints(start) if case["new"] > 1 else None, freq=torch.from_numpy(_frequencies(case)).cuda(),
                  qo=torch.zeros((n, case["heads"], case["dim"]), dtype=TYPES[case["type"]], device="cuda"))
        if own:
            H, _ = _ctx()
            _handles(st)
            st.update(rope=_rope_of(H, case), qh=H.heads(st["q"]), kh=H.heads(st["kn"]), vh=H.heads(st["vn"]),
                      oh=H.heads(st["qo"]))
        return st
    st.update(q=_randn(st["g"], (len(lens), case["heads"], case["dim"]), case["type"]))
    st["out"] = torch.zeros_like(st["q"])
    if own:
        H, _ = _ctx()
        _handles(st)
        st.update(qh=H.heads(st["q"]), oh=H.heads(st["out"]))
    return st


# ------------------------------------------------------------- run

def _run_rope(st):
    case = st["case"]
    if own:
        st["ctx"].rope_dev(st["rope"], st["code"], st["xh"], st["pos"], case["tokens"], case["heads"], case["dim"], st["oh"])
    else:
        st["out"].copy_(_rotate(st["x"].float(), st["pos"], st["freq"], case))
    return st["out"]


def _store(cache, scale, page, at, rows, case):
    """rows [tokens, kv, dim] in 32 bits to their places."""
    if scale is None:
        _tokens_first(cache, case)[page, at] = rows.to(cache.dtype)
        return
    rows = (rows / scale.unsqueeze(1)).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
    _tokens_first(cache, case).view(torch.uint8)[page, at] = rows.view(torch.uint8)


def _run_append(st):
    case = st["case"]
    if own:
        st["ctx"].paged_append_dev(st["kv"], st["batch"], st["code"], st["n"], st["kh"], st["vh"], token_start=st["start"],
                                   rope=st["rope"], q=st["qh"], q_out=st["oh"], n_heads=case["heads"])
    else:
        i = torch.arange(st["n"], device="cuda")
        if st["start"] is None:
            seq, pos = i, st["lens"].long() - 1
        else:
            start = st["start"].long()
            seq = torch.searchsorted(start, i, right=True) - 1
            pos = st["lens"].long()[seq] - (start[seq + 1] - i)
        page, at = st["table"][seq, pos // case["page"]].long(), pos % case["page"]
        _store(st["k"], st["ks"], page, at, _rotate(st["kn"].float(), pos, st["freq"], case), case)
        _store(st["v"], st["vs"], page, at, st["vn"].float(), case)
        st["qo"].copy_(_rotate(st["q"].float(), pos, st["freq"], case))
    return dict(k=st["k"], v=st["v"], q=st["qo"])


def _gathered(cache, scale, st):
    """[sessions, kv, positions, dim] in 32 bits."""
    case = st["case"]
    c = _tokens_first(cache.view(torch.uint8) if scale is not None else cache, case)[st["table"].long()]
    c = c.flatten(1, 2).transpose(1, 2)
    if scale is None:
        return c.float()
    return c.contiguous().view(cache.dtype).float() * scale.view(-1, 1, 1)


def _run_attn(st):
    case = st["case"]
    if own:
        st["ctx"].paged_attn_dev(st["kv"], st["batch"], st["code"], case["heads"], case["dim"] ** -0.5, st["qh"], st["oh"],
                                 window=case["window"])
        return st["out"]
    k, v = _gathered(st["k"], st["ks"], st), _gathered(st["v"], st["vs"], st)
    q = st["q"].float().unflatten(1, (case["kv"], -1))
    lens = st["lens"].view(-1, 1, 1, 1)
    at = torch.arange(k.shape[2], device="cuda")
    out_of = (at >= lens) | (at < lens - (case["window"] or 1 << 30))
    s = (torch.matmul(q, k.transpose(2, 3)) * case["dim"] ** -0.5).masked_fill(out_of, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(lens > 0, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(lens > 0, total, torch.ones_like(total))
    st["out"].copy_(o.flatten(1, 2))
    return st["out"]


def _q8k_parts(q8k):
    """Scales, quants and sums of 16 of the 292-byte blocks."""
    return q8k.view(torch.float32)[..., 0], q8k[..., 4:260].view(torch.int8), q8k[..., 260:].view(torch.int16)


def _run_norm(st):
    case = st["case"]
    d, q, sums = _q8k_parts(st["q8k"])
    out = dict(d=d, q=q, sums=sums)
    if case["add"]:
        out["sum"] = st["sum"]
    if case["y"]:
        out["y"] = st["y"]
    if own:
        st["ctx"].rmsnorm_q8k_dev(st["code"], st["x"], st["w"], EPS, st["q8k"], residual=st["r"], sum_out=st["sum"],
                                  y=st["y"])
        return out
    x = st["x"]
    if case["add"]:
        x = st["sum"].copy_(x.float() + st["r"].float())
    x = x.float()
    scale = (x.double().square().mean(-1, keepdim=True) + float(np.float32(EPS))).rsqrt().float()
    y = x * scale * st["w"]
    b = y[:, :case["cols"] // 256 * 256].unflatten(1, (-1, 256))
    top = b.abs().amax(-1, keepdim=True)
    full = torch.full_like(top, 127.0)
    d.copy_((top / full).squeeze(-1))
    t = b * torch.where(top > 0, full / top, torch.zeros_like(top))
    quants = torch.trunc(t + torch.copysign(torch.full_like(t, 0.5), t)).clamp(-127, 127)
    q.copy_(quants)
    sums.copy_(quants.unflatten(-1, (16, 16)).sum(-1))
    if case["y"]:
        st["y"].copy_(y)
    return out


def run(state):
    return {"rope": _run_rope, "append": _run_append, "attn": _run_attn, "norm": _run_norm}[state["case"]["kind"]](state)


# ------------------------------------------------------------- work

def work(case):
    size = SIZE[case["type"]]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"]
        return dict(bytes=2 * n * case["dim"] * size + 4 * case["tokens"], flops=3 * n * case["rot"])
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        b = n * size * (3 if case["add"] else 1) + (4 * n if case["y"] else 0)
        return dict(bytes=b + case["rows"] * (case["cols"] // 256) * 292 + 4 * case["cols"], flops=8 * n)
    lens, row = _lengths(case), case["kv"] * case["dim"]
    if case["kind"] == "append":
        n = sum(_new(case, lens))
        b = n * (2 * row * (size + SIZE[case["cache"]]) + 2 * case["heads"] * case["dim"] * size)
        return dict(bytes=b + 8 * len(lens), flops=3 * n * (case["heads"] + case["kv"]) * case["rot"])
    held = sum(min(n, case["window"] or n) for n in lens)
    b = held * 2 * row * SIZE[case["cache"]] + 2 * len(lens) * case["heads"] * case["dim"] * size
    return dict(bytes=b + 4 * held // case["page"] + 4 * len(lens), flops=4 * held * case["heads"] * case["dim"])


# ------------------------------------------------------------- in 64 bits

def _exact_rotation(x, pos, case):
    """x [tokens, heads, dim], pos [tokens], in 64 bits: pair i of a head
    turned as a complex number."""
    rot, f = case["rot"], []
    for i in range(case["rot"] // 2):
        w = math.exp(-2.0 * i / rot * math.log(case["base"]))
        if case["scaled"] == "linear":
            w /= FACTOR
        elif case["scaled"] == "factors":
            w /= float(_factors(case)[i])
        elif case["scaled"] == "yarn":
            ends = [rot / 2 * math.log(ORIG / (2 * math.pi * t)) / math.log(case["base"]) for t in (FAST, SLOW)]
            lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rot - 1)
            share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w * (1 - share) + w / FACTOR * share
        f.append(w)
    a = torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(a, _mscale(case)), a).unsqueeze(1)
    x = x.double().clone()
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., one], x[..., two]) * turn
    x[..., one], x[..., two] = z.real, z.imag
    return x


def _exact_append(st, lens):
    case = st["case"]
    k, v = (_tokens_first(t.double(), case) for t in (st["k"], st["v"]))
    new, at = _new(case, lens), 0
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, (n, length) in enumerate(zip(new, lens)):
        pos = torch.arange(length - n, length, device="cuda")
        rows = slice(at, at + n)
        at += n
        page, off = st["table"][s].long()[pos // case["page"]], pos % case["page"]
        kr, vr = _exact_rotation(st["kn"][rows], pos, case), st["vn"][rows].double()
        if st["ks"] is not None:
            kr, vr = ((r / t.double().view(-1, 1)).clamp(-E4M3_MAX, E4M3_MAX) for r, t in ((kr, st["ks"]), (vr, st["vs"])))
        k[page, off], v[page, off] = kr, vr
        q[rows] = _exact_rotation(st["q"][rows], pos, case)
    return dict(k=_tokens_first(k, case), v=_tokens_first(v, case), q=q)


def _exact_attn(st, lens):
    case = st["case"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv"]
    for s, n in enumerate(lens):
        lo = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        pos = torch.arange(lo, n, device="cuda")
        page, at = st["table"][s].long()[pos // case["page"]], pos % case["page"]
        for h in range(case["kv"]):
            kv = []
            for cache, scale in ((st["k"], st["ks"]), (st["v"], st["vs"])):
                c = _tokens_first(cache.view(torch.uint8) if scale is not None else cache, case)[page, at, h]
                kv.append(c.double() if scale is None else c.view(cache.dtype).double() * scale[h].double())
            q = st["q"][s, h * group:(h + 1) * group].double()
            p = torch.softmax(q @ kv[0].t().contiguous() / math.sqrt(case["dim"]), -1)
            out[s, h * group:(h + 1) * group] = p @ kv[1]
    return out


def _exact_norm(st):
    case = st["case"]
    x = st["x"].double()
    out = dict(sums=None, q=None)
    if case["add"]:
        # the sum is held in the inputs' type: what the norm sees is that
        out["sum"] = x + st["r"].double()
        x = out["sum"].to(TYPES[case["type"]]).double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["cols"] + float(np.float32(EPS))) * st["w"].double()
    if case["y"]:
        out["y"] = y
    out["d"] = y[:, :case["cols"] // 256 * 256].reshape(case["rows"], -1, 256).abs().amax(-1) / 127
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rotation(st["x"], st["pos"], case)
    if case["kind"] == "norm":
        return _exact_norm(st)
    return (_exact_append if case["kind"] == "append" else _exact_attn)(st, _lengths(case))
