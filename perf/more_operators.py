"""Timed cases of the cached-attention operators: appending a recording's new windows to a paged cache of keys and values with
the position rotation on the way, attention of the new windows over that cache, and attention over the pages that a bound on
their scores selects.

A case is a dict of plain values. `run` computes an operator in plain torch, or, where `own` is set, through the
kernel-level ABI (include/bnneon_hip.h) on device buffers, as a host that keeps its activations on the GPU calls it.
Everything depends on the seed alone.
"""
import functools
import math
import os
import sys

import torch

own = False
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@functools.cache
def _hip():
    sys.path.insert(0, os.path.join(ROOT, "birdnet-neon-engine_amd"))
    from bnneon import hip
    return hip


# ------------------------------------------------------------------------------------------------ the list
# windows: sequences (stations) of a call; rows: the longest one's new windows; past: the most windows in a sequence's cache
# ahead of them (ragged: sequences of unequal rows and pasts); page: windows to a page
def listed():
    return [
        # one live station's new window goes into the cache of its hour: a launch
        dict(name="append_live_one", op="append", windows=1, rows=1, past=719, ragged=False, heads=12, kv_heads=12, dk=128,
             dv=128, page=64, rd=128, pairs=False, gaps=False, bounds=False, f16=True),
        # the new windows of 64 live stations on duty cycles (positions with gaps), with the pages' bounds
        dict(name="append_live", op="append", windows=64, rows=1, past=720, ragged=True, heads=12, kv_heads=4, dk=128,
             dv=128, page=64, rd=128, pairs=False, gaps=True, bounds=True, f16=True),
        # an archive: up to an hour of 5 s windows of 24 stations
        dict(name="append_archive", op="append", windows=24, rows=720, past=720, ragged=True, heads=12, kv_heads=12, dk=128,
             dv=128, page=64, rd=128, pairs=False, gaps=False, bounds=True, f16=True),
        # fp32, odd widths, neighbouring values as pairs, a part of each head rotated
        dict(name="append_f32", op="append", windows=8, rows=500, past=300, ragged=True, heads=16, kv_heads=4, dk=70, dv=97,
             page=16, rd=42, pairs=True, gaps=True, bounds=True, f16=False),
        # one live station looks back over its day of 5 s windows
        dict(name="attn_live_one", op="attn", windows=1, rows=1, past=17279, ragged=False, heads=12, kv_heads=12, dk=128,
             dv=128, page=64, window=0, f16=True),
        # 64 live stations over up to a day, keys and values shared by three heads
        dict(name="attn_live", op="attn", windows=64, rows=1, past=17279, ragged=True, heads=12, kv_heads=4, dk=128, dv=128,
             page=64, window=0, f16=True),
        # ten minutes of new windows of 24 stations over what their caches hold, small pages
        dict(name="attn_chunks", op="attn", windows=24, rows=120, past=5000, ragged=True, heads=12, kv_heads=4, dk=128,
             dv=128, page=16, window=0, f16=True),
        # a day of one station from an empty cache
        dict(name="attn_day", op="attn", windows=1, rows=17280, past=0, ragged=False, heads=12, kv_heads=12, dk=128, dv=128,
             page=64, window=0, f16=True),
        # all in fp32, odd widths, each window over the 256 up to it
        dict(name="attn_f32", op="attn", windows=8, rows=250, past=900, ragged=True, heads=16, kv_heads=4, dk=64, dv=97,
             page=16, window=256, f16=False),
        # one live station over a week of 5 s windows: 32 pages of it
        dict(name="sparse_live_one", op="sparse", windows=1, rows=1, past=120959, ragged=False, heads=12, kv_heads=4, dk=128,
             dv=128, page=64, pages=32, f16=True),
        # 16 live stations over up to three days: 16 pages
        dict(name="sparse_live", op="sparse", windows=16, rows=1, past=51839, ragged=True, heads=12, kv_heads=4, dk=128,
             dv=128, page=64, pages=16, f16=True),
        # a minute or two of new windows of a few stations, in fp32
        dict(name="sparse_chunk_f32", op="sparse", windows=6, rows=24, past=6000, ragged=True, heads=8, kv_heads=2, dk=72,
             dv=88, page=32, pages=12, f16=False),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "sparse"])
    f16 = rng.random() < 0.7
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 2, 3, 4] if kv <= 4 else [1, 2])
    dk, dv = _log(rng, 24, 256), _log(rng, 24, 256)
    if rng.random() < 0.6:
        dk, dv = (dk + 15) // 16 * 16, (dv + 15) // 16 * 16
    page = rng.choice([16, 32, 64, 128])
    b = _log(rng, 1, 64)
    c = dict(op=op, windows=b, heads=heads, kv_heads=kv, dk=dk, dv=dv, page=page, f16=f16)
    if op == "append":
        most = 24 * 720 * 12 * 384 // (heads * dk + kv * (dk + dv))
        rows = min(_log(rng, 1, max(1, most // b)), 17280)
        rd = dk // 2 * 2 if rng.random() < 0.5 else 2 * rng.randint(0, dk // 2)
        c.update(rows=rows, past=rng.randint(0, 720), rd=rd, pairs=rng.random() < 0.3, gaps=rng.random() < 0.5,
                 bounds=rng.random() < 0.6)
    elif op == "attn":
        # score entries times widths of a day from an empty cache at 16-bit rates; fp32 products take 16 times as long
        most = 17280 * 17280 * 12 * 128 // (1 if f16 else 16) // (heads * (dk + dv))
        past = min(_log(rng, 1, 17280), (2 << 30) // (b * kv * (dk + dv) * (2 if f16 else 4))) - 1
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        while rows > 1 and b * rows * (past + rows) > min(most, (4 << 30) // heads):
            rows = rows * 2 // 3
        c.update(rows=rows, past=past, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))
    else:
        past = _log(rng, 500, 120000)
        while b * (past + 64) * kv * (dk + dv) * (2 if f16 else 4) > (2 << 30):
            past = past * 2 // 3
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(64, 320 // b)))
        c.update(rows=rows, past=past, pages=_log(rng, 3, max(3, 2048 // page)))
    c["ragged"] = b > 1 and rng.random() < 0.6
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lens(c):
    """New rows of each sequence, from 1 to the longest: plain numbers of the case alone (a program knows its lengths)."""
    b, t = c["windows"], c["rows"]
    return [t if not c["ragged"] or i == 0 else 1 + (i * 7919 * 31) % t for i in range(b)]


def _pasts(c):
    b, n = c["windows"], c["past"]
    return [n if not c["ragged"] or i == 0 else (i * 104729 * 17) % (n + 1) for i in range(b)]


#: pages that each selection starts with and ends with, beside those that the bounds choose
FIRST, LAST = 1, 2


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, dict(c=case)
    b, p, h, hk, dk, dv = c["windows"], c["page"], c["heads"], c["kv_heads"], c["dk"], c["dv"]
    t = torch.float16 if c["f16"] else torch.float32
    lens, pasts = _lens(c), _pasts(c)
    rows = s["rows"] = sum(lens)
    need = [-(-(m + n) // p) for m, n in zip(pasts, lens)]
    pages, ldt = sum(need) + 3, max(need) + 2

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    s["lens"], s["past"], s["start"] = ints(lens), ints(pasts), ints([sum(lens[:i]) for i in range(b)])
    # pages as a pool that has been in use for a while hands them out, -1 where a sequence has no page yet
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((b, ldt), -1, dtype=torch.int32, device="cuda")
    for i in range(b):
        table[i, :need[i]] = order[sum(need[:i]):sum(need[:i + 1])]
    s["table"] = table
    # q, k and v side by side in a projection's rows
    s["qkv"] = normal(rows, h * dk + hk * (dk + dv), std=1.2).to(t)
    s["kc"], s["vc"] = normal(pages, hk, p, dk, dtype=t), normal(pages, hk, p, dv, dtype=t)
    s["lo"] = s["hi"] = None
    if c["op"] == "sparse" or c.get("bounds"):
        # the bounds of the pages' tokens so far: append's first state, or what it has left to the operators that read it
        held = torch.zeros(pages, dtype=torch.int32, device="cuda")
        for i in range(b):
            have = pasts[i] + (lens[i] if c["op"] == "sparse" else 0)
            held[table[i, :need[i]].long()] = (have - p * torch.arange(need[i], device="cuda")).clamp(0, p).int()
        there = (torch.arange(p, device="cuda")[None] < held[:, None])[:, None, :, None]
        s["lo"] = torch.where(there, s["kc"], torch.inf).amin(2)
        s["hi"] = torch.where(there, s["kc"], -torch.inf).amax(2)
    if c["op"] == "append":
        s["freq"] = (10000.0 ** (-2 * torch.arange(c["rd"] // 2, dtype=torch.float64, device="cuda") / max(1, c["rd"]))).float()
        s["pos"] = None
        if c["gaps"]:  # a minute of 5 s windows in every ten
            at = torch.cat([torch.arange(m, m + n) for m, n in zip(pasts, lens)])
            s["pos"] = (at // 12 * 120 + at % 12).int().cuda()
        s["qr"] = torch.empty((rows, h * dk), dtype=t, device="cuda")
    else:
        s["o"] = torch.empty((rows, h * dv), dtype=t, device="cuda")
        s["sel"] = torch.empty((rows, hk, c.get("pages", 0)), dtype=torch.int32, device="cuda") if c["op"] == "sparse" else None
    if own:
        _plan(s)
    return s


# ------------------------------------------------------------------------------------------------ the framework's
def _p(t):
    return None if t is None else t.data_ptr()


def _plan(s):
    """The descriptors and the workspace that a program keeps between calls."""
    hip, c, qkv, es = _hip(), s["c"], s["qkv"], s["qkv"].element_size()
    h, hk, dk, dv, ld = c["heads"], c["kv_heads"], c["dk"], c["dv"], s["qkv"].shape[1]
    cache = hip.KvCache(k=_p(s["kc"]), v=_p(s["vc"]), k_ps=hk * c["page"] * dk, v_ps=hk * c["page"] * dv, f16=c["f16"],
                        pages=s["kc"].shape[0], page=c["page"], Hk=hk, dk=dk, dv=dv, lo=_p(s["lo"]), hi=_p(s["hi"]),
                        table=_p(s["table"]), ldt=s["table"].shape[1], past=_p(s["past"]))
    seqs = (c["rows"], c["windows"], s["rows"], _p(s["start"]), _p(s["lens"]))
    if c["op"] == "append":
        rot = hip.Rotary(rd=c["rd"], pairs=c["pairs"], freq=_p(s["freq"]), pos=_p(s["pos"]))
        s["append"] = (cache, rot, _p(qkv) + es * h * dk, ld, _p(qkv) + es * (h + hk) * dk, ld, _p(qkv), ld, _p(s["qr"]),
                       h * dk, h, *seqs)
        return
    a = hip.KvAttn(q=_p(qkv), ldq=ld, o=_p(s["o"]), ldo=h * dv, H=h, scale=dk ** -0.5, window=c.get("window", 0),
                   sel=_p(s["sel"]), nsel=c.get("pages", 0))
    n = hip.lib().bnh_kv_attn_work_bytes(cache, a, *seqs[:3])
    if c["op"] == "sparse":
        n = max(n, hip.lib().bnh_kv_select_work_bytes(cache, a, *seqs[:3]))
    s["ws"] = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
    s["select"] = (cache, a, FIRST, LAST, *seqs, _p(s["ws"]), n)
    s["attn"] = (cache, a, *seqs, _p(s["ws"]), n)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(hip, s):
    hip.check(hip.lib().bnh_kv_append(*s["append"], _stream()), "kv_append")
    return s["qr"], s["kc"], s["vc"], *([s["lo"], s["hi"]] if s["lo"] is not None else [])


def _own_attn(hip, s):
    hip.check(hip.lib().bnh_kv_attn(*s["attn"], _stream()), "kv_attn")
    return s["o"]


def _own_sparse(hip, s):
    stream = _stream()
    hip.check(hip.lib().bnh_kv_select(*s["select"], stream), "kv_select")
    hip.check(hip.lib().bnh_kv_attn(*s["attn"], stream), "kv_attn")
    return s["sel"], s["o"]


# ------------------------------------------------------------------------------------------------ plain torch
def _tokens(s):
    """Sequence and token of each row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["start"], row.int(), right=True) - 1
    return seq, row - s["start"][seq] + s["past"][seq]


def _rotate(x, cos, sin, rd, pairs):
    """x [rows][heads][dk] in 32 bits, its first rd values rotated."""
    r = x[..., :rd]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :rd // 2], r[..., rd // 2:])
    cos, sin = cos[:, None], sin[:, None]
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([r, x[..., rd:]], -1)


def _plain_append(s):
    c, t = s["c"], s["kc"].dtype
    h, hk, dk, dv, p, rd = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["page"], c["rd"]
    seq, at = _tokens(s)
    angle = (at if s["pos"] is None else s["pos"]).double()[:, None] * s["freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = s["qkv"].float()
    q = _rotate(x[:, :h * dk].reshape(-1, h, dk), cos, sin, rd, c["pairs"])
    k = _rotate(x[:, h * dk:(h + hk) * dk].reshape(-1, hk, dk), cos, sin, rd, c["pairs"])
    page = s["table"][seq, at // p].long()
    s["kc"][page, :, at % p] = k.to(t)
    s["vc"][page, :, at % p] = x[:, (h + hk) * dk:].reshape(-1, hk, dv).to(t)
    s["qr"].copy_(q.reshape(s["rows"], h * dk))
    if s["lo"] is None:
        return s["qr"], s["kc"], s["vc"]
    # the pages that have new tokens, from all that they hold now
    n = (c["rows"] + p - 2) // p + 1
    i = s["past"][:, None] // p + torch.arange(n, device="cuda")
    end = s["past"] + s["lens"]
    at, which = (i * p < end[:, None]).nonzero(as_tuple=True)
    i = i[at, which]
    page = s["table"][at, i].long()
    there = (i[:, None] * p + torch.arange(p, device="cuda") < end[at, None])[:, None, :, None]
    keys = s["kc"][page]
    s["lo"][page] = torch.where(there, keys, torch.inf).amin(2)
    s["hi"][page] = torch.where(there, keys, -torch.inf).amax(2)
    return s["qr"], s["kc"], s["vc"], s["lo"], s["hi"]


def _softmax_product(scores, seen, v):
    """exp(scores - their largest) over what is seen, by v, over their sum; scores are overwritten."""
    scores.masked_fill_(~seen, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -torch.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return torch.matmul(scores, v) / torch.where(total == 0, 1.0, total)


def _plain_attn(s):
    c, b = s["c"], s["c"]["windows"]
    h, hk, dk, dv, p, w = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["page"], c["window"]
    seq, at = _tokens(s)
    most, t = max(m + n for m, n in zip(_pasts(c), _lens(c))), c["rows"]
    j = torch.arange(most, device="cuda")
    page = s["table"][:, j // p].long()  # [b][most], -1 past a sequence's end
    row = (s["start"][:, None] + torch.arange(t, device="cuda")).clamp(max=s["rows"] - 1).long()
    q = s["qkv"][:, :h * dk].float()[row].reshape(b, t, hk, h // hk, dk).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, dk)
    k = s["kc"][page.clamp(min=0), :, j % p].float().permute(0, 2, 3, 1).contiguous()
    v = s["vc"][page.clamp(min=0), :, j % p].float().permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q * dk ** -0.5, k).reshape(b, hk, h // hk, t, most)
    i = (s["past"][:, None] + torch.arange(t, device="cuda"))[:, :, None]
    seen = (j <= i) & (page >= 0)[:, None]
    if w:
        seen &= j > i - w
    o = _softmax_product(scores, seen[:, None, None], v[:, :, None])
    s["o"].copy_(o.permute(0, 3, 1, 2, 4).reshape(b, t, h * dv)[seq, at - s["past"][seq]])
    return s["o"]


def _plain_sparse(s):
    c = s["c"]
    h, hk, dk, dv, p, n, rows = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["page"], c["pages"], s["rows"]
    seq, at = _tokens(s)
    q = s["qkv"][:, :h * dk].reshape(rows, hk, h // hk, dk)
    # each page's bound in 64 bits, where which of two near scores is larger decides
    ids = torch.arange(s["table"].shape[1], device="cuda")
    table = s["table"].long()
    there = (table >= 0)[seq] & (ids * p <= at[:, None])
    lo, hi = (x[table.clamp(min=0)].double().permute(0, 2, 3, 1).contiguous() for x in (s["lo"], s["hi"]))
    lo, hi = (torch.where((table >= 0)[:, None, None], x, 0.0) for x in (lo, hi))
    t = c["rows"]
    row = (s["start"][:, None] + torch.arange(t, device="cuda")).clamp(max=rows - 1).long()
    u = q.double()[row].permute(0, 2, 3, 1, 4).reshape(c["windows"], hk, -1, dk)
    bound = torch.matmul(u.clamp(min=0), hi) + torch.matmul(u.clamp(max=0), lo)
    bound = bound.reshape(c["windows"], hk, h // hk, t, -1).sum(2).permute(0, 2, 1, 3)[seq, at - s["past"][seq]]
    always = (ids < FIRST) | (ids > (at[:, None] // p) - LAST)
    bound = torch.where(always[:, None], torch.inf, bound).masked_fill(~there[:, None], -torch.inf)
    best, which = torch.sort(bound, dim=-1, descending=True, stable=True)
    which = torch.nn.functional.pad(which[..., :n].masked_fill(best[..., :n] == -torch.inf, 1 << 30), (0, max(0, n - len(ids))),
                                    value=1 << 30)
    sel = torch.sort(which, dim=-1)[0]
    sel = torch.where(sel == 1 << 30, -1, sel)
    s["sel"].copy_(sel)
    # its tokens
    j = (sel.clamp(min=0)[..., None] * p + torch.arange(p, device="cuda")).reshape(rows, hk, n * p)
    page = table[seq[:, None, None], sel.clamp(min=0)]
    g = torch.arange(hk, device="cuda")[None, :, None]
    k = s["kc"][page, g].reshape(rows, hk, n * p, dk).float().transpose(-1, -2).contiguous()
    v = s["vc"][page, g].reshape(rows, hk, n * p, dv).float()
    seen = (j <= at[:, None, None]) & (sel >= 0).repeat_interleave(p, -1)
    o = _softmax_product(torch.matmul(q.float() * dk ** -0.5, k), seen[:, :, None], torch.where(seen[..., None], v, 0.0))
    s["o"].copy_(o.reshape(rows, h * dv))
    return s["sel"], s["o"]


_PLAIN = {"append": _plain_append, "attn": _plain_attn, "sparse": _plain_sparse}
_OWN = {"append": _own_append, "attn": _own_attn, "sparse": _own_sparse}


def run(state):
    op = state["c"]["op"]
    return _OWN[op](_hip(), state) if own else _PLAIN[op](state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_append(s):
    c = s["c"]
    h, hk, dk, dv, p, rd = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["page"], c["rd"]
    kc, vc = s["kc"].double(), s["vc"].double()
    x = s["qkv"].double()
    q, k = x[:, :h * dk].reshape(-1, h, dk).clone(), x[:, h * dk:(h + hk) * dk].reshape(-1, hk, dk).clone()
    v = x[:, (h + hk) * dk:].reshape(-1, hk, dv)
    first = [(e, e + rd // 2) if not c["pairs"] else (2 * e, 2 * e + 1) for e in range(rd // 2)]
    at = torch.cat([torch.arange(m, m + n) for m, n in zip(_pasts(c), _lens(c))]).cuda()
    pos = (at if s["pos"] is None else s["pos"]).double()
    for e, (i, j) in enumerate(first):
        turn = torch.polar(torch.ones_like(pos), pos * s["freq"][e].double())[:, None]
        for y in (q, k):
            z = torch.complex(y[..., i].contiguous(), y[..., j].contiguous()) * turn
            y[..., i], y[..., j] = z.real, z.imag
    out, n = [q.reshape(-1, h * dk), kc, vc], 0
    lo, hi = (None, None) if s["lo"] is None else (s["lo"].double(), s["hi"].double())
    for i, (m, r) in enumerate(zip(_pasts(c), _lens(c))):
        page = s["table"][i].long()[at[n:n + r] // p]
        kc[page, :, at[n:n + r] % p] = k[n:n + r]
        vc[page, :, at[n:n + r] % p] = v[n:n + r]
        n += r
        if lo is not None:
            for a in range(m // p, (m + r - 1) // p + 1):
                keys = kc[int(s["table"][i, a]), :, :min(p, m + r - a * p)]
                lo[int(s["table"][i, a])], hi[int(s["table"][i, a])] = keys.amin(1), keys.amax(1)
    return tuple(out + ([] if lo is None else [lo, hi]))


def _rows_of(s, i):
    """A sequence's rows as a slice, and its tokens."""
    n = sum(_lens(s["c"])[:i])
    m, r = _pasts(s["c"])[i], _lens(s["c"])[i]
    return slice(n, n + r), torch.arange(m, m + r, device="cuda")


def _held(s, i, g, end):
    """Keys and values of sequence i and shared head g in 64 bits, in order."""
    p = s["c"]["page"]
    page = s["table"][i, :-(-end // p)].long()
    return (x[page, g].reshape(-1, x.shape[-1])[:end].double() for x in (s["kc"], s["vc"]))


def _exact_attn(s):
    c, dk, dv, group = s["c"], s["c"]["dk"], s["c"]["dv"], s["c"]["heads"] // s["c"]["kv_heads"]
    o = torch.empty((s["rows"], c["heads"], dv), dtype=torch.float64, device="cuda")
    for i in range(c["windows"]):
        row, at = _rows_of(s, i)
        j = torch.arange(int(at[-1]) + 1, device="cuda")
        hidden = (j[None] > at[:, None]) | (j[None] <= at[:, None] - (c["window"] or 1 << 40))
        for g in range(c["kv_heads"]):
            k, v = _held(s, i, g, len(j))
            for head in range(g * group, (g + 1) * group):
                x = s["qkv"][row, head * dk:(head + 1) * dk].double() @ k.t() / math.sqrt(dk)
                x = x.masked_fill_(hidden, -torch.inf)
                x = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                o[row, head] = x @ v
    return o.reshape(s["rows"], -1)


def _exact_sparse(s):
    c = s["c"]
    dk, dv, p, n, group = c["dk"], c["dv"], c["page"], c["pages"], c["heads"] // c["kv_heads"]
    sel = torch.full((s["rows"], c["kv_heads"], n), -1, dtype=torch.int32, device="cuda")
    o = torch.empty((s["rows"], c["heads"], dv), dtype=torch.float64, device="cuda")
    for i in range(c["windows"]):
        row, at = _rows_of(s, i)
        for g in range(c["kv_heads"]):
            k, v = _held(s, i, g, int(at[-1]) + 1)
            for r, t in zip(range(row.start, row.stop), at.tolist()):
                q = s["qkv"][r].double()[g * group * dk:(g + 1) * group * dk].reshape(group, dk)
                have = t // p + 1
                page = s["table"][i, :have].long()
                corner = torch.where(q[:, None] >= 0, s["hi"][page, g].double(), s["lo"][page, g].double())
                score = (q[:, None] * corner).sum((0, 2))
                score[:FIRST] = score[max(0, have - LAST):] = torch.inf
                mine = torch.argsort(score, descending=True, stable=True)[:n].sort()[0]
                sel[r, g, :len(mine)] = mine.int()
                j = (mine[:, None] * p + torch.arange(p, device="cuda")).flatten()
                j = j[j <= t]
                x = torch.softmax(q @ k[j].t() / math.sqrt(dk), -1)
                o[r, g * group:(g + 1) * group] = x @ v[j]
    return sel, o.reshape(s["rows"], -1)


def exact(case, seed):
    c = case
    if c["op"] == "attn":
        if sum(n * (m + n) for m, n in zip(_pasts(c), _lens(c))) * c["heads"] * (c["dk"] + c["dv"] + 100) * 1e-13 > 5:
            return None
    if c["windows"] * c["kv_heads"] * (sum(_lens(c)) / c["windows"] if c["op"] == "sparse" else 5) > 12000:
        return None
    return {"append": _exact_append, "attn": _exact_attn, "sparse": _exact_sparse}[c["op"]](prepare(case, seed))


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    h, hk, dk, dv, p, es = c["heads"], c["kv_heads"], c["dk"], c["dv"], c["page"], 2 if c["f16"] else 4
    lens, pasts = _lens(c), _pasts(c)
    rows, held = sum(lens), sum(lens) + sum(pasts)
    if c["op"] == "append":
        pages = sum((m + n - 1) // p - m // p + 1 for m, n in zip(pasts, lens)) if c["bounds"] else 0
        return dict(bytes=es * (2 * rows * (h * dk + hk * (dk + dv)) + 2 * pages * hk * dk), flops=6 * rows * (h + hk) * c["rd"])
    inout = es * rows * h * (dk + dv)
    if c["op"] == "attn":
        w = c["window"] or 1 << 40

        def sees(m, n):  # tokens that n rows after m see, all together, and the tokens that any of them sees
            full = min(n, max(0, w - m - 1))  # rows that see all up to them
            return full * m + full * (full + 1) // 2 + (n - full) * min(w, m + n), min(m + n, w + n - 1)

        pairs, seen = map(sum, zip(*(sees(m, n) for m, n in zip(pasts, lens))))
        return dict(bytes=inout + es * hk * (dk + dv) * seen, flops=2 * pairs * h * (dk + dv))
    n = c["pages"]
    pages = sum(-(-(m + r) // p) for m, r in zip(pasts, lens))
    scored = sum(r * (m + r) // p for m, r in zip(pasts, lens))
    taken = sum(r * min(n * p, m + r) for m, r in zip(pasts, lens))
    read = sum(min(r * n * p, m + r) for m, r in zip(pasts, lens))
    return dict(bytes=inout + 4 * rows * hk * n + 2 * es * pages * hk * dk + es * hk * (dk + dv) * read,
                flops=2 * scored * h * dk + 2 * taken * h * (dk + dv))
