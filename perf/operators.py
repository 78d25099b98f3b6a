"""Timed cases of the temporal context operators: the norms around a block, a projection with the adapters of many
stations beside it, and linear attention with a decay for each head, as they run over the embeddings of a recording's
windows.

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
KIND = {"none": 0, "rms": 1, "layer": 2}
ACT = {"none": 0, "silu": 1, "relu": 2, "sigmoid": 3}
EPS = 1e-5


@functools.cache
def _hip():
    sys.path.insert(0, os.path.join(ROOT, "birdnet-neon-engine_amd"))
    from bnneon import hip
    return hip


# ------------------------------------------------------------------------------------------------ the list
def listed():
    return [
        # 24 live stations have one new 5 s window each: the exit of one block and the entry of the next, where a
        # launch counts (Perch-shaped embeddings, fp32 residual stream, fp16 block)
        dict(name="norm_live", op="norm", windows=24, rows=1, c=1536, f16=True, x16=False, post="rms", gate="rows",
             gate_act="silu", pre="rms"),
        # ten minutes of 3 s windows of a few stations, all in fp32, an odd width (features beside the embedding), one
        # gate for a station
        dict(name="norm_station_f32", op="norm", windows=6, rows=200, c=1027, f16=False, x16=False, post="layer",
             gate="window", gate_act="sigmoid", pre="layer"),
        # a day of 5 s windows of one station in an archive, all in fp16
        dict(name="norm_archive", op="norm", windows=1, rows=17280, c=1536, f16=True, x16=True, post="rms",
             gate="rows", gate_act="silu", pre="rms"),
        # 24 live stations, one row each and an adapter each: the output projection with its residual
        dict(name="lora_live", op="lora", windows=24, rows=1, k=1536, n=1536, r=16, adapters=64, act="none", res=True),
        # a few windows of many stations: the projection into q, k, v and the gate
        dict(name="lora_stations", op="lora", windows=64, rows=4, k=1536, n=6144, r=8, adapters=32, act="none",
             res=False),
        # recordings of odd length and a layer of odd widths, SiLU after it
        dict(name="lora_odd", op="lora", windows=37, rows=45, k=1030, n=1101, r=12, adapters=9, act="silu", res=False),
        # an archive: an hour of 5 s windows of 24 stations through q, k, v and the gate
        dict(name="lora_archive", op="lora", windows=24, rows=720, k=1536, n=6144, r=16, adapters=24, act="none",
             res=False),
        # one live station's new window
        dict(name="linattn_live_one", op="linattn", windows=1, rows=1, ragged=False, heads=12, kv_heads=12, dk=128,
             dv=128, f16=True, state=True),
        # the new windows of 64 live stations
        dict(name="linattn_live", op="linattn", windows=64, rows=1, ragged=False, heads=12, kv_heads=12, dk=128, dv=128,
             f16=True, state=True),
        # recordings of up to an hour of 5 s windows side by side, going on from their stations' states
        dict(name="linattn_ragged", op="linattn", windows=24, rows=720, ragged=True, heads=12, kv_heads=12, dk=128,
             dv=128, f16=True, state=True),
        # a day of 5 s windows of one station: one long sequence
        dict(name="linattn_day", op="linattn", windows=1, rows=17280, ragged=False, heads=12, kv_heads=12, dk=128,
             dv=128, f16=True, state=False),
        # all in fp32, keys shared by four heads, values of an odd width
        dict(name="linattn_f32", op="linattn", windows=8, rows=500, ragged=True, heads=16, kv_heads=4, dk=64, dv=97,
             f16=False, state=True),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "lora", "linattn"])
    if op == "norm":
        c, b = _log(rng, 100, 2048), _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, (17280 * 1536) // (c * b)))
        f16 = rng.random() < 0.6
        return dict(op=op, windows=b, rows=rows, c=c, f16=f16, x16=f16 and rng.random() < 0.5,
                    post=rng.choice(["none", "rms", "layer"]), gate=rng.choice(["none", "window", "rows"]),
                    gate_act=rng.choice(["none", "silu", "sigmoid"]), pre=rng.choice(["rms", "layer"]))
    if op == "lora":
        k, n, b = _log(rng, 200, 2048), _log(rng, 200, 6144), _log(rng, 1, 256)
        if rng.random() < 0.6:
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        rows = _log(rng, 1, max(1, (17280 * 1536 * 6144) // (b * k * n)) if b > 1 else 4096)
        rows = min(rows, (17280 // b) or 1)
        return dict(op=op, windows=b, rows=rows, k=k, n=n, r=_log(rng, 4, 64), adapters=_log(rng, 1, 64),
                    act=rng.choice(["none", "silu", "relu"]), res=rng.random() < 0.4)
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 1, 2]) if kv > 4 else kv * rng.choice([1, 2, 4])
    dk, dv = _log(rng, 24, 128), _log(rng, 24, 128)
    if rng.random() < 0.6:
        dk, dv = (dk + 15) // 16 * 16, (dv + 15) // 16 * 16
    b = _log(rng, 1, 64)
    rows = _log(rng, 1, max(1, 17280 * 12 // (b * heads)))
    return dict(op=op, windows=b, rows=min(rows, 17280), ragged=rows > 1 and rng.random() < 0.5, heads=heads,
                kv_heads=kv, dk=dk, dv=dv, f16=rng.random() < 0.7, state=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _lens(c):
    """Rows of each sequence, from 1 to the longest: plain numbers of the case alone (a program knows its lengths)."""
    b, t = c["windows"], c["rows"]
    return [t if not c["ragged"] or i == 0 else 1 + (i * 7919 * 31) % t for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    c, s = case, dict(c=case)
    b, m = c["windows"], c["rows"]
    if c["op"] == "norm":
        tf, tx = (torch.float16 if h else torch.float32 for h in (c["f16"], c["x16"]))
        n = c["c"]
        s["f"] = normal(b, m, n, std=0.7).to(tf)
        s["x"] = (normal(b, m, n, std=2.0) + 0.3).to(tx)
        s["gate"] = None if c["gate"] == "none" else normal(b, m if c["gate"] == "rows" else 1, n).to(tf)
        s["scale"] = 0.1 + 0.5 * normal(n).abs()
        for k in ("post", "pre"):
            s[k + "_w"] = 1 + 0.2 * normal(n) if c[k] != "none" else None
            s[k + "_b"] = 0.1 * normal(n) if c[k] == "layer" else None
        s["y"], s["n"] = torch.empty_like(s["x"]), torch.empty_like(s["f"])
    elif c["op"] == "lora":
        k, n, r, a = c["k"], c["n"], c["r"], c["adapters"]
        s["x"] = normal(b, m, k).half()
        s["w"] = normal(n, k, std=k ** -0.5).half()
        s["bias"] = normal(n, std=0.1)
        s["a"] = normal(a, r, k, std=k ** -0.5).half()
        s["b"] = normal(a, n, r, std=0.5 * r ** -0.5).half()
        s["alpha"] = 0.5 + torch.rand(a, generator=g, device="cuda")
        # one station in nine has no adapter
        s["idx"] = torch.randint(-1 if a < 9 else -(a // 8), a, (b,), generator=g, device="cuda").clamp_(min=-1).int()
        s["res"] = normal(b, m, n).half() if c["res"] else None
        s["out"] = torch.empty((b, m, n), dtype=torch.float16, device="cuda")
        if own:
            hip = _hip()
            s["ws_bytes"] = hip.lib().bnh_pw_lora_work_bytes(m, b, n, k, r)
            s["ws"] = torch.empty(max(16, s["ws_bytes"]), dtype=torch.uint8, device="cuda")
    else:
        h, hk, dk, dv = c["heads"], c["kv_heads"], c["dk"], c["dv"]
        t = torch.float16 if c["f16"] else torch.float32
        lens = _lens(c)
        start = [sum(lens[:i]) for i in range(b)]
        rows, width = sum(lens), hk * (2 * dk) + h * dv
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        # q, k and v side by side in a projection's rows: queries and keys in kv_heads groups, a value head each
        s["qkv"] = normal(rows, width).to(t)
        # log decays of a gate: from near 0 (long memory) to about -2, spread over the heads
        bias = torch.linspace(-5.0, 0.5, h, device="cuda")
        s["g"] = -torch.nn.functional.softplus(normal(rows, h) + bias)
        s["s0"] = normal(b, h, dk, dv, std=2.0) if c["state"] else None
        s["s1"] = torch.empty((b, h, dk, dv), device="cuda")
        s["o"] = torch.empty((rows, h * dv), dtype=t, device="cuda")
        s["rows"] = rows
        if own:
            hip = _hip()
            s["ws_bytes"] = hip.lib().bnh_linattn_work_bytes(_linattn_args(hip, s), m, b)
            s["ws"] = torch.empty(max(16, s["ws_bytes"]), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ the framework's
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(hip, s):
    c, n = s["c"], s["c"]["c"]
    row = c["rows"] * n
    gate = s["gate"]
    a = hip.BlockNorm(f=_p(s["f"]), f_ws=row, ldf=n, f16=c["f16"],
                      post=hip.Norm(KIND[c["post"]], EPS, _p(s["post_w"]), _p(s["post_b"])), gate=_p(gate),
                      g_ws=row if c["gate"] == "rows" else n, ldg=n if c["gate"] == "rows" else 0,
                      gate_act=ACT[c["gate_act"]], scale=_p(s["scale"]), rs=0.5, x=_p(s["x"]), x_ws=row, ldx=n,
                      x16=c["x16"], y=_p(s["y"]), y_ws=row, ldy=n,
                      pre=hip.Norm(KIND[c["pre"]], EPS, _p(s["pre_w"]), _p(s["pre_b"])), n=_p(s["n"]), n_ws=row, ldn=n)
    hip.check(hip.lib().bnh_block_norm(a, c["rows"], n, c["windows"], _stream()), "block_norm")
    return s["y"], s["n"]


def _own_lora(hip, s):
    c, k, n = s["c"], s["c"]["k"], s["c"]["n"]
    m = c["rows"]
    L = hip.Lora(n=c["adapters"], r=c["r"], a=_p(s["a"]), b=_p(s["b"]), scale=_p(s["alpha"]))
    e = hip.Epi16(ACT[c["act"]], _p(s["out"]), m * n, n, 0, 0, _p(s["res"]), m * n, n)
    hip.check(hip.lib().bnh_pw_lora(_p(s["x"]), m * k, k, m, c["windows"], _p(s["w"]), k, n, k, _p(s["bias"]), L,
                                    _p(s["idx"]), e, _p(s["ws"]), s["ws_bytes"], _stream()), "pw_lora")
    return s["out"]


def _linattn_args(hip, s):
    c = s["c"]
    h, hk, dk, dv, qkv = c["heads"], c["kv_heads"], c["dk"], c["dv"], s["qkv"]
    ld, es = qkv.shape[1], qkv.element_size()
    return hip.LinAttn(q=_p(qkv), k=_p(qkv) + es * hk * dk, v=_p(qkv) + es * 2 * hk * dk, o=_p(s["o"]), f16=c["f16"],
                       ldq=ld, ldk=ld, ldv=ld, ldo=h * dv, H=h, Hq=hk, Hk=hk, Hv=h, dk=dk, dv=dv, g=_p(s["g"]), ldg=h,
                       scale=dk ** -0.5, s0=_p(s["s0"]), s1=_p(s["s1"]), slots=c["windows"], slot=None)


def _own_linattn(hip, s):
    c = s["c"]
    hip.check(hip.lib().bnh_linattn(_linattn_args(hip, s), c["rows"], c["windows"], s["rows"], _p(s["start"]),
                                    _p(s["lens"]), _p(s["ws"]), s["ws_bytes"], _stream()), "linattn")
    return s["o"], s["s1"]


# ------------------------------------------------------------------------------------------------ plain torch
def _norm(u, kind, w, b):
    if kind == "none":
        return u
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w
    return u if b is None else u + b


def _act(u, act):
    if act == "relu":
        return torch.relu(u)
    return u if act == "none" else torch.sigmoid(u) * (u if act == "silu" else 1)


def _plain_norm(s):
    c = s["c"]
    u = _norm(s["f"].float(), c["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        u = u * _act(s["gate"].float(), c["gate_act"])
    y = s["x"].float() + 0.5 * s["scale"] * u
    n = _norm(y, c["pre"], s["pre_w"], s["pre_b"])
    return y.to(s["x"].dtype), n.to(s["f"].dtype)


def _plain_lora(s):
    c = s["c"]
    x, idx = s["x"].float(), s["idx"].long()
    y = (x.reshape(-1, c["k"]) @ s["w"].float().t()).reshape(s["out"].shape) + s["bias"]
    at = idx.clamp(min=0)
    alpha = torch.where(idx >= 0, s["alpha"][at], 0.0)
    t = torch.matmul(x, s["a"][at].float().transpose(1, 2).contiguous())
    y = y + alpha[:, None, None] * torch.matmul(t, s["b"][at].float().transpose(1, 2).contiguous())
    y = _act(y, c["act"])
    return (y if s["res"] is None else y + s["res"].float()).half()


def _segments(g):
    """exp of the sum of g over (j, i], [..., i, j], and 0 where j > i."""
    n = g.shape[-1]
    low = torch.ones((n, n), dtype=torch.bool, device=g.device).tril()
    sums = torch.where(low.tril(-1), g[..., :, None], 0.0).cumsum(-2)
    return torch.where(low, torch.exp(sums), 0.0)


def _plain_linattn(s):
    c, b, t = s["c"], s["c"]["windows"], s["c"]["rows"]
    h, hk, dk, dv = c["heads"], c["kv_heads"], c["dk"], c["dv"]
    size = min(64, t)
    n = -(-t // size)
    at = torch.arange(n * size, device="cuda")[None]
    there = at < s["lens"][:, None]
    row = (s["start"][:, None] + at).clamp(max=s["rows"] - 1).long()

    def heads(x, groups):  # [b][h][n][size][d] of the padded sequences, zero past their ends
        x = torch.where(there[..., None], x[row], 0.0).reshape(b, n, size, groups, -1).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(h // groups, 1).contiguous()

    x = s["qkv"].float()
    q, k, v = heads(x[:, :hk * dk], hk), heads(x[:, hk * dk:2 * hk * dk], hk), heads(x[:, 2 * hk * dk:], h)
    g = heads(s["g"], h)[..., 0]
    decay = _segments(g)
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay, v)
    new = torch.matmul((k * decay[..., -1, :, None]).transpose(-1, -2).contiguous(), v)
    first = torch.zeros((b, h, dk, dv), device="cuda") if s["s0"] is None else s["s0"]
    over = _segments(torch.nn.functional.pad(g.sum(-1), (1, 0)))  # from one chunk's end to another's
    states = torch.matmul(over, torch.cat([first[:, :, None], new], 2).reshape(b, h, n + 1, dk * dv))
    states = states.reshape(b, h, n + 1, dk, dv)
    o = (o + torch.exp(g.cumsum(-1))[..., None] * torch.matmul(q, states[:, :, :n])) * dk ** -0.5
    o = o.permute(0, 2, 3, 1, 4).reshape(b, n * size, h * dv)[there]
    return o.to(s["o"].dtype), states[:, :, n].contiguous()


_PLAIN = {"norm": _plain_norm, "lora": _plain_lora, "linattn": _plain_linattn}
_OWN = {"norm": _own_norm, "lora": _own_lora, "linattn": _own_linattn}


def run(state):
    op = state["c"]["op"]
    return _OWN[op](_hip(), state) if own else _PLAIN[op](state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_norm(s):
    c = s["c"]

    def norm(u, name):
        if c[name] == "none":
            return u
        mean = u.mean(-1, keepdim=True) if c[name] == "layer" else 0.0
        y = (u - mean) / torch.sqrt(((u - mean) ** 2).mean(-1, keepdim=True) + EPS) * s[name + "_w"].double()
        return y + s[name + "_b"].double() if c[name] == "layer" else y

    def act(u):
        return {"none": u, "silu": u / (1 + torch.exp(-u)), "sigmoid": 1 / (1 + torch.exp(-u))}[c["gate_act"]]

    gate = 1.0 if s["gate"] is None else act(s["gate"].double())
    y = s["x"].double() + 0.5 * s["scale"].double() * gate * norm(s["f"].double(), "post")
    return y, norm(y, "pre")


def _exact_lora(s):
    c, out = s["c"], []
    shared = s["x"].double() @ s["w"].double().t() + s["bias"].double()
    for w, a in enumerate(s["idx"].tolist()):
        x, y = s["x"][w].double(), shared[w]
        if a >= 0:
            y = y + s["alpha"][a].double() * ((x @ s["a"][a].double().t()) @ s["b"][a].double().t())
        y = {"none": y, "relu": y.clamp(min=0), "silu": y / (1 + torch.exp(-y))}[c["act"]]
        out.append(y if s["res"] is None else y + s["res"][w].double())
    return torch.stack(out)


def _exact_linattn(s):
    """The recurrence, row by row, all sequences of one length at a time left behind as they end."""
    c = s["c"]
    b, h, hk, dk, dv = c["windows"], c["heads"], c["kv_heads"], c["dk"], c["dv"]
    state = torch.zeros((b, h, dk, dv), dtype=torch.float64, device="cuda")
    if s["s0"] is not None:
        state += s["s0"]
    o = torch.zeros((s["rows"], h, dv), dtype=torch.float64, device="cuda")
    lens, start = _lens(c), s["start"].tolist()
    group = torch.arange(h, device="cuda") // (h // hk)
    cuts = sorted(set(lens))
    for lo, hi in zip([0] + cuts, cuts):
        live = [i for i in range(b) if lens[i] >= hi]
        first = torch.tensor([start[i] for i in live], device="cuda")
        at = torch.tensor(live, device="cuda")
        now = state[at]
        for t in range(lo, hi):
            x = s["qkv"][first + t].double()
            q, k = x[:, :hk * dk].reshape(-1, hk, dk)[:, group], x[:, hk * dk:2 * hk * dk].reshape(-1, hk, dk)[:, group]
            v = x[:, 2 * hk * dk:].reshape(-1, h, dv)
            now = now * torch.exp(s["g"][first + t].double())[..., None, None] + k[..., None] * v[..., None, :]
            o[first + t] = dk ** -0.5 * (q[..., None] * now).sum(-2)
        state[at] = now
    return o.reshape(s["rows"], h * dv), state


def exact(case, seed):
    c = case
    if c["op"] == "linattn" and c["rows"] * (40e-6 + c["windows"] * c["heads"] * c["dk"] * c["dv"] * 4e-11) > 10:
        return None
    return {"norm": _exact_norm, "lora": _exact_lora, "linattn": _exact_linattn}[c["op"]](prepare(case, seed))


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    b, m = c["windows"], c["rows"]
    if c["op"] == "norm":
        ef, ex, n = 2 if c["f16"] else 4, 2 if c["x16"] else 4, c["c"]
        gate = {"none": 0, "window": b, "rows": b * m}[c["gate"]]
        return dict(bytes=n * (b * m * 2 * (ef + ex) + gate * ef + 4 * 3), flops=20 * b * m * n)
    if c["op"] == "lora":
        k, n, r = c["k"], c["n"], c["r"]
        used = min(b, c["adapters"])
        return dict(bytes=2 * (n * k + b * m * (k + n * (2 if c["res"] else 1)) + used * r * (k + n)) + 4 * n,
                    flops=2 * b * m * (n * k + r * (k + n)))
    h, hk, dk, dv, rows = c["heads"], c["kv_heads"], c["dk"], c["dv"], sum(_lens(c))
    es = 2 if c["f16"] else 4
    return dict(bytes=rows * (es * (2 * hk * dk + 2 * h * dv) + 4 * h) + 4 * b * h * dk * dv * (2 if c["state"] else 1),
                flops=4 * rows * h * dk * dv)
