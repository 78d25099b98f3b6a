"""Temporal context over the windows of recordings: blocks of norm, gated linear attention and projections with an adapter
for each station, over the embeddings that a net leaves on the device, with random weights.

    python -m bnneon.contextnet        # an archive and live windows of the same stations, timed

Per block, for the rows (windows) x of all stations:
    q, k, v, gate = W_in norm(x) + the station's adapter
    o = linear attention of q, k, v with a decay for each head, from the station's state
    f = W_out o + the station's adapter
    x = x + scale silu(gate) norm(f)
The residual stream is fp32, the rest fp16. An archive's rows go through in one call, a live station's one at a time; the
states carry over between calls.

Blocks named in `cached` have attention over a cache of the station's windows in its place: q and k are rotated by the window's
number in its recording, k and v go into pages that the stations share, and each window looks at all up to it, or at the
`seen` pages (the station's first, the last two, and those with the largest bounds on their scores).
"""
import numpy as np

from . import hip


class ContextNet:
    def __init__(self, dim=1536, heads=12, layers=2, stations=24, rank=16, seed=0, cached=(), windows=17280, page=64, pages=None,
                 seen=0):
        if heads < 1 or dim < 1 or dim % heads or dim // heads > 256 or dim > 16384:
            raise ValueError(f"dim {dim} is not {heads} heads of at most 256")
        if layers < 1 or stations < 1 or not 1 <= rank <= 256:
            raise ValueError(f"{layers} layers of {stations} stations' adapters of rank {rank}: one at least, rank up to 256")
        cached = tuple(sorted(set(int(i) for i in cached)))
        if cached and not 0 <= cached[0] <= cached[-1] < layers:
            raise ValueError(f"cached blocks {cached} of {layers}")
        if windows < 1 or not 16 <= page <= 1024 or page & (page - 1) or (pages is not None and pages < 1):
            raise ValueError(f"a cache of {pages} pages of {page}, up to {windows} windows a station")
        if -(-windows // page) * page >= (1 << 31) - 1024:
            raise ValueError(f"{windows} windows a station: below 2^31 - 1024 of them")
        if seen and not 3 <= seen <= 1 << 20:
            raise ValueError(f"{seen} pages seen: 3 at least, the first and the last two among them, or 0 for all")
        self.dim, self.heads, self.layers, self.stations, self.rank = dim, heads, layers, stations, rank
        self.cached, self.windows, self.page, self.seen = cached, windows, page, seen
        rng = np.random.default_rng(seed)

        def dev(a, dtype):
            return hip.DeviceArray.from_host(np.asarray(a, dtype))

        def linear(n, k):
            """A projection [n][k] with bias and adapters of every station."""
            w = rng.standard_normal((n, k), np.float32) / np.sqrt(k)
            a = rng.standard_normal((stations, rank, k), np.float32) / np.sqrt(k)
            b = rng.standard_normal((stations, n, rank), np.float32) * (0.3 / np.sqrt(rank))
            bias = 0.02 * rng.standard_normal(n, np.float32)
            host = dict(w=w.astype(np.float16), a=a.astype(np.float16), b=b.astype(np.float16), bias=bias)
            d = {key: dev(h, h.dtype) for key, h in host.items()}
            d["lora"] = hip.Lora(stations, rank, d["a"].ptr, d["b"].ptr, None)
            return host, d

        self.host, self.blocks = [], []
        for _ in range(layers):
            hin, din = linear(4 * dim, dim)
            hout, dout = linear(dim, dim)
            h = dict(win=hin, wout=hout, pre=1 + 0.1 * rng.standard_normal(dim).astype(np.float32),
                     post=1 + 0.1 * rng.standard_normal(dim).astype(np.float32),
                     scale=np.full(dim, 0.2, np.float32))
            self.host.append(h)
            self.blocks.append(dict(win=din, wout=dout, **{k: dev(h[k], np.float32) for k in ("pre", "post", "scale")}))
        self.final = 1 + 0.1 * rng.standard_normal(dim).astype(np.float32)
        self.dfinal = dev(self.final, np.float32)
        # memories of 4 to 2000 windows
        self.g = -1 / np.geomspace(4, 2000, heads).astype(np.float32)
        self.dg = dev(self.g, np.float32)
        d = dim // heads
        self.state = [hip.DeviceArray.zeros((stations, heads, d, d), np.float32) if i not in cached else None
                      for i in range(layers)]
        if cached:
            self.ldt = -(-windows // page)
            self.pages = pages or stations * self.ldt
            self.cache = {i: {k: hip.DeviceArray.zeros((self.pages, heads, n, d), np.float16)
                              for k, n in (("k", page), ("v", page)) + ((("lo", 1), ("hi", 1)) if seen else ())} for i in cached}
            # a turn in 2 pi windows to one in about a day
            self.rd = d // 2 * 2
            self.freq = (17280.0 ** (-2 * np.arange(self.rd // 2) / max(1, self.rd))).astype(np.float32)
            self.dfreq = dev(self.freq if self.rd else np.zeros(1), np.float32)
            self._empty()

    def _empty(self):
        self.free = list(range(self.pages))[::-1]
        self.table = np.full((self.stations, self.ldt), -1, np.int32)
        self.past = np.zeros(self.stations, np.int32)

    def reset(self):
        """As a new net: all states zero, all pages free. Waits for the device first, as forget() does."""
        hip.device_sync()
        for s in self.state:
            if s is not None:
                s.fill(0)
        if self.cached:
            self._empty()

    def plan(self, lens, stations):
        """The buffers of a call on sequences of the given lengths, one each of the stations given (a program that makes the
        same call again keeps it)."""
        lens, stations = [int(n) for n in lens], [int(s) for s in stations]
        if len(lens) != len(stations) or not lens or min(lens) < 0 or sum(lens) < 1:
            raise ValueError("a length and a station for each sequence, and a row at least")
        if len(set(stations)) != len(stations) or not all(0 <= s < self.stations for s in stations):
            raise ValueError("the stations of a call are different ones of this net's")
        L, rows, dim = hip.lib(), sum(lens), self.dim
        half = lambda n: hip.DeviceArray((rows, n), np.float16)  # noqa: E731
        p = dict(B=len(lens), T=max(lens), rows=rows, x=hip.DeviceArray((rows, dim), np.float32), n=half(dim),
                 qkvg=half(4 * dim), o=half(dim), f=half(dim),
                 start=hip.DeviceArray.from_host(np.cumsum([0] + lens[:-1]).astype(np.int32)),
                 len=hip.DeviceArray.from_host(np.array(lens, np.int32)),
                 slot=hip.DeviceArray.from_host(np.array(stations, np.int32)),
                 idx=hip.DeviceArray.from_host(np.repeat(np.array(stations, np.int32), lens)))
        p["la"], p["lens"], p["stations"] = [], lens, stations
        for s in self.state:
            d, q = dim // self.heads, p["qkvg"].ptr
            p["la"].append(None if s is None else
                           hip.LinAttn(q=q, k=q + 2 * dim, v=q + 4 * dim, o=p["o"].ptr, f16=1, ldq=4 * dim, ldk=4 * dim,
                                       ldv=4 * dim, ldo=dim, H=self.heads, Hq=self.heads, Hk=self.heads, Hv=self.heads,
                                       dk=d, dv=d, g=self.dg.ptr, ldg=0, scale=d ** -0.5, s0=s.ptr, s1=s.ptr,
                                       slots=self.stations, slot=p["slot"].ptr))
        n_in = L.bnh_pw_lora_work_bytes(1, rows, 4 * dim, dim, self.rank)
        n_out = L.bnh_pw_lora_work_bytes(1, rows, dim, dim, self.rank)
        n_la = max((L.bnh_linattn_work_bytes(a, p["T"], p["B"]) for a in p["la"] if a is not None), default=0)
        if self.cached:
            n_la = max(n_la, self._plan_cached(p))
        p["wb"] = max(n_in, n_out, n_la, 16)
        p["work"] = hip.DeviceArray(p["wb"], np.uint8)
        return p

    def _plan_cached(self, p):
        """The descriptors of the cached blocks, and the workspace that they need."""
        L, d, n, H = hip.lib(), self.dim // self.heads, 0, self.heads
        # no pages until advance() writes them: a run ahead of it stores nothing
        p["table"] = hip.DeviceArray.from_host(np.full((p["B"], self.ldt), -1, np.int32))
        p["past"] = hip.DeviceArray.zeros((p["B"],), np.int32)
        p["sel"] = hip.DeviceArray((p["rows"], H, self.seen), np.int32) if self.seen else None
        p["kv"], q = {}, p["qkvg"].ptr
        for i, c in self.cache.items():
            bounds = (c["lo"].ptr, c["hi"].ptr) if self.seen else (None, None)
            kv = hip.KvCache(k=c["k"].ptr, v=c["v"].ptr, k_ps=H * self.page * d, v_ps=H * self.page * d, f16=1, pages=self.pages,
                             page=self.page, Hk=H, dk=d, dv=d, lo=bounds[0], hi=bounds[1], table=p["table"].ptr, ldt=self.ldt,
                             past=p["past"].ptr)
            a = hip.KvAttn(q=q, ldq=4 * self.dim, o=p["o"].ptr, ldo=self.dim, H=H, scale=d ** -0.5, window=0, sel=hip.ptr(p["sel"]),
                           nsel=self.seen)
            p["kv"][i] = kv, a
            n = max(n, L.bnh_kv_attn_work_bytes(kv, a, p["T"], p["B"], p["rows"]))
            if self.seen:
                n = max(n, L.bnh_kv_select_work_bytes(kv, a, p["T"], p["B"], p["rows"]))
        return n

    def advance(self, p, stream=None):
        """Pages for the windows of the plan's next run, and where they go, on the device (run() calls it; a program that replays
        a captured run calls it before each). Nothing moves if there are not enough pages."""
        if not self.cached:
            return
        need = [(s, self.past[s] + n) for s, n in zip(p["stations"], p["lens"])]
        if any(n > self.windows for _, n in need):
            raise ValueError(f"more than {self.windows} windows of a station")
        have = {s: int((self.table[s] >= 0).sum()) for s, _ in need}
        if sum(max(0, -(-n // self.page) - have[s]) for s, n in need) > len(self.free):
            raise ValueError("the cache has no pages left")
        for s, n in need:
            for x in range(have[s], -(-int(n) // self.page)):
                self.table[s, x] = self.free.pop()
        hip.sync(stream)  # runs that still read the tables
        p["table"].upload(self.table[p["stations"]])
        p["past"].upload(self.past[p["stations"]])
        for s, n in need:
            self.past[s] = n

    def forget(self, station):
        """The station's next window is its first: its states are zero, and its pages free. Waits for all that runs on the device:
        a run on any stream may still store the station's states or read its pages, and what comes next on any stream finds
        the states cleared."""
        if not 0 <= station < self.stations:
            raise ValueError(f"station {station} of {self.stations}")
        hip.device_sync()
        for s in self.state:
            if s is not None:
                n = s.nbytes // self.stations
                hip.check(hip.lib().bnh_memset(s.ptr + station * n, 0, n), "bnh_memset")
        if self.cached:
            self.free += [int(x) for x in self.table[station] if x >= 0]
            self.table[station], self.past[station] = -1, 0

    def _look(self, p, i, stream):
        """o of a cached block: new keys and values into the cache, rotated, and q where it lies; then the attention."""
        L, (kv, a), q, dim = hip.lib(), p["kv"][i], p["qkvg"].ptr, self.dim
        seqs = p["T"], p["B"], p["rows"], p["start"].ptr, p["len"].ptr
        rot = hip.Rotary(self.rd, 0, self.dfreq.ptr, None)
        hip.check(L.bnh_kv_append(kv, rot, q + 2 * dim, 4 * dim, q + 4 * dim, 4 * dim, q, 4 * dim, q, 4 * dim, self.heads, *seqs,
                                  stream), "kv_append")
        if self.seen:
            hip.check(L.bnh_kv_select(kv, a, 1, 2, *seqs, p["work"].ptr, p["wb"], stream), "kv_select")
        hip.check(L.bnh_kv_attn(kv, a, *seqs, p["work"].ptr, p["wb"], stream), "kv_attn")

    def _linear(self, p, d, x, n, out, stream):
        e = hip.Epi16(0, out.ptr, n, n, 0, 0, None, 0, 0)
        # one row a window, so that every row has its own station's adapter
        hip.check(hip.lib().bnh_pw_lora(x.ptr, self.dim, self.dim, 1, p["rows"], d["w"].ptr, self.dim, n, self.dim,
                                        d["bias"].ptr, d["lora"], p["idx"].ptr, e, p["work"].ptr, p["wb"], stream),
                  "pw_lora")

    def run(self, p, stream=None, advance=True):
        """The blocks over p["x"], which holds the embeddings (rows of one sequence in time order): x in place, and its last
        norm in p["n"], fp16. The states of p's stations move on, and their caches, for which advance() has been called before
        where `advance` is not set. A run that fails leaves the caches where they were; linear attention ahead of the call that
        failed has moved its states on, so that the stations have to be forgotten if there is any."""
        if not (advance and self.cached):
            return self._blocks(p, stream)
        before = self.past.copy()
        self.advance(p, stream)
        try:
            self._blocks(p, stream)
        except BaseException:
            self.past[p["stations"]] = before[p["stations"]]
            raise

    def _blocks(self, p, stream):
        L, dim = hip.lib(), self.dim

        def norm(pre, f=None, b=None):
            a = hip.BlockNorm(f16=1, x=p["x"].ptr, ldx=dim, n=p["n"].ptr, ldn=dim, pre=hip.Norm(1, 1e-6, pre.ptr, None))
            if f is not None:
                a.f, a.ldf, a.post = f.ptr, dim, hip.Norm(1, 1e-6, b["post"].ptr, None)
                a.gate, a.ldg, a.gate_act = p["qkvg"].ptr + 6 * dim, 4 * dim, 1
                a.scale, a.rs, a.y, a.ldy = b["scale"].ptr, 1.0, p["x"].ptr, dim
            hip.check(L.bnh_block_norm(a, p["rows"], dim, 1, stream), "block_norm")

        norm(self.blocks[0]["pre"])
        for i, b in enumerate(self.blocks):
            self._linear(p, b["win"], p["n"], 4 * dim, p["qkvg"], stream)
            if i in self.cached:
                self._look(p, i, stream)
            else:
                hip.check(L.bnh_linattn(p["la"][i], p["T"], p["B"], p["rows"], p["start"].ptr, p["len"].ptr, p["work"].ptr,
                                        p["wb"], stream), "linattn")
            self._linear(p, b["wout"], p["o"], dim, p["f"], stream)
            norm(self.blocks[i + 1]["pre"] if i + 1 < self.layers else self.dfinal, p["f"], b)


def main():
    import time
    rng = np.random.default_rng(1)
    lens = [720 - 13 * i for i in range(24)]  # up to an hour of 5 s windows
    x = rng.standard_normal((sum(lens), 1536)).astype(np.float32)
    for what, kw in (("linear attention", {}), ("one block over the windows' cache", dict(cached=[1], windows=8192)),
                     ("one over 8 pages of it", dict(cached=[1], windows=8192, seen=8))):
        net = ContextNet(**kw)
        archive = net.plan(lens, range(net.stations))
        live = net.plan([1] * net.stations, range(net.stations))
        for name, p, n in (("archive", archive, 5), ("live", live, 200)):
            p["x"].upload(x[:p["rows"]])
            net.run(p)
            hip.sync()
            t = time.perf_counter()
            for _ in range(n):
                net.run(p)
            hip.sync()
            t = (time.perf_counter() - t) / n
            print(f"{what}, {name}: {p['rows']} windows of {p['B']} stations, {net.layers} blocks: {t * 1e6:.0f} us, "
                  f"{p['rows'] / t:.0f} windows/s")


if __name__ == "__main__":
    main()
