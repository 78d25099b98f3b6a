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
"""
import numpy as np

from . import hip


class ContextNet:
    def __init__(self, dim=1536, heads=12, layers=2, stations=24, rank=16, seed=0):
        if heads < 1 or dim < 1 or dim % heads or dim // heads > 256 or dim > 16384:
            raise ValueError(f"dim {dim} is not {heads} heads of at most 256")
        if layers < 1 or stations < 1 or not 1 <= rank <= 256:
            raise ValueError(f"{layers} layers of {stations} stations' adapters of rank {rank}: one at least, rank up to 256")
        self.dim, self.heads, self.layers, self.stations, self.rank = dim, heads, layers, stations, rank
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
        self.state = [hip.DeviceArray.zeros((stations, heads, d, d), np.float32) for _ in range(layers)]

    def reset(self):
        for s in self.state:
            s.fill(0)

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
        p["la"] = []
        for s in self.state:
            d, q = dim // self.heads, p["qkvg"].ptr
            p["la"].append(hip.LinAttn(q=q, k=q + 2 * dim, v=q + 4 * dim, o=p["o"].ptr, f16=1, ldq=4 * dim, ldk=4 * dim,
                                       ldv=4 * dim, ldo=dim, H=self.heads, Hq=self.heads, Hk=self.heads, Hv=self.heads,
                                       dk=d, dv=d, g=self.dg.ptr, ldg=0, scale=d ** -0.5, s0=s.ptr, s1=s.ptr,
                                       slots=self.stations, slot=p["slot"].ptr))
        n_in = L.bnh_pw_lora_work_bytes(1, rows, 4 * dim, dim, self.rank)
        n_out = L.bnh_pw_lora_work_bytes(1, rows, dim, dim, self.rank)
        n_la = L.bnh_linattn_work_bytes(p["la"][0], p["T"], p["B"])
        p["wb"] = max(n_in, n_out, n_la, 16)
        p["work"] = hip.DeviceArray(p["wb"], np.uint8)
        return p

    def _linear(self, p, d, x, n, out, stream):
        e = hip.Epi16(0, out.ptr, n, n, 0, 0, None, 0, 0)
        # one row a window, so that every row has its own station's adapter
        hip.check(hip.lib().bnh_pw_lora(x.ptr, self.dim, self.dim, 1, p["rows"], d["w"].ptr, self.dim, n, self.dim,
                                        d["bias"].ptr, d["lora"], p["idx"].ptr, e, p["work"].ptr, p["wb"], stream),
                  "pw_lora")

    def run(self, p, stream=None):
        """The blocks over p["x"], which holds the embeddings (rows of one sequence in time order): x in place, and its last
        norm in p["n"], fp16. The states of p's stations move on."""
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
            hip.check(L.bnh_linattn(p["la"][i], p["T"], p["B"], p["rows"], p["start"].ptr, p["len"].ptr, p["work"].ptr,
                                    p["wb"], stream), "linattn")
            self._linear(p, b["wout"], p["o"], dim, p["f"], stream)
            norm(self.blocks[i + 1]["pre"] if i + 1 < self.layers else self.dfinal, p["f"], b)


def main():
    import time
    net = ContextNet()
    rng = np.random.default_rng(1)
    lens = [720 - 13 * i for i in range(net.stations)]  # up to an hour of 5 s windows
    archive = net.plan(lens, range(net.stations))
    live = net.plan([1] * net.stations, range(net.stations))
    x = rng.standard_normal((archive["rows"], net.dim)).astype(np.float32)
    for name, p, n in (("archive", archive, 5), ("live", live, 200)):
        p["x"].upload(x[:p["rows"]])
        net.run(p)
        hip.sync()
        t = time.perf_counter()
        for _ in range(n):
            net.run(p)
        hip.sync()
        t = (time.perf_counter() - t) / n
        print(f"{name}: {p['rows']} windows of {p['B']} stations, {net.layers} blocks: {t * 1e6:.0f} us, "
              f"{p['rows'] / t:.0f} windows/s")


if __name__ == "__main__":
    main()
