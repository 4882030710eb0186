"""Layers held in 4 bits and the norms around a block, as cases that can be
timed and checked: the decode matvec over 4-bit weights, the routed experts
over 4-bit weights, weights quantised to 4 bits and read back, and the norm
after a block, its gate, the residual add and the next block's norm in one
pass.

4-bit weights: a row's elements k in groups of `group` (32, 64 or 128; the
last one may be short), an element (q - 8) * s with q of 0..15 and its
group's bf16 scale s.  Two codes a byte, the lower half the even element.

Each case runs in its plain form, elementary torch operations in 32 bits, or
through the package (`own`): Gpu, Engine and the kernels' descriptors.  The
shapes are those of a 4B-class layer (hidden 2560, 4096 wide attention, MLP
9216, vocabulary 151936), of the 27B-class projections (5120, 7168, 17408)
and of a 35B-A3B-class sparse layer (hidden 2048, 256 experts, top 8,
intermediate 512), and sizes between them that divide by little.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

EXPERTS, TOP_K, MH, MI = 256, 8, 2048, 512
EPS = 1e-6


def listed():
    return [
        # One sequence's output projection: the shortest launch of a decode
        # step, where latency counts.
        {"name": "mv_o_m1", "op": "matvec", "k": 4096, "n": 2560, "group": 32, "out": "Bf16", "m": 1},
        # One sequence's gate and up with the SwiGLU in it.
        {"name": "mv_gate_up_m1", "op": "matvec", "k": 2560, "n": 18432, "group": 64, "out": "Swiglu", "m": 1},
        # Three sequences on a shape that no tile divides, K in a short last
        # group and a short last tile.
        {"name": "mv_ragged_m3", "op": "matvec", "k": 5000, "n": 7001, "group": 128, "out": "Bf16", "m": 3},
        # Four sequences' logits in f32: the largest matrix of a step.
        {"name": "mv_head_m4", "op": "matvec", "k": 2560, "n": 151936, "group": 32, "out": "F32", "m": 4},
        # Sixteen sequences on the 27B-class down projection.
        {"name": "mv_down27_m16", "op": "matvec", "k": 17408, "n": 5120, "group": 128, "out": "Bf16", "m": 16},
        # The experts of one token, and of a decode batch of 64.
        {"name": "experts_t1", "op": "experts", "t": 1, "group": 32},
        {"name": "experts_t64", "op": "experts", "t": 64, "group": 128},
        # A small projection's weights quantised at load and read back, and
        # the 27B-class gate and up.
        {"name": "quant_1024", "op": "quant", "k": 1024, "n": 3584, "group": 64},
        {"name": "quant_gate_up27", "op": "quant", "k": 5120, "n": 34816, "group": 32},
        # One sequence between two blocks: post norm, add, next norm.
        {"name": "norm_m1", "op": "norm", "n": 2560, "m": 1, "post": True, "gate": "Off", "scales": False},
        # A short prompt with an element-wise gate on the block's output.
        {"name": "norm_gate_m57", "op": "norm", "n": 2560, "m": 57, "post": False, "gate": "Elements", "scales": False},
        # A long prompt's block with both norms and a layer's scales.
        {"name": "norm_m2048", "op": "norm", "n": 5120, "m": 2048, "post": True, "gate": "Rows", "scales": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "matvec", "experts", "quant", "norm", "norm"])
    group = rng.choice([32, 64, 128])
    if op == "matvec":
        out = rng.choice(["Bf16", "F32", "Swiglu"])
        k = 8 * _log(rng, 64, 2176)
        n = _log(rng, 1024, min(40960, 300_000_000 // k))
        if out == "Swiglu":  # gate and up, each whole 16-row tiles
            n = max(32, n // 32 * 32)
        return {"op": op, "k": k, "n": n, "group": group, "out": out, "m": _log(rng, 1, 16)}
    if op == "experts":
        return {"op": op, "t": _log(rng, 1, 64), "group": group}
    if op == "quant":
        return {"op": op, "k": 8 * _log(rng, 64, 640), "n": _log(rng, 1024, 34816), "group": group}
    return {"op": op, "n": _log(rng, 512, 8192), "m": _log(rng, 1, 1280), "post": rng.random() < 0.5,
            "gate": rng.choice(["Off", "Rows", "Elements", "Channels"]), "scales": rng.random() < 0.5}


# ---- the inputs, from the seed ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62))
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, std, generator=g)


def _activations(g, m, k):
    """N(0, 1) rows with a few channels a tenfold larger, as a model's are."""
    x = torch.empty((m, k), dtype=torch.float32, device="cuda").normal_(0, 1, generator=g)
    big = torch.rand((k,), device="cuda", generator=g) < 0.004
    return (x * torch.where(big, 10.0, 1.0)).to(torch.bfloat16)


def _codes(g, rows, k, group):
    """(bytes [rows][k / 2], scales [rows][groups]): the codes of normal
    weights of 0.02, whose groups' largest element is -8 scales."""
    q = torch.empty((rows, k), dtype=torch.float16, device="cuda").normal_(8.0, 3.2, generator=g)
    q = q.round_().clamp_(0, 15).to(torch.uint8)
    codes = q[:, 0::2] | (q[:, 1::2] << 4)
    s = torch.empty((rows, -(-k // group)), dtype=torch.float32, device="cuda").uniform_(0.004, 0.009, generator=g)
    sign = torch.rand(s.shape, device="cuda", generator=g) < 0.5
    return codes.contiguous(), torch.where(sign, -s, s).to(torch.bfloat16)


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "matvec":
        codes, scales = _codes(g, case["n"], case["k"], case["group"])
        return {"codes": codes, "scales": scales, "x": _activations(g, case["m"], case["k"])}
    if op == "experts":
        t, group = case["t"], case["group"]
        gu, gs = _codes(g, EXPERTS * 2 * MI, MH, group)
        dn, ds = _codes(g, EXPERTS * MH, MI, group)
        x = _activations(g, t, MH)
        scores = torch.empty((t, EXPERTS), dtype=torch.float32, device="cuda").normal_(0, 1, generator=g)
        ids = torch.sort(torch.sort(scores, dim=-1, descending=True, stable=True).indices[:, :TOP_K], dim=-1).values
        # The routed pairs (row * TOP_K + slot) by expert: what moe_sort
        # makes of a route, with its table of tiles of up to 16 rows.
        flat = ids.reshape(-1)
        order = torch.sort(flat, stable=True).indices
        count = torch.bincount(flat, minlength=EXPERTS)
        first = torch.cumsum(count, 0) - count
        per = (count + 15) // 16
        e = torch.repeat_interleave(torch.arange(EXPERTS, device="cuda"), per)
        at = 16 * (torch.arange(len(e), device="cuda") - torch.repeat_interleave(torch.cumsum(per, 0) - per, per))
        table = torch.stack([e, first[e] + at, torch.minimum(count[e] - at, torch.full_like(at, 16))], 1)
        tiles = torch.zeros(1 + 3 * (-(-t * TOP_K // 16) + EXPERTS), dtype=torch.int32, device="cuda")
        tiles[0] = len(e)
        tiles[1:1 + table.numel()] = table.reshape(-1).to(torch.int32)
        return {"gu": gu, "gs": gs, "dn": dn, "ds": ds, "x": x, "list": order.to(torch.int32), "tiles": tiles,
                "expert": flat[order].to(torch.int64)}
    if op == "quant":
        # Weights whose rows differ in size, as a checkpoint's do.
        w = torch.empty((case["n"], case["k"]), dtype=torch.float32, device="cuda").normal_(0, 0.02, generator=g)
        row = torch.empty((case["n"], 1), dtype=torch.float32, device="cuda").uniform_(0.3, 3.0, generator=g)
        return {"w": w.mul_(row).to(torch.bfloat16)}
    m, n = case["m"], case["n"]
    v = {"x": _activations(g, m, n), "y": _normal(g, (m, n), 0.5), "w_pre": _normal(g, (n,), 0.1)}
    if case["post"]:
        v["w_post"] = _normal(g, (n,), 0.1)
    shape = {"Off": None, "Rows": (m,), "Elements": (m, n), "Channels": (n,)}[case["gate"]]
    if shape:
        v["gate"] = _normal(g, shape)
    if case["scales"]:
        v["scales"] = torch.tensor([0.875, 1.1875], dtype=torch.float32, device="cuda")
    return v


# ---- the library and its buffers ----

_lib = {}


def _open():
    """The process's package, its device context and its engine."""
    if not _lib:
        sys.path.insert(0, os.path.join(os.getcwd(), "herbert-metal-bf16_amd"))
        import herbert_hip as hb
        gpu = hb.Gpu.open()
        _lib["hb"], _lib["gpu"], _lib["engine"] = hb, gpu, hb.Engine(gpu)
    return _lib["hb"], _lib["gpu"], _lib["engine"]


class _View:
    """A library buffer as an array torch can wrap; holds on to its owner."""

    def __init__(self, owner, shape, typestr):
        hb, gpu, _ = _open()
        p = ctypes.c_void_p()
        hb.check(hb.lib.hb_buffer_ptr(gpu.h, owner.id, ctypes.byref(p)))
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (p.value, False), "version": 2}


class _Buf:
    """A device buffer of the library, of the tensor `t`'s size or `shape`."""

    def __init__(self, shape, dtype=torch.bfloat16, t=None):
        _, self.gpu, _ = _open()
        self.shape, self.dtype = tuple(shape), dtype
        size = torch.empty(0, dtype=dtype).element_size()
        self.id = self.gpu.alloc(max(1, int(np.prod(self.shape))) * size)
        if t is not None:
            self.t.copy_(t)

    @property
    def t(self):
        plain = {torch.bfloat16: ("<i2", torch.int16), torch.float32: ("<f4", torch.float32), torch.int32: ("<i4", torch.int32),
                 torch.uint8: ("|u1", torch.uint8)}[self.dtype]
        return torch.as_tensor(_View(self, self.shape, plain[0]), device="cuda").view(self.dtype)

    def __del__(self):
        self.gpu.free(self.id)


def _buf_of(t):
    return _Buf(t.shape, t.dtype, t)


def _packed(codes, scales, k, n, group, count=1):
    """The library's 4-bit weights of natural codes and scales."""
    hb, gpu, _ = _open()
    c, s = _buf_of(codes), _buf_of(scales)
    w = _Buf((hb.q4_bytes(k, n, group) * count,), torch.uint8)
    torch.cuda.synchronize()
    gpu.launch(gpu.pipeline(hb.q4_pack(k, n, group)), [hb.r(c.id), hb.r(s.id), hb.r(w.id)], count)
    gpu.sync()
    return w


def prepare(case, seed):
    v = _inputs(case, seed)
    if own:
        return _prepare_own(case, v)
    return {"case": case, **v}


def _prepare_own(case, v):
    hb, gpu, eng = _open()
    # One stream for torch and the library, as a program that holds tensors
    # over the library's buffers has it: what run gives is in order with what
    # torch does before and after.
    gpu.set_stream(torch.cuda.current_stream().cuda_stream)
    op = case["op"]
    bufs, out = {}, {}
    if op == "matvec":
        k, n, group, m, kind = case["k"], case["n"], case["group"], case["m"], hb.Out[case["out"]]
        bufs["w"] = _packed(v["codes"], v["scales"], k, n, group)
        bufs["x"] = _buf_of(v["x"])
        bufs["y"] = _Buf((m, n // 2 if kind == hb.Out.Swiglu else n), torch.float32 if kind == hb.Out.F32 else torch.bfloat16)
        torch.cuda.synchronize()
        r = {name: hb.r(b.id) for name, b in bufs.items()}
        kern = eng.mv_q4(k, n, kind, group, m, [r["w"]], r["x"], r["y"])
        steps = [(kern, [r["w"], r["x"], r["y"]], m)]
        out["y"] = bufs["y"].t
    elif op == "experts":
        t, group = case["t"], case["group"]
        bufs["gu"] = _packed(v["gu"], v["gs"], MH, 2 * MI, group, EXPERTS)
        bufs["dn"] = _packed(v["dn"], v["ds"], MI, MH, group, EXPERTS)
        for name in ("x", "list", "tiles"):
            bufs[name] = _buf_of(v[name])
        bufs["state"] = _buf_of(torch.tensor([0, 0, 0, t], dtype=torch.int32, device="cuda"))
        bufs["h"], bufs["y"] = _Buf((t * TOP_K, MI)), _Buf((t * TOP_K, MH))
        r = {name: hb.r(b.id) for name, b in bufs.items()}
        gate_up = gpu.pipeline(hb.experts_q4(MH, 2 * MI, hb.Out.Swiglu, group, hb.Rows.Gather, TOP_K, EXPERTS, t))
        down = gpu.pipeline(hb.experts_q4(MI, MH, hb.Out.Bf16, group, hb.Rows.Scatter, TOP_K, EXPERTS, t))
        steps = [(gate_up, [r["state"], r["gu"], r["x"], r["h"], r["list"], r["tiles"]], t),
                 (down, [r["state"], r["dn"], r["h"], r["y"], r["list"], r["tiles"]], t)]
        out["h"], out["y"] = bufs["h"].t, bufs["y"].t
    elif op == "quant":
        k, n, group = case["k"], case["n"], case["group"]
        bufs["w"] = _buf_of(v["w"])
        bufs["q"], bufs["back"] = _Buf((hb.q4_bytes(k, n, group),), torch.uint8), _Buf((n, k))
        r = {name: hb.r(b.id) for name, b in bufs.items()}
        steps = [(gpu.pipeline(hb.q4_quantize(k, n, group)), [r["w"], r["q"]], 1),
                 (gpu.pipeline(hb.q4_dequantize(k, n, group)), [r["q"], r["back"]], 1)]
        out["w"] = bufs["back"].t
    else:
        m, n = case["m"], case["n"]
        bufs = {name: _buf_of(t) for name, t in v.items()}
        bufs["xo"], bufs["h"] = _Buf((m, n)), _Buf((m, n))
        kern = gpu.pipeline(hb.block_norm(n, EPS, plus_one=True, post=case["post"], pre=True, gate=hb.Gate[case["gate"]],
                                          scales=case["scales"]))
        names = ["x", "y", "xo", "h"] + [b for b in ("w_post", "gate", "scales", "w_pre") if b in bufs]
        steps = [(kern, [hb.r(bufs[b].id) for b in names], m)]
        out["x"], out["h"] = bufs["xo"].t, bufs["h"].t
    torch.cuda.synchronize()
    return {"gpu": gpu, "steps": steps, "out": out, "bufs": bufs}


# ---- a pass ----

def _weights(codes, scales, k, group, dtype):
    """The values the codes stand for, [rows][k]."""
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], k).to(dtype) - 8
    return q * scales.to(dtype).repeat_interleave(group, 1)[:, :k]


def _swiglu(g, u):
    return g / (1 + torch.exp(-g)) * u


def _rms(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (w + 1)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "matvec":
        y = s["x"].float() @ _weights(s["codes"], s["scales"], case["k"], case["group"], torch.float32).T
        if case["out"] == "Swiglu":
            y = _swiglu(y[:, :case["n"] // 2], y[:, case["n"] // 2:])
        return {"y": y if case["out"] == "F32" else y.to(torch.bfloat16)}
    if op == "experts":
        # Every row against every expert's weights, then the routed ones.
        row, e = s["list"].long() // TOP_K, s["expert"]
        pairs = torch.arange(len(e), device="cuda")
        w = _weights(s["gu"], s["gs"], MH, case["group"], torch.float32)
        gu = (s["x"].float() @ w.T).reshape(-1, EXPERTS, 2 * MI)[row, e]
        h = _swiglu(gu[:, :MI], gu[:, MI:]).to(torch.bfloat16)
        w = _weights(s["dn"], s["ds"], MI, case["group"], torch.float32)
        y = torch.empty((len(e), MH), dtype=torch.bfloat16, device="cuda")
        y[s["list"].long()] = (h.float() @ w.T).reshape(-1, EXPERTS, MH)[pairs, e].to(torch.bfloat16)
        return {"h": h, "y": y}
    if op == "quant":
        n, k, group = case["n"], case["k"], case["group"]
        w = torch.zeros((n, -(-k // group) * group), dtype=torch.float32, device="cuda")
        w[:, :k] = s["w"]
        w = w.reshape(n, -1, group)
        hi, lo = w.amax(-1, keepdim=True), w.amin(-1, keepdim=True)
        scale = (torch.where(hi >= -lo, hi, lo) / -8).to(torch.bfloat16).float()
        q = torch.where(scale == 0, torch.zeros_like(w), torch.round(w / scale)).clamp(-8, 7)
        return {"w": (q * scale).reshape(n, -1)[:, :k].to(torch.bfloat16).contiguous()}
    x, v = s["x"].float(), s["y"].float()
    if case["post"]:
        v = _rms(v, s["w_post"].float())
    if case["gate"] == "Rows":
        v = v / (1 + torch.exp(-s["gate"].float()[:, None]))
    elif case["gate"] == "Elements":
        v = v / (1 + torch.exp(-s["gate"].float()))
    elif case["gate"] == "Channels":
        v = v * s["gate"].float()
    xo = (x * s["scales"][0] + v * s["scales"][1] if case["scales"] else x + v).to(torch.bfloat16)
    return {"x": xo, "h": _rms(xo.float(), s["w_pre"].float()).to(torch.bfloat16)}


def run(state):
    if own:
        for kern, ranges, m in state["steps"]:
            state["gpu"].launch(kern, ranges, m)
        return state["out"]
    return _run_plain(state)


# ---- what a pass cannot do without ----

def _q4(k, n, group):
    return n * k / 2 + 2.0 * n * -(-k // group)


def work(case):
    op = case["op"]
    if op == "matvec":
        m, k, n = case["m"], case["k"], case["n"]
        y = m * n * (4.0 if case["out"] == "F32" else 1.0 if case["out"] == "Swiglu" else 2.0)
        return {"bytes": _q4(k, n, case["group"]) + 2.0 * m * k + y, "flops": 2.0 * m * n * k}
    if op == "experts":
        t = case["t"]
        hit = EXPERTS * (1.0 - (1.0 - TOP_K / EXPERTS) ** t)  # experts with rows
        per = _q4(MH, 2 * MI, case["group"]) + _q4(MI, MH, case["group"])
        rows = 2.0 * t * MH + 2.0 * t * TOP_K * (2 * MI + MH)
        return {"bytes": hit * per + rows + 4.0 * t * TOP_K, "flops": 2.0 * t * TOP_K * 3 * MI * MH}
    if op == "quant":
        w = 2.0 * case["k"] * case["n"]
        return {"bytes": 2 * w + 2 * _q4(case["k"], case["n"], case["group"]), "flops": 4.0 * case["k"] * case["n"]}
    m, n = case["m"], case["n"]
    gate = {"Off": 0, "Rows": m, "Elements": m * n, "Channels": n}[case["gate"]]
    return {"bytes": 2.0 * (4 * m * n + gate + n * (2 if case["post"] else 1)), "flops": 12.0 * m * n}


# ---- the same in 64 bits ----

def _values64(codes, scales, k, group):
    lo, hi = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    w = torch.empty((codes.shape[0], k), dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = lo - 8, hi - 8
    at = torch.arange(k, device="cuda") // group
    return w.mul_(scales.double()[:, at])


def exact(case, seed):
    v = _inputs(case, seed)
    op = case["op"]
    if op == "matvec":
        n = case["n"]
        parts = [v["x"].double() @ _values64(v["codes"][i:i + 8192], v["scales"][i:i + 8192], case["k"], case["group"]).t()
                 for i in range(0, n, 8192)]
        y = torch.cat(parts, 1)
        if case["out"] == "Swiglu":
            y = y[:, :n // 2] * torch.sigmoid(y[:, :n // 2]) * y[:, n // 2:]
        return {"y": y}
    if op == "experts":
        pairs = len(v["expert"])
        h = torch.empty((pairs, MI), dtype=torch.float64, device="cuda")
        y = torch.empty((pairs, MH), dtype=torch.float64, device="cuda")
        order = v["list"].long()
        for e in v["expert"].unique().tolist():
            p = (v["expert"] == e).nonzero()[:, 0]
            gu = slice(e * 2 * MI, (e + 1) * 2 * MI)
            both = v["x"][order[p] // TOP_K].double() @ _values64(v["gu"][gu], v["gs"][gu], MH, case["group"]).t()
            h[p] = both[:, :MI] * torch.sigmoid(both[:, :MI]) * both[:, MI:]
            dn = slice(e * MH, (e + 1) * MH)
            y[order[p]] = h[p] @ _values64(v["dn"][dn], v["ds"][dn], MI, case["group"]).t()
        return {"h": h, "y": y}
    if op == "quant":
        n, k, group = case["n"], case["k"], case["group"]
        back = torch.empty((n, k), dtype=torch.float64, device="cuda")
        for at in range(0, k, group):
            w = v["w"][:, at:at + group].double()
            above, below = w.max(1, keepdim=True).values, w.min(1, keepdim=True).values
            far = torch.where(above + below < 0, below, above)  # of the largest size
            scale = (-far / 8).to(torch.bfloat16).double()
            q = torch.round(w / scale).clamp(-8, 7)
            back[:, at:at + group] = torch.where(scale == 0, 0.0, q * scale)
        return {"w": back}

    def rms(a, w):
        return a * (a.square().sum(-1, keepdim=True) / a.shape[-1] + EPS).rsqrt() * (1.0 + w.double())

    a, b = v["x"].double(), v["y"].double()
    if case["post"]:
        b = rms(b, v["w_post"])
    if case["gate"] == "Channels":
        b = b * v["gate"].double()
    elif case["gate"] != "Off":
        gate = torch.sigmoid(v["gate"].double())
        b = b * (gate[:, None] if case["gate"] == "Rows" else gate)
    if case["scales"]:
        a, b = a * v["scales"][0].double(), b * v["scales"][1].double()
    a = a + b
    return {"x": a, "h": rms(a, v["w_pre"])}
