"""A router and 8-bit layers, as cases that can be timed and checked: routing
to experts (softmax or sigmoid scores, a bias, groups, top-k, renormalised
weights), bf16 quantised to 8-bit floating point and read back, matrix products
of 8-bit operands with a scale for each block of 128, for few rows and for
many, a whole MLP and the routed experts over 8-bit weights.

8-bit operands: e4m3 codes q and f32 scales s, an element q * s.  A weight
matrix has a scale for each block of 128 x 128, a row of activations one for
each 128 of its elements: with a = max(|largest|, 2^-100), s = a / 448 and q =
the e4m3 nearest to 448 x / a, ties to even.  A product takes its bf16 x, quantises it and
multiplies; sums are f32.  The SwiGLU between two products is bf16, and
quantised as any x.

Each case runs in its plain form, elementary torch operations in 32 bits (the
router's choice in 64, where two experts may stand close), or through the
package (`own`).  The shapes are those of a 4B-class layer (hidden 2560, fused
projections 10240, MLP 9216, vocabulary 151936), of the 27B-class projections (5120,
34816) and of a 35B-A3B-class sparse layer (hidden 2048, 256 experts, top 8,
intermediate 512), and sizes between them that divide by little.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

TINY = 2.0 ** -100
EXPERTS, TOP_K, MH, MI = 256, 8, 2048, 512


def listed():
    return [
        # One token's router: softmax over bf16 scores, the shortest launch.
        {"name": "route_m1", "op": "route", "m": 1, "experts": 256, "top_k": 8, "sigmoid": False, "bias": False,
         "groups": 1, "top_groups": 1, "group_top": 1, "f32": False},
        # A long prompt's router with balance biases and groups of experts.
        {"name": "route_groups_m8192", "op": "route", "m": 8192, "experts": 256, "top_k": 8, "sigmoid": True, "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "f32": True},
        # A short prompt's rows quantised and read back, on a length that no
        # block divides.
        {"name": "quant_rows_m57", "op": "quant_rows", "m": 57, "k": 5008},
        # The 27B-class gate and up quantised at load and read back.
        {"name": "quant_gate_up27", "op": "quant", "k": 5120, "n": 34816},
        # One sequence's output projection: the shortest launch of a decode
        # step, where latency counts.
        {"name": "mv_o_m1", "op": "matvec", "k": 4096, "n": 2560, "out": "Bf16", "m": 1},
        # Four sequences' logits in f32: the largest matrix of a step.
        {"name": "mv_head_m4", "op": "matvec", "k": 2560, "n": 151936, "out": "F32", "m": 4},
        # A large decode batch's fused projection.
        {"name": "gemm_qkv_m48", "op": "gemm", "k": 2560, "n": 10240, "out": "Bf16", "m": 48},
        # A prompt on a shape that no tile divides.
        {"name": "gemm_ragged_m509", "op": "gemm", "k": 5008, "n": 7001, "out": "F32", "m": 509},
        # A long prompt's 27B-class gate and up: the largest product.
        {"name": "gemm_gate_up27_m8192", "op": "gemm", "k": 5120, "n": 34816, "out": "Bf16", "m": 8192},
        # A block of a 4B-class prompt through its MLP.
        {"name": "mlp_m2048", "op": "mlp", "hidden": 2560, "inter": 9216, "m": 2048},
        # The experts of a small decode batch, and of a block of a prompt.
        {"name": "experts_t8", "op": "experts", "t": 8},
        {"name": "experts_t2048", "op": "experts", "t": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "quant_rows", "quant", "matvec", "matvec", "gemm", "gemm", "gemm", "mlp", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 16 // groups), 512 // groups)
        top_groups = rng.randint(max(1, groups // 2), groups)
        return {"op": op, "m": _log(rng, 1, 8192), "experts": experts, "top_k": rng.randint(1, min(10, experts * top_groups // groups)),
                "sigmoid": rng.random() < 0.5, "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_top": rng.choice([1, 2]), "f32": rng.random() < 0.5}
    if op == "quant_rows":
        return {"op": op, "m": _log(rng, 1, 8192), "k": 16 * _log(rng, 32, 1088)}
    if op == "quant":
        return {"op": op, "k": 16 * _log(rng, 32, 320), "n": _log(rng, 512, 34816)}
    if op == "matvec":
        k = 16 * _log(rng, 32, 1088)
        return {"op": op, "k": k, "n": _log(rng, 512, min(65536, 380_000_000 // k)), "out": rng.choice(["Bf16", "F32"]),
                "m": _log(rng, 1, 16)}
    if op == "gemm":
        k, n = 16 * _log(rng, 32, 1088), _log(rng, 512, 18432)
        return {"op": op, "k": k, "n": n, "out": rng.choice(["Bf16", "F32"]), "m": _log(rng, 17, min(8192, 1_400_000_000_000 // (k * n)))}
    if op == "mlp":
        return {"op": op, "hidden": 16 * _log(rng, 32, 320), "inter": 128 * _log(rng, 4, 72), "m": _log(rng, 17, 2048)}
    return {"op": op, "t": _log(rng, 1, 2048)}


# ---- the inputs, from the seed ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62))
    return g


def _activations(g, m, k):
    """N(0, 1) rows with a few channels a tenfold larger, as a model's are."""
    x = torch.empty((m, k), dtype=torch.float32, device="cuda").normal_(0, 1, generator=g)
    big = torch.rand((k,), device="cuda", generator=g) < 0.004
    return (x * torch.where(big, 10.0, 1.0)).to(torch.bfloat16)


def _blocks(n):
    return -(-n // 128)


def _weights8(g, n, k):
    """(codes [n][k] e4m3, scales [blocks][blocks] f32) of normal weights, each
    block's largest near 4.5 deviations."""
    q = torch.empty((n, k), dtype=torch.float16, device="cuda").normal_(0, 96.0, generator=g).clamp_(-448, 448)
    s = torch.empty((_blocks(n), _blocks(k)), dtype=torch.float32, device="cuda").uniform_(1.5e-4, 2.8e-4, generator=g)
    return q.to(torch.float8_e4m3fn), s


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "route":
        # Scores of a trained router: a common part over the tokens, so that
        # some experts are chosen more often; the biases push against it.
        m, e = case["m"], case["experts"]
        common = torch.empty((e,), dtype=torch.float32, device="cuda").normal_(0, 0.7, generator=g)
        s = torch.empty((m, e), dtype=torch.float32, device="cuda").normal_(0, 1.3, generator=g) + common
        v = {"scores": s if case["f32"] else s.to(torch.bfloat16)}
        if case["bias"]:
            v["bias"] = -0.1 * common + torch.empty((e,), dtype=torch.float32, device="cuda").normal_(0, 0.02, generator=g)
        return v
    if op == "quant_rows":
        return {"x": _activations(g, case["m"], case["k"])}
    if op == "quant":
        # Weights whose rows differ in size, as a checkpoint's do.
        w = torch.empty((case["n"], case["k"]), dtype=torch.float32, device="cuda").normal_(0, 0.02, generator=g)
        row = torch.empty((case["n"], 1), dtype=torch.float32, device="cuda").uniform_(0.3, 3.0, generator=g)
        return {"w": w.mul_(row).to(torch.bfloat16)}
    if op in ("matvec", "gemm"):
        w, s = _weights8(g, case["n"], case["k"])
        return {"w": w, "s": s, "x": _activations(g, case["m"], case["k"])}
    if op == "mlp":
        h, i = case["hidden"], case["inter"]
        gu, gs = _weights8(g, 2 * i, h)
        dn, ds = _weights8(g, h, i)
        return {"gu": gu, "gs": gs, "dn": dn, "ds": ds, "x": _activations(g, case["m"], h)}
    t = case["t"]
    gu, gs = _weights8(g, EXPERTS * 2 * MI, MH)
    dn, ds = _weights8(g, EXPERTS * MH, MI)
    x = _activations(g, t, MH)
    scores = torch.empty((t, EXPERTS), dtype=torch.float32, device="cuda").normal_(0, 1, generator=g)
    ids = torch.sort(torch.sort(scores, dim=-1, descending=True, stable=True).indices[:, :TOP_K], dim=-1).values
    return {"gu": gu, "gs": gs, "dn": dn, "ds": ds, "x": x, "ids": ids}


# ---- the library and its buffers ----

_lib = {}


def _open():
    """The process's package and its device context."""
    if not _lib:
        sys.path.insert(0, os.path.join(os.getcwd(), "herbert-metal-bf16_amd"))
        import herbert_hip as hb
        _lib["hb"], _lib["gpu"] = hb, hb.Gpu.open()
    return _lib["hb"], _lib["gpu"]


class _View:
    """A library buffer as an array torch can wrap; holds on to its owner."""

    def __init__(self, owner, shape, typestr):
        hb, gpu = _open()
        p = ctypes.c_void_p()
        hb.check(hb.lib.hb_buffer_ptr(gpu.h, owner.id, ctypes.byref(p)))
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (p.value, False), "version": 2}


class _Buf:
    """A device buffer of the library, of the tensor `t`'s size or `shape`."""

    def __init__(self, shape, dtype=torch.bfloat16, t=None):
        _, self.gpu = _open()
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


def _matrix(codes, scales, k, n, count=1):
    """The library's 8-bit matrices: each its codes, then its scales."""
    hb, _ = _open()
    size = hb.f8_bytes(k, n)
    b = _Buf((count, size), torch.uint8)
    b.t[:, :n * k].copy_(codes.view(torch.uint8).reshape(count, n * k))
    at = scales.numel() // count * 4
    b.t[:, n * k:n * k + at].copy_(scales.view(torch.uint8).reshape(count, at))
    return b


def prepare(case, seed):
    v = _inputs(case, seed)
    if own:
        return _prepare_own(case, v)
    s = {"case": case, **v}
    if case["op"] == "experts":
        # The pairs (row * TOP_K + slot) by expert, and the most of one: what
        # a program that batches the experts' products keeps as its plan.
        flat = v["ids"].reshape(-1)
        s["order"] = torch.sort(flat, stable=True).indices
        s["expert"] = flat[s["order"]]
        count = torch.bincount(flat, minlength=EXPERTS)
        s["at"] = torch.arange(len(flat), device="cuda") - (torch.cumsum(count, 0) - count)[s["expert"]]
        s["cap"] = int(count.max())
    return s


def _prepare_own(case, v):
    hb, gpu = _open()
    # One stream for torch and the library, as a program that holds tensors
    # over the library's buffers has it: what run gives is in order with what
    # torch does before and after.
    gpu.set_stream(torch.cuda.current_stream().cuda_stream)
    op = case["op"]
    bufs, out = {}, {}

    def step(desc, names, m):
        return gpu.pipeline(desc), [hb.r(bufs[b].id) for b in names], m

    if op == "route":
        m, k = case["m"], case["top_k"]
        bufs = {name: _buf_of(t) for name, t in v.items()}
        bufs["route"] = _Buf((m, 2 * k), torch.int32)
        score = hb.Score.Sigmoid if case["sigmoid"] else hb.Score.Softmax
        desc = hb.route_topk(case["experts"], k, score=score, bias=case["bias"], groups=case["groups"], top_groups=case["top_groups"],
                             group_top=case["group_top"], renorm=True, scale=2.5, f32=case["f32"])
        steps = [step(desc, ["scores", "route"] + (["bias"] if case["bias"] else []), m)]
        out["ids"], out["weights"] = bufs["route"].t[:, :k], bufs["route"].t[:, k:].view(torch.float32)
    elif op == "quant_rows":
        m, k = case["m"], case["k"]
        bufs = {"x": _buf_of(v["x"]), "q": _Buf((m, hb.f8_row_bytes(k)), torch.uint8), "back": _Buf((m, k))}
        steps = [step(hb.f8_quantize_rows(k), ["x", "q"], m), step(hb.f8_dequantize_rows(k), ["q", "back"], m)]
        out["x"] = bufs["back"].t
    elif op == "quant":
        k, n = case["k"], case["n"]
        bufs = {"w": _buf_of(v["w"]), "q": _Buf((hb.f8_bytes(k, n),), torch.uint8), "back": _Buf((n, k))}
        steps = [step(hb.f8_quantize(k, n), ["w", "q"], 1), step(hb.f8_dequantize(k, n), ["q", "back"], 1)]
        out["w"] = bufs["back"].t
    elif op in ("matvec", "gemm"):
        k, n, m, kind = case["k"], case["n"], case["m"], hb.Out[case["out"]]
        bufs = {"w": _matrix(v["w"], v["s"], k, n), "x": _buf_of(v["x"]),
                "y": _Buf((m, n), torch.float32 if kind == hb.Out.F32 else torch.bfloat16)}
        if op == "matvec":
            steps = [step(hb.matvec_f8(k, n, kind, mv_m=m), ["w", "x", "y"], m)]
        else:
            bufs["state"] = _buf_of(torch.tensor([0, 0, 0, m], dtype=torch.int32, device="cuda"))
            bufs["x8"] = _Buf((m, hb.f8_row_bytes(k)), torch.uint8)
            steps = [step(hb.f8_quantize_rows(k), ["x", "x8"], m),
                     step(hb.gemm_f8(k, n, kind, rows=m), ["state", "w", "x8", "y", "state", "state"], m)]
        out["y"] = bufs["y"].t
    elif op == "mlp":
        h, i, m = case["hidden"], case["inter"], case["m"]
        bufs = {"gu": _matrix(v["gu"], v["gs"], h, 2 * i), "dn": _matrix(v["dn"], v["ds"], i, h), "x": _buf_of(v["x"]),
                "x8": _Buf((m, hb.f8_row_bytes(h)), torch.uint8), "h8": _Buf((m, hb.f8_row_bytes(i)), torch.uint8), "y": _Buf((m, h)),
                "state": _buf_of(torch.tensor([0, 0, 0, m], dtype=torch.int32, device="cuda"))}
        steps = [step(hb.f8_quantize_rows(h), ["x", "x8"], m),
                 step(hb.gemm_f8(h, 2 * i, hb.Out.Swiglu, rows=m), ["state", "gu", "x8", "h8", "state", "state"], m),
                 step(hb.gemm_f8(i, h, hb.Out.Bf16, rows=m), ["state", "dn", "h8", "y", "state", "state"], m)]
        out["y"] = bufs["y"].t
    else:
        t = case["t"]
        pairs, bm = t * TOP_K, hb.f8_tile_rows(t, TOP_K, EXPERTS)
        bufs = {"gu": _matrix(v["gu"], v["gs"], MH, 2 * MI, EXPERTS), "dn": _matrix(v["dn"], v["ds"], MI, MH, EXPERTS),
                "x": _buf_of(v["x"]), "state": _buf_of(torch.tensor([0, 0, 0, t], dtype=torch.int32, device="cuda")),
                "list": _Buf((pairs,), torch.int32), "tiles": _Buf((1 + 3 * hb.moe_tiles(t, TOP_K, EXPERTS, bm),), torch.int32),
                "y": _Buf((pairs, MH))}
        route = torch.zeros((t, 2 * TOP_K), dtype=torch.int32, device="cuda")
        route[:, :TOP_K] = v["ids"]
        bufs["route"] = _buf_of(route)
        k, r, n = step(hb.Desc(kind=hb.Kind.SORT, experts=EXPERTS, top_k=TOP_K, bm=bm, rows_max=t), ["state", "route", "list", "tiles"], t)
        torch.cuda.synchronize()
        gpu.launch(k, r, n)
        steps, xin = [], "x"
        if bm > 16:
            # Tiles of more rows take x and h as 8-bit rows.
            bufs["x8"], bufs["h"] = _Buf((t, hb.f8_row_bytes(MH)), torch.uint8), _Buf((pairs, hb.f8_row_bytes(MI)), torch.uint8)
            steps, xin = [step(hb.f8_quantize_rows(MH), ["x", "x8"], t)], "x8"
        else:
            bufs["h"] = _Buf((pairs, MI))
        steps += [step(hb.experts_f8(MH, 2 * MI, hb.Out.Swiglu, hb.Rows.Gather, TOP_K, EXPERTS, t, bm),
                       ["state", "gu", xin, "h", "list", "tiles"], t),
                  step(hb.experts_f8(MI, MH, hb.Out.Bf16, hb.Rows.Scatter, TOP_K, EXPERTS, t, bm),
                       ["state", "dn", "h", "y", "list", "tiles"], t)]
        out["y"] = bufs["y"].t
    torch.cuda.synchronize()
    return {"gpu": gpu, "steps": steps, "out": out, "bufs": bufs}


# ---- a pass ----

def _quantized(x):
    """The values that x's rows stand for in 8 bits, f32."""
    m, k = x.shape
    v = torch.zeros((m, _blocks(k) * 128), dtype=torch.float32, device=x.device)
    v[:, :k] = x
    v = v.reshape(m, -1, 128)
    big = v.abs().amax(-1, keepdim=True).clamp_min(TINY)
    q = (v * 448.0 / big).to(torch.float8_e4m3fn).float()
    return (q * (big / 448.0)).reshape(m, -1)[:, :k]


def _weights(codes, scales, n, k):
    """The values of matrices of n rows of k, f32."""
    s = scales.reshape(-1, _blocks(n), _blocks(k))
    s = s.repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
    return codes.float().reshape(-1, n, k) * s


def _swiglu(g, u):
    return g / (1 + torch.exp(-g)) * u


def _run_route(s):
    case, x = s["case"], s["scores"].double()
    e, groups, k = case["experts"], case["groups"], case["top_k"]
    if case["sigmoid"]:
        p = 1 / (1 + torch.exp(-x))
    else:
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    c = p + s["bias"].double() if case["bias"] else p
    if groups > 1:
        best = torch.sort(c.reshape(-1, groups, e // groups), dim=-1, descending=True).values[:, :, :case["group_top"]].sum(-1)
        keep = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        live = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True).repeat_interleave(e // groups, 1)
        c = torch.where(live, c, torch.full_like(c, -math.inf))
    ids = torch.sort(torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k], dim=-1).values
    w = torch.gather(p, 1, ids)
    return {"ids": ids.to(torch.int32), "weights": (w / w.sum(-1, keepdim=True) * 2.5).float()}


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _run_route(s)
    if op == "quant_rows":
        return {"x": _quantized(s["x"]).to(torch.bfloat16)}
    if op == "quant":
        n, k = case["n"], case["k"]
        w = torch.zeros((_blocks(n) * 128, _blocks(k) * 128), dtype=torch.float32, device="cuda")
        w[:n, :k] = s["w"]
        w = w.reshape(_blocks(n), 128, _blocks(k), 128)
        big = w.abs().amax((1, 3), keepdim=True).clamp_min(TINY)
        q = (w * 448.0 / big).to(torch.float8_e4m3fn).float()
        return {"w": (q * (big / 448.0)).reshape(_blocks(n) * 128, -1)[:n, :k].to(torch.bfloat16).contiguous()}
    if op in ("matvec", "gemm"):
        y = _quantized(s["x"]) @ _weights(s["w"], s["s"], case["n"], case["k"])[0].T
        return {"y": y if case["out"] == "F32" else y.to(torch.bfloat16)}
    if op == "mlp":
        h, i = case["hidden"], case["inter"]
        gu = _quantized(s["x"]) @ _weights(s["gu"], s["gs"], 2 * i, h)[0].T
        hh = _quantized(_swiglu(gu[:, :i], gu[:, i:]).to(torch.bfloat16))
        return {"y": (hh @ _weights(s["dn"], s["ds"], h, i)[0].T).to(torch.bfloat16)}
    # The experts: each one's rows in a batch padded to the most of one.
    order, e, at, cap = s["order"], s["expert"], s["at"], s["cap"]
    x = torch.zeros((EXPERTS, cap, MH), dtype=torch.float32, device="cuda")
    x[e, at] = _quantized(s["x"])[order // TOP_K]
    gu = torch.bmm(_weights(s["gu"], s["gs"], 2 * MI, MH), x.transpose(1, 2).contiguous())
    gu = gu.transpose(1, 2)[e, at]
    h = torch.zeros((EXPERTS, cap, MI), dtype=torch.float32, device="cuda")
    hq = _quantized(_swiglu(gu[:, :MI], gu[:, MI:]).to(torch.bfloat16))
    h[e, at] = hq
    y = torch.empty((len(e), MH), dtype=torch.bfloat16, device="cuda")
    d = torch.bmm(_weights(s["dn"], s["ds"], MH, MI), h.transpose(1, 2).contiguous())
    y[order] = d.transpose(1, 2)[e, at].to(torch.bfloat16)
    return {"y": y}


def run(state):
    if own:
        for kern, ranges, m in state["steps"]:
            state["gpu"].launch(kern, ranges, m)
        return state["out"]
    return _run_plain(state)


# ---- what a pass cannot do without ----

def _f8(k, n):
    return n * k + 4.0 * _blocks(n) * _blocks(k)


def work(case):
    op = case["op"]
    if op == "route":
        m, e = case["m"], case["experts"]
        return {"bytes": m * e * (4.0 if case["f32"] else 2.0) + 8.0 * m * case["top_k"] + (4.0 * e if case["bias"] else 0.0),
                "flops": 4.0 * m * e}
    if op == "quant_rows":
        m, k = case["m"], case["k"]
        return {"bytes": 2.0 * (2.0 * m * k + m * k + 4.0 * m * _blocks(k)), "flops": 4.0 * m * k}
    if op == "quant":
        k, n = case["k"], case["n"]
        return {"bytes": 2.0 * (2.0 * n * k + _f8(k, n)), "flops": 4.0 * n * k}
    if op in ("matvec", "gemm"):
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": _f8(k, n) + 2.0 * m * k + m * n * (4.0 if case["out"] == "F32" else 2.0), "flops": 2.0 * m * n * k}
    if op == "mlp":
        m, h, i = case["m"], case["hidden"], case["inter"]
        return {"bytes": _f8(h, 2 * i) + _f8(i, h) + 4.0 * m * h, "flops": 6.0 * m * h * i}
    t = case["t"]
    hit = EXPERTS * (1.0 - (1.0 - TOP_K / EXPERTS) ** t)  # experts with rows
    return {"bytes": hit * (_f8(MH, 2 * MI) + _f8(MI, MH)) + 2.0 * t * MH + 2.0 * t * TOP_K * MH + 4.0 * t * TOP_K,
            "flops": 2.0 * t * TOP_K * 3 * MI * MH}


# ---- the same in 64 bits ----

def _e4m3_64(v):
    """v rounded to e4m3, ties to even: steps of 2^(e - 3), e no less than -6."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _rows_64(x):
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], 128):
        part = x[:, at:at + 128]
        top = part.abs().max(1, keepdim=True).values.clamp(min=TINY)
        out[:, at:at + 128] = _e4m3_64(448 * part / top) * (top / 448)
    return out


def _values_64(codes, scales, first, last):
    """Rows first..last - 1 of one matrix in 64 bits."""
    row = torch.arange(first, last, device="cuda") // 128
    col = torch.arange(codes.shape[1], device="cuda") // 128
    return codes[first:last].double() * scales.double()[row][:, col]


def _product_64(x, codes, scales):
    n = codes.shape[0]
    return torch.cat([x @ _values_64(codes, scales, i, min(i + 8192, n)).t() for i in range(0, n, 8192)], 1)


def _mlp_64(x, gu, gs, dn, ds):
    both = _product_64(_rows_64(x), gu, gs)
    i = both.shape[1] // 2
    h = (both[:, :i] * torch.sigmoid(both[:, :i]) * both[:, i:]).to(torch.bfloat16)
    return _product_64(_rows_64(h), dn, ds)


def exact(case, seed):
    v = _inputs(case, seed)
    op = case["op"]
    if op == "route":
        s, e, groups = v["scores"].double(), case["experts"], case["groups"]
        p = torch.sigmoid(s) if case["sigmoid"] else torch.softmax(s, -1)
        c = p.clone()
        if case["bias"]:
            c += v["bias"].double()
        index = torch.arange(e, device="cuda")
        if groups > 1:
            size = e // groups
            total = c.reshape(-1, groups, size).topk(min(case["group_top"], size), -1).values.sum(-1)
            # A group stays if fewer than top_groups stand before it.
            a, b = total[:, :, None], total[:, None, :]
            first = index[:groups]
            before = ((b > a) | ((b == a) & (first[None, None, :] < first[None, :, None]))).sum(-1)
            c[(before >= case["top_groups"])[:, index // size]] = -math.inf
        ids = []
        for _ in range(case["top_k"]):
            best = c.amax(-1, keepdim=True)
            i = torch.where(c == best, index, e).amin(-1, keepdim=True)
            c.scatter_(1, i, -math.inf)
            ids.append(i)
        ids = torch.cat(ids, 1).sort(-1).values
        w = p.gather(1, ids)
        return {"ids": ids.to(torch.int32), "weights": 2.5 * w / w.sum(-1, keepdim=True)}
    if op == "quant_rows":
        return {"x": _rows_64(v["x"])}
    if op == "quant":
        back = torch.empty((case["n"], case["k"]), dtype=torch.float64, device="cuda")
        for i in range(0, case["n"], 128):
            w = v["w"][i:i + 128].double()
            for at in range(0, case["k"], 128 * 64):
                part = torch.nn.functional.pad(w[:, at:at + 128 * 64], (0, -w[:, at:at + 128 * 64].shape[1] % 128))
                part = part.reshape(w.shape[0], -1, 128)
                top = part.abs().amax((0, 2), keepdim=True).clamp(min=TINY)
                got = (_e4m3_64(448 * part / top) * (top / 448)).reshape(w.shape[0], -1)
                back[i:i + 128, at:at + 128 * 64] = got[:, :min(128 * 64, case["k"] - at)]
        return {"w": back}
    if op in ("matvec", "gemm"):
        return {"y": _product_64(_rows_64(v["x"]), v["w"], v["s"])}
    if op == "mlp":
        return {"y": _mlp_64(v["x"], v["gu"], v["gs"], v["dn"], v["ds"])}
    y = torch.empty((case["t"] * TOP_K, MH), dtype=torch.float64, device="cuda")
    ids = v["ids"].reshape(-1)
    for e in ids.unique().tolist():
        p = (ids == e).nonzero()[:, 0]
        gu, dn = slice(e * 2 * MI, (e + 1) * 2 * MI), slice(e * MH, (e + 1) * MH)
        gs, ds = slice(e * (2 * MI // 128), (e + 1) * (2 * MI // 128)), slice(e * (MH // 128), (e + 1) * (MH // 128))
        y[p] = _mlp_64(v["x"][p // TOP_K], v["gu"][gu], v["gs"][gs], v["dn"][dn], v["ds"][ds])
    return {"y": y}
