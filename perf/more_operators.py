"""Operators of a gated transformer layer's training step and of its single tokens, as cases that can be
prepared, run, priced and checked.

Three kinds of call through the Python binding of the C ABI:

  rope   RMS norm of each head of q and k with the position rotation in the same pass, forward (for new
         tokens also into their rows of a k/v cache: "step") and backward with the gradients of the gains
  gate   gated product act(X Wg^T + bg) * (X Wu^T + bu), forward; backward with the gradients of input,
         weights and biases
  clip   global norm of many gradient tensors of several types, averaged and clipped

`run` computes them with elementary torch operations, or, where `own` is set, with the framework's kernels.
Sizes: the model of the benchmark (heads of 64 x 24, width 1536, FFN 6144, 64 memory + 1024 latent tokens)
and the ranges around them.
"""
import importlib.util
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of eight sequences: q for the attention, k and v into the caches
        dict(name="rope_step_bf16_b8_h32_8_d128", kind="rope", dir="step", type="bf16", batch=8, tokens=1, heads=32, kv=8,
             dim=128, rot=128, near=False, cache=1024, far=0, ragged=False),
        # the benchmark model's heads in its micro-batch
        dict(name="rope_fwd_bf16_b2_h24_s1088_d64", kind="rope", dir="fwd", type="bf16", batch=2, tokens=1088, heads=24, kv=24,
             dim=64, rot=32, near=False, cache=0, far=0, ragged=False),
        # a long sequence with grouped heads, far from position 0
        dict(name="rope_fwd_f16_b1_h32_8_s8192_d128", kind="rope", dir="fwd", type="f16", batch=1, tokens=8192, heads=32, kv=8,
             dim=128, rot=128, near=True, cache=0, far=1000000, ragged=False),
        # training of the benchmark model's heads
        dict(name="rope_bwd_bf16_b2_h24_s1088_d64", kind="rope", dir="bwd", type="bf16", batch=2, tokens=1088, heads=24, kv=24,
             dim=64, rot=32, near=False, cache=0, far=0, ragged=False),
        # training on a padded batch with grouped heads, in f32
        dict(name="rope_bwd_f32_b3_h16_2_s2049_d128", kind="rope", dir="bwd", type="f32", batch=3, tokens=2049, heads=16, kv=2,
             dim=128, rot=64, near=False, cache=0, far=0, ragged=True),
        # one token through a gated FFN
        dict(name="gate_fwd_bf16_1x1536x6144_silu", kind="gate", dir="fwd", type="bf16", m=1, k=1536, n=6144, act="silu",
             bias=False, keep=False),
        # the micro-batch's gated FFN as training runs it
        dict(name="gate_fwd_bf16_2176x1536x6144_silu", kind="gate", dir="fwd", type="bf16", m=2176, k=1536, n=6144, act="silu",
             bias=True, keep=True),
        # a large layer's
        dict(name="gate_fwd_f16_8191x4096x8192_gelu_tanh", kind="gate", dir="fwd", type="f16", m=8191, k=4096, n=8192,
             act="gelu_tanh", bias=False, keep=False),
        # the micro-batch's backward
        dict(name="gate_bwd_bf16_2176x1536x6144_silu", kind="gate", dir="bwd", type="bf16", m=2176, k=1536, n=6144, act="silu",
             bias=True, keep=True),
        # widths that no alignment helps
        dict(name="gate_bwd_f16_1031x1001x2731_gelu", kind="gate", dir="bwd", type="f16", m=1031, k=1001, n=2731, act="gelu",
             bias=True, keep=True),
        # the benchmark model's adapters (self.qkv, self.out, ff.proj, ff.out of 24 blocks at rank 32), a tensor each
        dict(name="clip_f32_288_adapters", kind="clip", set="adapters", seed=0, count=4, clip=1.0, packed=False),
        # the weights of twelve gated layers in bf16, their gains in f32
        dict(name="clip_bf16_12_layers", kind="clip", set="layers", seed=0, count=1, clip=1.0, packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["rope", "gate", "clip"], [5, 5, 2])[0]
    if kind == "rope":
        d = rng.choice(["fwd", "fwd", "step", "bwd", "bwd"])
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 3, 4, 8, 24])
        heads = kv * (rng.choice([1, 2, 4, 8]) if kv < 24 else 1)
        batch = rng.randint(1, 8)
        tokens = rng.choice([1, 1, 1, 2, 5]) if d == "step" else _log(rng, 1, 16384)
        tokens = max(1, min(tokens, 8192 * 5000 // (batch * (heads + kv) * dim)))
        return dict(kind=kind, dir=d, type=rng.choice(["bf16", "f16", "f32"]), batch=batch, tokens=tokens, heads=heads, kv=kv,
                    dim=dim, rot=rng.choice([0, 16, dim // 32 * 16, dim]), near=rng.random() < 0.4,
                    cache=_log(rng, 16, 1024) if d == "step" else 0, far=rng.choice([0, 0, 5000, 1000000]),
                    ragged=d != "step" and rng.random() < 0.5)
    if kind == "gate":
        m, k, n = _log(rng, 1, 3500), _log(rng, 16, 6144), _log(rng, 16, 6144)
        if rng.random() < 0.75:
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        d = rng.choice(["fwd", "bwd"])
        return dict(kind=kind, dir=d, type=rng.choice(["bf16", "f16"]), m=m, k=k, n=n,
                    act=rng.choice(["none", "relu", "silu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.5,
                    keep=d == "bwd" or rng.random() < 0.5)
    return dict(kind=kind, set="drawn", seed=rng.randrange(1 << 30), count=rng.choice([1, 1, 3, 8]),
                clip=rng.choice([0.0, 1.0, 1.0, 1.0, 1e6]), packed=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------- binding
def _binding():
    if "sa3k" not in sys.modules:
        spec = importlib.util.spec_from_file_location("sa3k", os.path.join(ROOT, "sa3.cpp_amd", "sa3k.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["sa3k"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["sa3k"]


def _code(name):
    k = _binding()
    return {"f32": k.TYPE_F32, "f16": k.TYPE_F16, "bf16": k.TYPE_BF16}[name]


_CTX = []


def _ctx():
    """the program's one context"""
    if not _CTX:
        _CTX.append(_binding().Context(0))
    return _CTX[0]


class _Ref:
    """a tensor's device address, as the binding takes it (the tensor keeps its memory)"""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _ref(t):
    return None if t is None else _Ref(t)


class _State:
    """what a program keeps between calls"""

    plan = None
    closes = False   # the plan has a handle to release

    def __del__(self):
        if self.closes and self.plan is not None:
            self.plan.destroy()


class _Draw:
    """seeded tensors on the GPU, in the order they are asked for"""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, shape, sd=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, sd, generator=self.g).to(dtype)

    def ints(self, lo, hi, shape):
        return torch.randint(lo, hi, shape, device="cuda", dtype=torch.int32, generator=self.g)


# ------------------------------------------------------------------------------- head norm, rotation
EPS, BASE = 1e-6, 1e4


def _lens(c):
    """tokens of each sample: all, or from all down to half of them"""
    return [c["tokens"] - (b * c["tokens"]) // (2 * c["batch"]) if c["ragged"] else c["tokens"] for b in range(c["batch"])]


def _rope_inputs(case, seed):
    c, d, t, s = case, _Draw(seed), TYPES[case["type"]], _State()
    B, S, H, K, D = c["batch"], c["tokens"], c["heads"], c["kv"], c["dim"]
    s.qkv = d.normal((B, S, H + 2 * K, D), 1.5, 0.0, t)   # the projection's output, the heads beside each other
    s.q, s.k, s.v = s.qkv[:, :, :H], s.qkv[:, :, H:H + K], s.qkv[:, :, H + K:]
    s.gq, s.gk = d.normal((D,), 0.2, 1.0), d.normal((D,), 0.2, 1.0)
    s.len = torch.tensor(_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    i = torch.arange(S, device="cuda", dtype=torch.int32)[None, :]
    if c["dir"] == "step":   # the samples' caches are filled to different lengths; the new tokens come behind that
        S0 = min(S, c["cache"])
        start = d.ints(0, c["cache"] - S0 + 1, (B, 1))
        s.slot = (start + i).contiguous()
        s.pos = (s.slot + c["far"]).contiguous()
    else:
        s.slot = None
        s.pos = (d.ints(0, c["far"] + 1, (B, 1)) + i).contiguous() if c["far"] else None   # none: 0, 1, 2, ..
    s.dq, s.dk = (d.normal((B, S, n, D), 1.0, 0.0, t) for n in (H, K)) if c["dir"] == "bwd" else (None, None)
    return s


def _prepare_rope(case, seed):
    c, s = case, _rope_inputs(case, seed)
    B, S, H, K, D = c["batch"], c["tokens"], c["heads"], c["kv"], c["dim"]
    if c["dir"] == "bwd":
        s.dqkv = torch.zeros_like(s.qkv)   # (dv is written there by the attention's backward)
        s.dgq, s.dgk = torch.empty_like(s.gq), torch.empty_like(s.gk)
    else:
        s.yq = torch.zeros((B, S, H, D), device="cuda", dtype=s.q.dtype)
        if c["dir"] == "step":
            s.yk, s.yv = (torch.zeros((B, K, c["cache"], D), device="cuda", dtype=s.q.dtype).transpose(1, 2) for _ in range(2))
        else:
            s.yk, s.yv = torch.zeros((B, S, K, D), device="cuda", dtype=s.q.dtype), None
    return s


def _strides(t):
    """(sample, token, head) strides of [B][S][H][D]"""
    return t.stride(0), t.stride(1), t.stride(2)


def _turns(c, s):
    """cos and sin [B or 1][S][1][rot / 2] in f32, of angles in 64 bits"""
    i = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64)
    freq = torch.pow(torch.tensor(BASE, device="cuda", dtype=torch.float64), -2.0 * i / max(c["rot"], 1))
    pos = torch.arange(c["tokens"], device="cuda")[None] if s.pos is None else s.pos
    a = (pos.double()[:, :, None] * freq)[:, :, None, :]
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(c, x, cs, sn):
    """x [B][S][H][D] in f32 with the pairs of its first dims turned"""
    r = c["rot"]
    if r == 0:
        return x
    y = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["near"] else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * cs - x[..., b] * sn
    y[..., b] = x[..., b] * cs + x[..., a] * sn
    return y


def _rows(c):
    """[B][S][1][1]: whether a token is in its sequence"""
    return (torch.arange(c["tokens"], device="cuda")[None] < torch.tensor(_lens(c), device="cuda")[:, None])[:, :, None, None]


def _run_rope(s):
    c = s.case
    B, S, H, K, D = c["batch"], c["tokens"], c["heads"], c["kv"], c["dim"]
    if own:
        k = _binding()
        if s.plan is None:   # the shape is set up once
            out = dict(q_out_strides=_strides(s.yq), k_out_strides=_strides(s.yk)) if c["dir"] != "bwd" else {}
            if c["dir"] == "step":
                out["v_out_strides"] = _strides(s.yv)
            s.plan = k.HeadNorm(_ctx(), _code(c["type"]), B, S, H, K, D, c["rot"], neighbours=c["near"], eps=EPS, rope_base=BASE,
                                cache_tokens=c["cache"], q_strides=_strides(s.q), k_strides=_strides(s.k),
                                v_strides=_strides(s.v), **out)
        if c["dir"] == "bwd":
            dq, dk = s.dqkv[:, :, :H], s.dqkv[:, :, H:H + K]
            s.plan.backward(_Ref(s.q), _Ref(s.k), _Ref(s.dq), _Ref(s.dk), _Ref(s.gq), _Ref(s.gk), _Ref(dq), _Ref(dk),
                            dq_gain=_Ref(s.dgq), dk_gain=_Ref(s.dgk), pos=_ref(s.pos), len=_ref(s.len))
            return [s.dqkv, s.dgq, s.dgk]
        step = c["dir"] == "step"
        s.plan.forward(_Ref(s.q), _Ref(s.k), _Ref(s.gq), _Ref(s.gk), _Ref(s.yq), _Ref(s.yk), v=_Ref(s.v) if step else None,
                       v_out=_ref(s.yv), pos=_ref(s.pos), slot=_ref(s.slot), len=_ref(s.len))
        return [s.yq, s.yk] + ([s.yv] if step else [])
    cs, sn = _turns(c, s)
    if c["dir"] == "bwd":
        row, outs = _rows(c), []
        for x, dy, gain in ((s.q, s.dq, s.gq), (s.k, s.dk, s.gk)):
            x = x.float()
            xh = x * torch.rsqrt(x.square().mean(3, keepdim=True) + EPS)
            r = torch.rsqrt(x.square().mean(3, keepdim=True) + EPS)
            w = torch.where(row, _rotate(c, dy.float(), cs, -sn), torch.zeros_like(x))
            h = w * gain
            outs.append((r * (h - xh * (h * xh).mean(3, keepdim=True)), (w * xh).sum((0, 1, 2), dtype=torch.float64).float()))
        (dq, dgq), (dk, dgk) = outs
        return [torch.cat([dq, dk, torch.zeros_like(dk)], 2).to(s.q.dtype), dgq, dgk]
    ys = []
    for x, gain in ((s.q, s.gq), (s.k, s.gk)):
        x = x.float()
        n = x * torch.rsqrt(x.square().mean(3, keepdim=True) + EPS) * gain
        ys.append(_rotate(c, n, cs, sn).to(s.q.dtype))
    if c["dir"] == "step":
        b = torch.arange(B, device="cuda")[:, None]
        ok = s.slot < c["cache"]   # (a cache shorter than the step takes what it has rows for)
        b, sl = b.expand_as(s.slot)[ok], s.slot.long()[ok]
        s.yk[b, sl], s.yv[b, sl] = ys[1][ok], s.v[ok]
        s.yq.copy_(ys[0])
        return [s.yq, s.yk, s.yv]
    row = _rows(c)
    return [torch.where(row, y, old) for y, old in zip(ys, (s.yq, s.yk))]   # rows behind a sequence are left as they were


def _exact_rope(case, seed):
    """by complex numbers, the gradients by differentiation"""
    c, s = case, _rope_inputs(case, seed)
    r, n = c["rot"], c["batch"] * c["tokens"] * (c["heads"] + c["kv"]) * c["dim"]
    if n > 3e8:
        return None
    pos = (torch.arange(c["tokens"], device="cuda").expand(c["batch"], -1) if s.pos is None else s.pos).double()
    e = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                    pos[:, :, None, None] * BASE ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / max(r, 1)))

    def head(x, gain):
        y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * gain
        if r == 0:
            return y
        p = y[..., :r].reshape(*y.shape[:3], r // 2, 2) if c["near"] else torch.stack(y[..., :r].chunk(2, -1), -1)
        z = torch.view_as_real(torch.view_as_complex(p.contiguous()) * e)
        z = z.flatten(-2) if c["near"] else torch.cat([z[..., 0], z[..., 1]], -1)
        return torch.cat([z, y[..., r:]], -1)

    row = _rows(c).double()
    if c["dir"] == "bwd":
        leaves = [t.double().requires_grad_() for t in (s.q, s.k, s.gq, s.gk)]
        ((head(leaves[0], leaves[2]) * s.dq.double() * row).sum() + (head(leaves[1], leaves[3]) * s.dk.double() * row).sum()).backward()
        gq, gk = leaves[0].grad, leaves[1].grad
        return [torch.cat([gq, gk, torch.zeros_like(gk)], 2), leaves[2].grad, leaves[3].grad]
    yq, yk = head(s.q.double(), s.gq.double()) * row, head(s.k.double(), s.gk.double()) * row
    if c["dir"] == "fwd":
        return [yq, yk]
    kc = torch.zeros((c["batch"], c["cache"], c["kv"], c["dim"]), device="cuda", dtype=torch.float64)
    vc = torch.zeros_like(kc)
    for b in range(c["batch"]):
        for i, at in enumerate(s.slot[b].tolist()):
            if at < c["cache"]:
                kc[b, at], vc[b, at] = yk[b, i], s.v[b, i].double()
    return [yq, kc, vc]


def _work_rope(c):
    el = 4.0 if c["type"] == "f32" else 2.0
    rows = sum(_lens(c))
    n = rows * (c["heads"] + c["kv"]) * c["dim"]
    if c["dir"] == "bwd":
        return {"bytes": 3.0 * el * n + 16.0 * c["dim"], "flops": 16.0 * n}
    v = rows * c["kv"] * c["dim"] if c["dir"] == "step" else 0
    return {"bytes": 2.0 * el * (n + v) + 8.0 * c["dim"] + 4.0 * rows, "flops": 8.0 * n}


# ---------------------------------------------------------------------------------- gated product
def _gate_inputs(case, seed):
    c, d, t, s = case, _Draw(seed), TYPES[case["type"]], _State()
    m, k, n = c["m"], c["k"], c["n"]
    s.x = d.normal((m, k), 1.0, 0.0, t)
    s.wg, s.wu = (d.normal((n, k), k ** -0.5, 0.0, t) for _ in range(2))
    s.bg, s.bu = (d.normal((n,), 0.1) for _ in range(2)) if c["bias"] else (None, None)
    if c["dir"] == "bwd":   # what a forward kept
        s.g, s.u = (_affine(s.x, w, b).to(t) for w, b in ((s.wg, s.bg), (s.wu, s.bu)))
        s.dy = d.normal((m, n), 1.0, 0.0, t)
    return s


def _affine(x, w, b):
    z = torch.matmul(x.float(), w.float().t())
    return z if b is None else z + b


def _prepare_gate(case, seed):
    s = _gate_inputs(case, seed)
    if case["dir"] == "fwd":
        s.y = torch.empty((case["m"], case["n"]), device="cuda", dtype=s.x.dtype)
        s.g, s.u = (torch.empty_like(s.y) for _ in range(2)) if case["keep"] else (None, None)
    else:
        s.dx, s.dwg, s.dwu = torch.empty_like(s.x), torch.empty_like(s.wg), torch.empty_like(s.wu)
        s.dbg, s.dbu = (torch.empty(case["n"], device="cuda") for _ in range(2)) if case["bias"] else (None, None)
    return s


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _run_gate(s):
    c = s.case
    if own:
        k = _binding()
        act = {"none": k.ACT_NONE, "relu": k.ACT_RELU, "silu": k.ACT_SILU, "gelu": k.ACT_GELU,
               "gelu_tanh": k.ACT_GELU_TANH}[c["act"]]
        if c["dir"] == "fwd":
            k.gated_linear_fwd(_ctx(), _code(c["type"]), act, _Ref(s.x), _Ref(s.wg), _Ref(s.wu), c["m"], c["n"], c["k"],
                               _Ref(s.y), gate_bias=_ref(s.bg), up_bias=_ref(s.bu), gate=_ref(s.g), up=_ref(s.u))
            return [s.y] + ([s.g, s.u] if c["keep"] else [])
        k.gated_linear_bwd(_ctx(), _code(c["type"]), act, _Ref(s.dy), _Ref(s.g), _Ref(s.u), _Ref(s.x), _Ref(s.wg), _Ref(s.wu),
                           c["m"], c["n"], c["k"], dx=_Ref(s.dx), dw_gate=_Ref(s.dwg), dw_up=_Ref(s.dwu),
                           db_gate=_ref(s.dbg), db_up=_ref(s.dbu))
        return [s.dx, s.dwg, s.dwu] + ([s.dbg, s.dbu] if c["bias"] else [])
    t = s.x.dtype
    if c["dir"] == "fwd":
        g, u = _affine(s.x, s.wg, s.bg), _affine(s.x, s.wu, s.bu)
        y = (_act(g, c["act"]) * u).to(t)
        return [y] + ([g.to(t), u.to(t)] if c["keep"] else [])
    x, dy, g, u = s.x.float(), s.dy.float(), s.g.float(), s.u.float()
    dg, du = dy * u * _act_slope(g, c["act"]), dy * _act(g, c["act"])
    dx = torch.matmul(dg, s.wg.float()) + torch.matmul(du, s.wu.float())
    out = [dx.to(t), torch.matmul(dg.t(), x).to(t), torch.matmul(du.t(), x).to(t)]
    return out + ([dg.sum(0), du.sum(0)] if c["bias"] else [])


def _exact_gate(case, seed):
    c, s = case, _gate_inputs(case, seed)
    f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[c["act"]]
    x, wg, wu = s.x.double(), s.wg.double(), s.wu.double()
    if c["dir"] == "fwd":
        zero = torch.zeros((), device="cuda", dtype=torch.float64)
        g = torch.addmm(s.bg.double() if c["bias"] else zero, x, wg.t())
        u = torch.addmm(s.bu.double() if c["bias"] else zero, x, wu.t())
        return [f(g) * u] + ([g, u] if c["keep"] else [])
    g, u = s.g.double().requires_grad_(), s.u.double().requires_grad_()
    (f(g) * u).backward(s.dy.double())
    out = [torch.cat([g.grad, u.grad], 1) @ torch.cat([wg, wu]), g.grad.t() @ x, u.grad.t() @ x]
    return out + ([g.grad.sum(0), u.grad.sum(0)] if c["bias"] else [])


def _work_gate(c):
    m, n, k = float(c["m"]), float(c["n"]), float(c["k"])
    b = 8 * n if c["bias"] else 0.0
    if c["dir"] == "fwd":
        return {"bytes": 2 * (m * k + 2 * n * k + m * n * (3 if c["keep"] else 1)) + b, "flops": 4 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 4 * n * k + 3 * m * n) + b, "flops": 8 * m * n * k}


# -------------------------------------------------------------------------------- many gradients
def _tensors(c):
    """[(elements, type)] of a case's gradients"""
    if c["set"] == "adapters":
        out = []
        for _ in range(24):
            for i, o in ((1536, 7680), (1536, 1536), (1536, 12288), (6144, 1536)):
                out += [(32 * i, "f32"), (32 * o, "f32"), (o, "f32")]   # A, B, magnitude
        return out
    if c["set"] == "layers":
        out = []
        for _ in range(12):
            out += [(n * 1536, "bf16") for n in (4608, 1536, 6144, 6144, 6144)] + [(n, "f32") for n in (1536, 1536, 64, 64)]
        return out
    rng = random.Random(c["seed"])
    kinds = rng.choice([["f32"], ["bf16"], ["f16"], ["f32", "bf16"], ["f32", "f16", "bf16"]])
    most, out, total = _log(rng, 64, 8000000), [], 0
    for _ in range(_log(rng, 1, 600)):
        n = _log(rng, 1, most)
        total += n
        if total > 4e8:
            break
        out.append((n, rng.choice(kinds)))
    return out


def _clip_inputs(case, seed):
    c, d, s = case, _Draw(seed), _State()
    s.flat, s.parts = {}, []   # a buffer a type; (type, start, elements) of each tensor
    end = {}
    for n, t in _tensors(c):
        at = end.get(t, 0)
        s.parts.append((t, at, n))
        at += n
        end[t] = at if c["packed"] else -(-at // 64) * 64   # end to end, or each at an aligned address of its own
    for t in sorted(end):
        s.flat[t] = torch.zeros(end[t], device="cuda", dtype=TYPES[t])
    for t, at, n in s.parts:
        s.flat[t][at:at + n] = d.normal((n,), 0.01, 0.0, TYPES[t])
    return s


def _prepare_clip(case, seed):
    s = _clip_inputs(case, seed)
    s.closes = True
    s.out = {t: torch.zeros_like(f) for t, f in s.flat.items()}
    s.stat = torch.zeros(2, device="cuda", dtype=torch.float64)   # the norm, and the factor it was clipped by
    return s


def _run_clip(s):
    c = s.case
    if own:
        k = _binding()
        if s.plan is None:   # the program's list of gradients
            el = {t: f.element_size() for t, f in s.flat.items()}
            s.plan = k.Tensors(_ctx(), [(s.flat[t].data_ptr() + at * el[t], n, _code(t), s.out[t].data_ptr() + at * el[t], _code(t))
                                        for t, at, n in s.parts])
        s.plan.clip(c["count"], c["clip"], stat=_Ref(s.stat))
        return [s.out[t] for t in sorted(s.out)] + [s.stat]
    inv = 1.0 / c["count"]
    avg = [s.flat[t][at:at + n].float() * inv for t, at, n in s.parts]
    norm = torch.sqrt(torch.stack([a.double().square().sum() for a in avg]).sum())
    scale = torch.where((norm > c["clip"]) & (c["clip"] > 0), c["clip"] / (norm + 1e-6), torch.ones_like(norm)).float()
    for (t, at, n), a in zip(s.parts, avg):
        s.out[t][at:at + n] = (a * scale).to(TYPES[t])
    s.stat.copy_(torch.stack([norm, scale.double()]))
    return [s.out[t] for t in sorted(s.out)] + [s.stat]


def _exact_clip(case, seed):
    c, s = case, _clip_inputs(case, seed)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(f, dtype=torch.float64)) ** 2 for f in s.flat.values())) / c["count"]
    scale = c["clip"] / (norm + 1e-6) if 0 < c["clip"] < norm else 1.0
    return [s.flat[t].double() * (scale / c["count"]) for t in sorted(s.flat)] + \
           [torch.tensor([norm, scale], device="cuda", dtype=torch.float64)]


def _work_clip(c):
    n = {"f32": 0, "f16": 0, "bf16": 0}
    for k, t in _tensors(c):
        n[t] += k
    return {"bytes": 8.0 * n["f32"] + 4.0 * (n["f16"] + n["bf16"]), "flops": 4.0 * sum(n.values())}


# ------------------------------------------------------------------------------------------------
_KINDS = {"rope": (_prepare_rope, _run_rope, _exact_rope, _work_rope),
          "gate": (_prepare_gate, _run_gate, _exact_gate, _work_gate),
          "clip": (_prepare_clip, _run_clip, _exact_clip, _work_clip)}


def prepare(case, seed):
    s = _KINDS[case["kind"]][0](case, seed)
    s.case = case
    return s


def run(state):
    return _KINDS[state.case["kind"]][1](state)


def exact(case, seed):
    return _KINDS[case["kind"]][2](case, seed)


def work(case):
    return _KINDS[case["kind"]][3](case)
