"""The layer operators of sa3k as cases that can be prepared, run, priced and checked.

Three kinds of call, each in both directions, through the Python binding of the C ABI:

  norm   layer norm (with the residual sum in front of it), forward; backward with the gradients of
         gain and offset
  attn   attention with a sliding window and first tokens that stay visible, forward, over a long cache
         with one or a few queries ("step"), and backward
  prod   matrix product with bias, activation and residual in its epilogue, forward; backward with the
         gradients of input, weight and bias

`run` computes them with elementary torch operations, or, where `own` is set, with the framework's kernels.
Sizes: the model of the benchmark (heads of 64 x 24, width 1536, FFN 6144, 64 memory + 1024 latent tokens)
and the ranges around them.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False
LOG2E = 1.4426950408889634
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through the model's norm: a step of generation, latency only
        dict(name="norm_fwd_f16_1x1536", kind="norm", dir="fwd", type="f16", rows=1, cols=1536, res=True),
        # the residual stream of the benchmark's micro-batch, four of them at once
        dict(name="norm_fwd_bf16_8704x1536", kind="norm", dir="fwd", type="bf16", rows=8704, cols=1536, res=True),
        # the same stream's backward, at an odd length and width, in f32 as a trainer keeps its stream
        dict(name="norm_bwd_f32_4099x1025", kind="norm", dir="bwd", type="f32", rows=4099, cols=1025, res=True),
        # the benchmark model's self-attention with its 64 memory tokens visible to every latent
        dict(name="attn_fwd_bf16_b2_h24_s1088_w128_64", kind="attn", dir="fwd", type="bf16", batch=2, heads=24, kv=24,
             dim=64, sq=1088, sk=1088, left=128, right=128, sinks=64, causal=False, ragged=False),
        # a long causal sequence with grouped heads: prefill
        dict(name="attn_fwd_bf16_b1_h32_8_s8192_w1023_4", kind="attn", dir="fwd", type="bf16", batch=1, heads=32, kv=8,
             dim=128, sq=8192, sk=8192, left=1023, right=0, sinks=4, causal=True, ragged=False),
        # one new token a sequence over long caches that are filled to different lengths
        dict(name="attn_step_bf16_b8_h32_8_c16384", kind="attn", dir="step", type="bf16", batch=8, heads=32, kv=8,
             dim=128, sq=1, sk=16384, left=4095, right=0, sinks=4, causal=True, ragged=True),
        # training of the benchmark model's self-attention
        dict(name="attn_bwd_bf16_b2_h24_s1088_w128_64", kind="attn", dir="bwd", type="bf16", batch=2, heads=24, kv=24,
             dim=64, sq=1088, sk=1088, left=128, right=128, sinks=64, causal=False, ragged=False),
        # training on a padded batch of causal sequences with grouped heads
        dict(name="attn_bwd_f16_b3_h16_2_s2049_w511_4", kind="attn", dir="bwd", type="f16", batch=3, heads=16, kv=2,
             dim=128, sq=2049, sk=2049, left=511, right=0, sinks=4, causal=True, ragged=True),
        # one token through the FFN up-projection
        dict(name="prod_fwd_bf16_1x1536x6144_silu", kind="prod", dir="fwd", type="bf16", m=1, k=1536, n=6144, act="silu",
             res=False, keep=False),
        # the FFN down-projection of the micro-batch onto the residual stream
        dict(name="prod_fwd_bf16_2176x6144x1536_res", kind="prod", dir="fwd", type="bf16", m=2176, k=6144, n=1536,
             act="none", res=True, keep=False),
        # training of the FFN up-projection
        dict(name="prod_bwd_bf16_2176x1536x6144_gelu", kind="prod", dir="bwd", type="bf16", m=2176, k=1536, n=6144,
             act="gelu", res=False, keep=True),
        # a large layer's up-projection that keeps what its backward needs
        dict(name="prod_fwd_f16_8191x4096x8192_gelu_tanh", kind="prod", dir="fwd", type="f16", m=8191, k=4096, n=8192,
             act="gelu_tanh", res=False, keep=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["norm", "attn", "prod"], [3, 5, 4])[0]
    if kind == "norm":
        return dict(kind=kind, dir=rng.choice(["fwd", "bwd"]), type=rng.choice(["f32", "bf16", "f16"]),
                    rows=_log(rng, 1, 16384), cols=_log(rng, 16, 8192), res=rng.random() < 0.5)
    if kind == "attn":
        dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        sinks = rng.choice([0, 1, 4, 64])
        c = dict(kind=kind, dir=rng.choice(["fwd", "step", "bwd"]), type=rng.choice(["bf16", "f16"]),
                 batch=rng.randint(1, 4), heads=heads, kv=kv, dim=dim)
        if c["dir"] == "step":
            return dict(c, sq=rng.choice([1, 1, 1, 2, 5]), sk=_log(rng, 16, 32768), left=rng.choice([-1, 255, 4095]),
                        right=0, sinks=sinks, causal=True, ragged=rng.random() < 0.7)
        s = _log(rng, 1, 4096)
        s = min(s, int(math.sqrt((6e8 if c["dir"] == "bwd" else 1.5e9) / (c["batch"] * heads))))
        causal = rng.random() < 0.5
        left = rng.choice([-1, 16, 128, 1000])
        return dict(c, sq=s, sk=s, left=left, right=0 if causal else left, sinks=sinks, causal=causal,
                    ragged=rng.random() < 0.5)
    m, k, n = _log(rng, 1, 3500), _log(rng, 16, 6144), _log(rng, 16, 6144)
    if rng.random() < 0.75:
        k, n = -(-k // 8) * 8, -(-n // 8) * 8
    d = rng.choice(["fwd", "bwd"])
    return dict(kind=kind, dir=d, type=rng.choice(["bf16", "f16"]), m=m, k=k, n=n,
                act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), res=d == "fwd" and rng.random() < 0.5,
                keep=d == "bwd" or rng.random() < 0.5)


# ---------------------------------------------------------------------------------------- binding
def _binding():
    if "sa3k" not in sys.modules:
        spec = importlib.util.spec_from_file_location("sa3k", os.path.join(ROOT, "sa3.cpp_amd", "sa3k.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["sa3k"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["sa3k"]


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


class _Draw:
    """seeded tensors on the GPU, in the order they are asked for"""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, shape, sd=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, sd, generator=self.g).to(dtype)


# ------------------------------------------------------------------------------------------- norm
EPS = 1e-5


def _norm_inputs(case, seed):
    d, t = _Draw(seed), TYPES[case["type"]]
    shape = (case["rows"], case["cols"])
    s = _State()
    s.x = d.normal(shape, 1.5, 0.2, t)
    s.r = d.normal(shape, 0.5, 0.0, t) if case["res"] else None   # forward: the residual; backward: the sum's gradient
    s.gamma, s.beta = d.normal(shape[1:], 0.1, 1.0), d.normal(shape[1:], 0.1)
    s.dy = d.normal(shape, 1.0, 0.0, t)
    return s


def _prepare_norm(case, seed):
    s = _norm_inputs(case, seed)
    s.y, s.sum = torch.empty_like(s.x), torch.empty_like(s.x)
    if case["dir"] == "fwd":
        s.mean, s.rstd = torch.empty(case["rows"], device="cuda"), torch.empty(case["rows"], device="cuda")
    else:
        x = s.x.double()
        s.mean = x.mean(1).float()
        s.rstd = (1 / torch.sqrt(x.var(1, unbiased=False) + EPS)).float()
        s.dgamma, s.dbeta = torch.empty_like(s.gamma), torch.empty_like(s.beta)
    return s


def _run_norm(s):
    c = s.case
    if own:
        k = _binding()
        t = {"f32": k.TYPE_F32, "f16": k.TYPE_F16, "bf16": k.TYPE_BF16}[c["type"]]
        if c["dir"] == "fwd":
            k.layer_norm_fwd(_ctx(), t, _Ref(s.x), c["rows"], c["cols"], _Ref(s.gamma), _Ref(s.beta), EPS, _Ref(s.y),
                             mean=_Ref(s.mean), rstd=_Ref(s.rstd), residual=_ref(s.r), sum=_Ref(s.sum) if c["res"] else None)
            return [s.y, s.mean, s.rstd] + ([s.sum] if c["res"] else [])
        k.layer_norm_bwd(_ctx(), t, _Ref(s.dy), _Ref(s.x), c["rows"], c["cols"], _Ref(s.gamma), _Ref(s.mean), _Ref(s.rstd),
                         _Ref(s.y), dsum=_ref(s.r), dgamma=_Ref(s.dgamma), dbeta=_Ref(s.dbeta))
        return [s.y, s.dgamma, s.dbeta]
    if c["dir"] == "fwd":
        t = (s.x.float() + s.r.float()).to(s.x.dtype) if c["res"] else s.x   # the norm is of the sum as it is stored
        x = t.float()
        mean = x.mean(1)
        d = x - mean[:, None]
        rstd = 1 / torch.sqrt(d.square().mean(1) + EPS)
        y = (d * rstd[:, None] * s.gamma + s.beta).to(s.x.dtype)
        return [y, mean, rstd] + ([t] if c["res"] else [])
    dy = s.dy.float()
    xh = (s.x.float() - s.mean[:, None]) * s.rstd[:, None]
    h = dy * s.gamma
    dx = s.rstd[:, None] * (h - h.mean(1)[:, None] - xh * (h * xh).mean(1)[:, None])
    if c["res"]:
        dx = dx + s.r.float()
    return [dx.to(s.x.dtype), (dy * xh).sum(0), dy.sum(0)]


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    x = s.x.double()
    if case["dir"] == "fwd":
        if case["res"]:
            x = (s.x.double() + s.r.double()).to(s.x.dtype).double()
        var, mean = torch.var_mean(x, 1, unbiased=False)
        y = torch.nn.functional.layer_norm(x, x.shape[1:], s.gamma.double(), s.beta.double(), EPS)
        return [y, mean, torch.rsqrt(var + EPS)] + ([x] if case["res"] else [])
    x, g, b = x.requires_grad_(), s.gamma.double().requires_grad_(), s.beta.double().requires_grad_()
    torch.nn.functional.layer_norm(x, x.shape[1:], g, b, EPS).backward(s.dy.double())
    return [x.grad + s.r.double() if case["res"] else x.grad, g.grad, b.grad]


def _work_norm(c):
    el = 4.0 if c["type"] == "f32" else 2.0
    n = c["rows"] * c["cols"]
    if c["dir"] == "fwd":
        return {"bytes": n * el * (4 if c["res"] else 2) + 8.0 * c["rows"] + 8.0 * c["cols"], "flops": 8.0 * n}
    return {"bytes": n * el * (4 if c["res"] else 3) + 8.0 * c["rows"] + 12.0 * c["cols"], "flops": 14.0 * n}


# -------------------------------------------------------------------------------------- attention
def _lens(c):
    """keys of each sample: the whole length, or from the whole down to half of it"""
    return [c["sk"] - (b * c["sk"]) // (2 * c["batch"]) if c["ragged"] else c["sk"] for b in range(c["batch"])]


def _attn_inputs(case, seed):
    c, d, t, s = case, _Draw(seed), TYPES[case["type"]], _State()
    B, H, K, D = c["batch"], c["heads"], c["kv"], c["dim"]
    if c["dir"] == "step":   # a cache a head, and the new tokens' queries
        s.q = d.normal((B, c["sq"], H, D), 1.0, 0.0, t)
        s.k, s.v = d.normal((B, K, c["sk"], D), 1.0, 0.0, t).transpose(1, 2), d.normal((B, K, c["sk"], D), 1.0, 0.0, t).transpose(1, 2)
    else:                    # the projection's output, the heads of q, k and v beside each other
        s.qkv = d.normal((B, c["sq"], H + 2 * K, D), 1.0, 0.0, t)
        s.q, s.k, s.v = s.qkv[:, :, :H], s.qkv[:, :, H:H + K], s.qkv[:, :, H + K:]
    s.kv_len = torch.tensor(_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    s.q_len = s.kv_len if c["dir"] != "step" else None
    s.do = d.normal((B, c["sq"], H, D), 1.0, 0.0, t)
    return s


def _rows(c, dev):
    """queries [1][Sq], and of each sample: its queries, its keys, and whether a row is in its sequence"""
    kl = torch.tensor(_lens(c), device=dev)[:, None]
    ql = kl if c["dir"] != "step" else torch.full_like(kl, c["sq"])
    i = torch.arange(c["sq"], device=dev)[None, :]
    return i, ql, kl, i < ql


def _visible(c, dev):
    """[B][Sq][Sk]: whether a query sees a key; and [B][Sq]: whether the query's row is in its sequence"""
    i, ql, kl, row = _rows(c, dev)
    j = torch.arange(c["sk"], device=dev)
    p = (i + kl - ql)[:, :, None]
    ok = (j < kl)[:, None, :] & row[:, :, None]
    if c["causal"]:
        ok = ok & (j <= p)
    near = torch.ones_like(ok)
    if c["left"] >= 0:
        near = near & (j >= p - c["left"])
    if c["right"] >= 0 and not c["causal"]:
        near = near & (j <= p + c["right"])
    return ok & (near | (j < c["sinks"])), row


def _attn_weights(c, s):
    """softmax weights [B][H][Sq][Sk] and the row's base-2 log-sum, from the inputs in 32 bits"""
    ok, _ = _visible(c, s.q.device)
    g = c["heads"] // c["kv"]
    q = s.q.float().transpose(1, 2)
    k = s.k.float().transpose(1, 2).repeat_interleave(g, 1)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous())
    sc.mul_(c["dim"] ** -0.5 * LOG2E)
    sc.masked_fill_(~ok[:, None], -math.inf)
    m = sc.amax(3, keepdim=True)
    sc.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp2_()
    l = sc.sum(3, keepdim=True)
    sc.div_(torch.where(l == 0, torch.ones_like(l), l))
    return sc, (m + torch.log2(l))[..., 0]


def _attn_fwd(c, s):
    p, lse = _attn_weights(c, s)
    v = s.v.float().transpose(1, 2).repeat_interleave(c["heads"] // c["kv"], 1)
    o = torch.matmul(p, v.contiguous()).transpose(1, 2).to(s.q.dtype).contiguous()
    row = _rows(c, s.q.device)[3]
    lse = torch.where(row[:, None, :], lse, torch.zeros_like(lse))   # rows behind a sequence are left as they were
    return o, lse


def _prepare_attn(case, seed):
    c, s = case, _attn_inputs(case, seed)
    B, H, D = c["batch"], c["heads"], c["dim"]
    s.o = torch.zeros((B, c["sq"], H, D), device="cuda", dtype=s.q.dtype)
    s.lse = torch.zeros((B, H, c["sq"]), device="cuda")
    if c["dir"] == "bwd":
        s.o, s.lse = _attn_fwd(c, s)
        s.dqkv = torch.zeros_like(s.qkv)
        K = c["kv"]
        s.dq, s.dk, s.dv = s.dqkv[:, :, :H], s.dqkv[:, :, H:H + K], s.dqkv[:, :, H + K:]
    s.plan = None
    return s


def _strides(t):
    """(sample, token, head) strides of [B][S][H][D]"""
    return t.stride(0), t.stride(1), t.stride(2)


def _run_attn(s):
    c = s.case
    if own:
        k = _binding()
        if s.plan is None:   # the shape is set up once
            s.plan = k.WindowAttn(_ctx(), k.TYPE_BF16 if c["type"] == "bf16" else k.TYPE_F16, c["batch"], c["heads"],
                                  c["kv"], c["sq"], c["sk"], c["dim"], left=c["left"], right=c["right"],
                                  sinks=c["sinks"], causal=c["causal"], q_strides=_strides(s.q),
                                  k_strides=_strides(s.k), v_strides=_strides(s.v))
        ql, kl = _ref(s.q_len), _ref(s.kv_len)
        if c["dir"] != "bwd":
            s.plan.forward(_Ref(s.q), _Ref(s.k), _Ref(s.v), _Ref(s.o), _Ref(s.lse), ql, kl)
            return [s.o, s.lse]
        s.plan.backward(_Ref(s.q), _Ref(s.k), _Ref(s.v), _Ref(s.o), _Ref(s.lse), _Ref(s.do), _Ref(s.dq), _Ref(s.dk),
                        _Ref(s.dv), ql, kl)
        return [s.dqkv]
    if c["dir"] != "bwd":
        return list(_attn_fwd(c, s))
    p, _ = _attn_weights(c, s)
    B, H, K, D, g = c["batch"], c["heads"], c["kv"], c["dim"], c["heads"] // c["kv"]
    row = _rows(c, s.q.device)[3]
    q, do = s.q.float().transpose(1, 2).contiguous(), (s.do.float() * row[:, :, None, None]).transpose(1, 2).contiguous()
    k, v = (t.float().transpose(1, 2).repeat_interleave(g, 1) for t in (s.k, s.v))
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds.sub_((do * s.o.float().transpose(1, 2)).sum(3, keepdim=True)).mul_(p).mul_(D ** -0.5)
    dq = torch.matmul(ds, k.contiguous())
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dk, dv = (t.view(B, K, g, c["sk"], D).sum(2) for t in (dk, dv))
    return [torch.cat([dq, dk, dv], 1).transpose(1, 2).to(s.q.dtype).contiguous()]


def _exact_attn(case, seed):
    c, s = case, _attn_inputs(case, seed)
    if c["batch"] * c["heads"] * c["sq"] * c["sk"] > 2.5e9:
        return None
    g = c["heads"] // c["kv"]
    ok, row = _visible(c, s.q.device)
    q, k, v = (t.double().permute(0, 2, 1, 3).contiguous().requires_grad_(c["dir"] == "bwd") for t in (s.q, s.k, s.v))
    kk, vv = (t[:, :, None].expand(-1, -1, g, -1, -1).reshape(t.shape[0], -1, t.shape[2], t.shape[3]) for t in (k, v))
    sc = (q @ kk.mT.contiguous()) / math.sqrt(c["dim"])
    sc = sc.masked_fill(~ok[:, None], -math.inf)
    none = ~ok.any(2)[:, None, :, None]
    lse = torch.logsumexp(sc.detach(), 3) * LOG2E
    o = torch.softmax(sc.masked_fill(none, 0.0), 3).masked_fill(none, 0.0) @ vv
    if c["dir"] != "bwd":
        return [o.transpose(1, 2).contiguous(), lse.masked_fill(~row[:, None, :], 0.0)]
    (o * (s.do.double() * row[:, :, None, None]).transpose(1, 2)).sum().backward()
    return [torch.cat([q.grad, k.grad, v.grad], 1).transpose(1, 2).contiguous()]


def _work_attn(c):
    n = np.array(_lens(c), dtype=np.int64)[:, None]
    nq = np.full_like(n, c["sq"]) if c["dir"] == "step" else n
    i = np.arange(c["sq"], dtype=np.int64)[None, :]
    p, row = i + n - nq, i < nq
    lo = np.maximum(p - c["left"], 0) if c["left"] >= 0 else np.zeros_like(p)
    last = np.minimum(p, n - 1) if c["causal"] else np.broadcast_to(n - 1, p.shape)
    top = last if c["causal"] or c["right"] < 0 else np.minimum(p + c["right"], last)
    first = np.minimum(c["sinks"], last + 1)   # first tokens that the row may see
    seen = (top - lo + 1) + np.minimum(first, lo) + np.maximum(0, first - (top + 1))
    pairs = int((seen * row).sum())
    low = np.where(row, lo, n).min(1)
    read = int((np.where(row, np.maximum(top, first - 1), 0).max(1) - low + 1 + np.minimum(c["sinks"], low)).sum())
    D, H, K, rows = c["dim"], c["heads"], c["kv"], int(row.sum())
    if c["dir"] == "bwd":   # q, o, do, dq; k, v, dk, dv
        return {"bytes": 2.0 * D * (4 * H * rows + 4 * K * read) + 4.0 * H * rows, "flops": 10.0 * D * H * pairs}
    return {"bytes": 2.0 * D * (2 * H * rows + 2 * K * read) + 4.0 * H * rows, "flops": 4.0 * D * H * pairs}


# ---------------------------------------------------------------------------------------- product
def _prod_inputs(case, seed):
    c, d, t, s = case, _Draw(seed), TYPES[case["type"]], _State()
    s.x = d.normal((c["m"], c["k"]), 1.0, 0.0, t)
    s.w = d.normal((c["n"], c["k"]), c["k"] ** -0.5, 0.0, t)
    s.b = d.normal((c["n"],), 0.1)
    s.r = d.normal((c["m"], c["n"]), 1.0, 0.0, t) if c["res"] else None
    s.dy = d.normal((c["m"], c["n"]), 1.0, 0.0, t) if c["dir"] == "bwd" else None
    s.z = (torch.matmul(s.x.float(), s.w.float().t()) + s.b).to(t) if c["dir"] == "bwd" else None
    return s


def _prepare_prod(case, seed):
    s = _prod_inputs(case, seed)
    if case["dir"] == "fwd":
        s.y = torch.empty((case["m"], case["n"]), device="cuda", dtype=s.x.dtype)
        s.z = torch.empty_like(s.y) if case["keep"] else None
    else:
        s.dx, s.dw, s.db = torch.empty_like(s.x), torch.empty_like(s.w), torch.empty_like(s.b)
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


def _run_prod(s):
    c = s.case
    if own:
        k = _binding()
        t = k.TYPE_BF16 if c["type"] == "bf16" else k.TYPE_F16
        act = {"none": k.ACT_NONE, "relu": k.ACT_RELU, "silu": k.ACT_SILU, "gelu": k.ACT_GELU,
               "gelu_tanh": k.ACT_GELU_TANH}[c["act"]]
        if c["dir"] == "fwd":
            k.linear_act_fwd(_ctx(), t, act, _Ref(s.x), _Ref(s.w), c["m"], c["n"], c["k"], _Ref(s.y), bias=_Ref(s.b),
                             residual=_ref(s.r), z=_ref(s.z))
            return [s.y] + ([s.z] if c["keep"] else [])
        k.linear_act_bwd(_ctx(), t, act, _Ref(s.dy), _Ref(s.x), _Ref(s.w), c["m"], c["n"], c["k"], z=_Ref(s.z),
                         dx=_Ref(s.dx), dw=_Ref(s.dw), db=_Ref(s.db))
        return [s.dx, s.dw, s.db]
    x, w = s.x.float(), s.w.float()
    if c["dir"] == "fwd":
        z = torch.matmul(x, w.t()) + s.b
        y = _act(z, c["act"])
        if c["res"]:
            y = y + s.r.float()
        return [y.to(s.x.dtype)] + ([z.to(s.x.dtype)] if c["keep"] else [])
    dz = s.dy.float() * _act_slope(s.z.float(), c["act"])
    return [torch.matmul(dz, w).to(s.x.dtype), torch.matmul(dz.t(), x).to(s.x.dtype), dz.sum(0)]


def _exact_prod(case, seed):
    c, s = case, _prod_inputs(case, seed)
    f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[c["act"]]
    if c["dir"] == "fwd":
        z = torch.addmm(s.b.double(), s.x.double(), s.w.double().t())
        y = f(z)
        return [y + s.r.double() if c["res"] else y] + ([z] if c["keep"] else [])
    z = s.z.double().requires_grad_()
    f(z).backward(s.dy.double())
    return [z.grad @ s.w.double(), z.grad.t() @ s.x.double(), z.grad.sum(0)]


def _work_prod(c):
    m, n, k = float(c["m"]), float(c["n"]), float(c["k"])
    if c["dir"] == "fwd":
        return {"bytes": 2 * (m * k + n * k + m * n * (1 + bool(c["res"]) + bool(c["keep"]))) + 4 * n, "flops": 2 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n) + 4 * n, "flops": 4 * m * n * k}


# ------------------------------------------------------------------------------------------------
_KINDS = {"norm": (_prepare_norm, _run_norm, _exact_norm, _work_norm),
          "attn": (_prepare_attn, _run_attn, _exact_attn, _work_attn),
          "prod": (_prepare_prod, _run_prod, _exact_prod, _work_prod)}


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
