"""The operators of the selective state-space layer, as timed and checked cases:
this framework's calls where `own` is true, their plain form in elementary torch
operations elsewhere.

A case is a dict of plain values whose "op" names the operator and whose "form"
says how it is called ("train": forward and the gradients of every input,
"prompt": forward alone with the state it leaves, "step": one token on a state):

  conv   y[t,c] = act(bias[c] + sum_k w[c,k] x[t-W+1+k, c]), the short causal
         convolution over [B,L,C] rows that are a slice of a wider projection
  scan   h[t] = exp(d[t] A) h[t-1] + d[t] x[t] (x) B[t],  y[t] = h[t] C[t] + D x[t]
         with d = softplus(dt + dt_bias) per head, x [B,L,H,P], B and C [B,L,G,N]
         shared by the H/G heads of a group, h [P,N] per head
  norm   LayerNorm over the last axis of x, or of x silu(gate)

"dtype" is the activations' type; parameters and states are fp32."""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PATHS = [_ROOT, os.path.join(_ROOT, "ttt-triton_amd")]

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # a layer's convolution in training at the benchmark's size: 12 heads of
        # 64 features and one group's B and C of 64
        dict(name="conv_train_b16_bf16", op="conv", form="train", B=16, L=2048, C=896, W=4, pad=780, act=True,
             state=False, dtype="bf16"),
        # a prompt of odd length and width in full precision, continued from an
        # earlier one
        dict(name="conv_prompt_b3_f32_odd", op="conv", form="prompt", B=3, L=1021, C=999, W=3, pad=0, act=True,
             state=True, dtype="f32"),
        # one token for each of 64 sequences
        dict(name="conv_step_b64_bf16", op="conv", form="step", B=64, L=1, C=896, W=4, pad=780, act=True, state=True,
             dtype="bf16"),
        # the scan in training at the benchmark's size (B 16, 2048 tokens, 12 heads of 64)
        dict(name="scan_train_b16_bf16", op="scan", form="train", B=16, L=2048, H=12, P=64, G=1, N=64, state=False,
             dtype="bf16"),
        # one long prompt: few chains, so the length has to be shared out
        dict(name="scan_prompt_b1_bf16_long", op="scan", form="prompt", B=1, L=16384, H=12, P=64, G=1, N=128,
             state=False, dtype="bf16"),
        # the small model's layer (4 heads of 32) in full precision
        dict(name="scan_train_b32_f32", op="scan", form="train", B=32, L=512, H=4, P=32, G=1, N=32, state=False,
             dtype="f32"),
        # odd sizes in fp16: every head its own B and C, a state carried in and out
        dict(name="scan_train_b3_f16_odd", op="scan", form="train", B=3, L=777, H=5, P=64, G=5, N=128, state=True,
             dtype="f16"),
        # one token for each of 64 sequences
        dict(name="scan_step_b64_bf16", op="scan", form="step", B=64, L=1, H=12, P=64, G=1, N=64, state=True,
             dtype="bf16"),
        # one token of one sequence: latency
        dict(name="scan_step_b1_bf16", op="scan", form="step", B=1, L=1, H=12, P=64, G=1, N=64, state=True,
             dtype="bf16"),
        # the layer's gated norm in training at the benchmark's size
        dict(name="norm_train_b16_bf16", op="norm", form="train", R=32768, D=768, gate=True, affine=True,
             dtype="bf16"),
        # a wide row of odd length in fp16, no gate
        dict(name="norm_train_wide_f16_odd", op="norm", form="train", R=4099, D=5001, gate=False, affine=True,
             dtype="f16"),
        # the rows of one token a sequence
        dict(name="norm_infer_b64_bf16", op="norm", form="prompt", R=64, D=768, gate=True, affine=True,
             dtype="bf16"),
    ]


def draw(rng):
    def span(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    dt = rng.choice(["bf16", "bf16", "f32", "f16"])
    op = rng.choice(["conv", "scan", "scan", "scan", "norm"])
    form = rng.choice(["train", "train", "prompt", "step"])
    if op == "norm":
        D = span(32, 8192)
        return dict(op=op, form="train" if rng.random() < 0.6 else "prompt", R=span(1, min(32768, 24000000 // D)),
                    D=D - D % 8 if rng.random() < 0.5 else D, gate=rng.random() < 0.5, affine=rng.random() < 0.8,
                    dtype=dt)
    if op == "conv":
        C = span(16, 2048)
        C = C - C % 8 if rng.random() < 0.6 else C
        B = span(1, 256 if form == "step" else 16)
        return dict(op=op, form=form, B=B, L=1 if form == "step" else span(1, max(1, min(8192, 24000000 // (B * C)))),
                    C=C, W=rng.choice([2, 3, 4, 4]), pad=rng.choice([0, 8, 780, 5]), act=rng.random() < 0.7,
                    state=form == "step" or rng.random() < 0.5, dtype=dt)
    G = rng.choice([1, 1, 2, 3, 4, 5])
    H, P, N = G * span(1, 12 // G), rng.choice([32, 64, 64]), rng.choice([16, 32, 64, 64, 128])
    B = span(1, 256 if form == "step" else 16)
    # no more than a quarter of the benchmark's tokens and heads: a wide state or fp32 costs that much more
    L = 1 if form == "step" else span(1, max(1, min(8192, 98000 // (B * H) * 64 // P)))
    return dict(op=op, form=form, B=B, L=L, H=H, P=P, G=G, N=N, state=form == "step" or rng.random() < 0.5, dtype=dt)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _Draw:
    """Seeded values, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 4093) + seed)

    def randn(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * std

    def rand(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")


def _inputs(c, seed):
    """{name: tensor}: activations as slices of the rows that a projection or the
    convolution leaves, parameters, states, and the gradients that reach the outputs."""
    r, dt = _Draw(seed), DT[c["dtype"]]
    train = c["form"] == "train"
    if c["op"] == "norm":
        R, D = c["R"], c["D"]
        v = dict(x=r.randn(R, D).to(dt))
        if c["gate"]:
            v["gate"] = r.randn(R, D + 24).to(dt)[:, :D]
        if c["affine"]:
            v.update(weight=1 + r.randn(D, std=0.1), bias=r.randn(D, std=0.1))
        if train:
            v["dy"] = r.randn(R, D).to(dt)
        return v
    B, L = c["B"], c["L"]
    if c["op"] == "conv":
        C, W = c["C"], c["W"]
        x = r.randn(B, L, C + c["pad"]).to(dt)[..., c["pad"]:]
        v = dict(x=x, weight=r.randn(C, W, std=W ** -0.5), bias=r.randn(C, std=0.1))
        if c["state"]:
            v["state"] = r.randn(B, W - 1, C).to(dt)
        if train:
            v["dy"] = r.randn(B, L, C).to(dt)
            v["dfinal"] = r.randn(B, W - 1, C).to(dt)
        return v
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    xbc = r.randn(B, L, H * P + 2 * G * N).to(dt)
    dt_log = math.log(1e-3) + r.rand(H) * math.log(100.0)  # steps of 0.001 to 0.1 where dt is 0
    v = dict(x=xbc[..., :H * P].unflatten(-1, (H, P)), dt=r.randn(B, L, H).to(dt), A=-(1 + 15 * r.rand(H)),
             Bm=xbc[..., H * P:H * P + G * N].unflatten(-1, (G, N)), Cm=xbc[..., H * P + G * N:].unflatten(-1, (G, N)),
             D=1 + r.randn(H, std=0.1), dt_bias=torch.log(torch.expm1(torch.exp(dt_log))))
    if c["state"]:
        v["state"] = r.randn(B, H, P, N, std=0.3)
    if train:
        v["dy"] = r.randn(B, L, H, P).to(dt)
        v["dfinal"] = r.randn(B, H, P, N, std=0.3)
    return v


_LEAVES = {"conv": ("x", "weight", "bias", "state"), "scan": ("x", "dt", "A", "Bm", "Cm", "D", "dt_bias", "state"),
           "norm": ("x", "gate", "weight", "bias")}


def prepare(c, seed):
    v = _inputs(c, seed)
    if c["form"] == "train":
        for k in _LEAVES[c["op"]]:
            if k in v:
                v[k] = v[k].detach().requires_grad_(True)
    elif c["op"] != "norm" and c["form"] == "step":
        for k in ("x", "dt", "Bm", "Cm"):
            if k in v:
                v[k] = v[k][:, 0]
    return {"c": c, "v": v}


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(x, weight, bias, state, act):
    """(y, the last W - 1 inputs), [B,L,C] and [B,W-1,C]."""
    W = weight.shape[1]
    if state is None:
        state = x.new_zeros(x.shape[0], W - 1, x.shape[2])
    seen = torch.cat([state, x], 1)
    y = (seen.float().unfold(1, W, 1) * weight).sum(-1) + bias
    return (_silu(y) if act else y).to(x.dtype), seen[:, -(W - 1):]


CHUNK = 64


def _plain_scan(x, dt, A, Bm, Cm, D, dt_bias, state):
    """(y [B,L,H,P], the last state): within chunks as one masked product, between
    them as one product over the chunks.  Sums of log-decays in 64 bits, since they
    are subtracted from each other."""
    B, L, H, P = x.shape
    G, N = Bm.shape[2:]
    nc = -(-L // CHUNK)
    pad = nc * CHUNK - L

    def chunks(t):  # [B,L,H,F] -> [B,H,nc,CHUNK,F], zeros behind the last token
        t = torch.cat([t, t.new_zeros(B, pad, *t.shape[2:])], 1)
        return t.reshape(B, nc, CHUNK, H, t.shape[3]).permute(0, 3, 1, 2, 4).contiguous()

    d = dt.float() + dt_bias
    d = torch.where(d > 20, d, torch.log1p(torch.exp(torch.clamp(d, max=20))))
    xs, d = chunks(x.float()), chunks(d[..., None])[..., 0]
    b, k = (chunks(t.float().repeat_interleave(H // G, 2)) for t in (Bm, Cm))
    la = torch.cumsum(d.double() * A.double()[:, None, None], -1)  # [B,H,nc,CHUNK]
    ones = torch.ones(CHUNK, CHUNK, device=x.device, dtype=torch.bool).tril()
    decay = torch.exp((la[..., :, None] - la[..., None, :]).masked_fill(~ones, -math.inf)).float()
    y = (torch.matmul(k, b.transpose(-1, -2).contiguous()) * decay * d[..., None, :]) @ xs
    w = torch.exp(la[..., -1:] - la).float() * d
    made = torch.matmul((xs * w[..., None]).transpose(-1, -2).contiguous(), b)  # [B,H,nc,P,N], what each chunk adds
    first = x.new_zeros(B, H, 1, P, N, dtype=torch.float32) if state is None else state[:, :, None]
    ends = torch.nn.functional.pad(torch.cumsum(la[..., -1], -1), (1, 0))  # [B,H,nc+1]
    ones = torch.ones(nc + 1, nc + 1, device=x.device, dtype=torch.bool).tril()
    carry = torch.exp((ends[..., :, None] - ends[..., None, :]).masked_fill(~ones, -math.inf)).float()
    h = torch.matmul(carry, torch.cat([first, made], 2).flatten(3)).unflatten(3, (P, N))  # entering each chunk
    y = y + torch.matmul(k, h[:, :, :-1].transpose(-1, -2).contiguous()) * torch.exp(la).float()[..., None]
    y = y + xs * D[:, None, None, None]
    return y.permute(0, 2, 3, 1, 4).reshape(B, nc * CHUNK, H, P)[:, :L].to(x.dtype), h[:, :, -1]


def _plain_scan_step(x, dt, A, Bm, Cm, state, D, dt_bias):
    H, G = x.shape[1], Bm.shape[1]
    d = dt.float() + dt_bias
    d = torch.where(d > 20, d, torch.log1p(torch.exp(torch.clamp(d, max=20))))
    b, k = (t.float().repeat_interleave(H // G, 1) for t in (Bm, Cm))
    h = state * torch.exp(d * A)[..., None, None] + (x.float() * d[..., None])[..., None] * b[:, :, None]
    state.copy_(h)
    return ((h * k[:, :, None]).sum(-1) + x.float() * D[:, None]).to(x.dtype)


def _plain_norm(x, weight, bias, gate):
    v = x.float()
    if gate is not None:
        v = v * _silu(gate.float())
    u = v - v.mean(-1, keepdim=True)
    y = u / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS)
    return (y if weight is None else y * weight + bias).to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _entry_points():
    sys.path[:0] = [p for p in _PATHS if p not in sys.path]
    from ttt_amd import norm, ssm
    return ssm, norm


def _forward(c, v):
    """The outputs of one forward pass, in a list."""
    op, form, state = c["op"], c["form"], v.get("state")
    if own:
        ssm, norm = _entry_points()
        if op == "norm":
            return [norm.layer_norm(v["x"], v.get("weight"), v.get("bias"), gate=v.get("gate"), eps=EPS)]
        if op == "conv":
            act = "silu" if c["act"] else None
            if form == "step":
                return [ssm.causal_conv_step(v["x"], state, v["weight"], v["bias"], activation=act), state]
            return list(ssm.causal_conv(v["x"], v["weight"], v["bias"], initial_state=state, activation=act,
                                        return_final_state=True))
        if form == "step":
            return [ssm.selective_scan_step(v["x"], v["dt"], v["A"], v["Bm"], v["Cm"], state, D=v["D"],
                                            dt_bias=v["dt_bias"]), state]
        return list(ssm.selective_scan(v["x"], v["dt"], v["A"], v["Bm"], v["Cm"], D=v["D"], dt_bias=v["dt_bias"],
                                       initial_state=state, return_final_state=True))
    if op == "norm":
        return [_plain_norm(v["x"], v.get("weight"), v.get("bias"), v.get("gate"))]
    if op == "conv":
        if form == "step":
            y, last = _plain_conv(v["x"][:, None], v["weight"], v["bias"], state, c["act"])
            state.copy_(last)
            return [y[:, 0], state]
        return list(_plain_conv(v["x"], v["weight"], v["bias"], state, c["act"]))
    if form == "step":
        return [_plain_scan_step(v["x"], v["dt"], v["A"], v["Bm"], v["Cm"], state, v["D"], v["dt_bias"]), state]
    return list(_plain_scan(v["x"], v["dt"], v["A"], v["Bm"], v["Cm"], v["D"], v["dt_bias"], state))


def run(s):
    c, v = s["c"], s["v"]
    if c["form"] != "train":
        with torch.no_grad():
            return _forward(c, v)
    out = _forward(c, v)
    leaves = [k for k in _LEAVES[c["op"]] if k in v]
    grads = torch.autograd.grad(out, [v[k] for k in leaves], [v[k] for k in ("dy", "dfinal") if k in v])
    return {"out": [t.detach() for t in out], **{"d" + k: g for k, g in zip(leaves, grads)}}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(c):
    sx, train = 4 if c["dtype"] == "f32" else 2, c["form"] == "train"
    if c["op"] == "norm":
        n = c["R"] * c["D"]
        acts = n * (2 + c["gate"]) + (n * (2 + c["gate"]) if train else 0)
        par = 8 * c["D"] * c["affine"]
        return {"bytes": acts * sx + par * (2 if train else 1),
                "flops": n * ((8 + 5 * c["gate"]) + (14 + 8 * c["gate"] if train else 0))}
    B, L = c["B"], c["L"]
    if c["op"] == "conv":
        n, W = B * L * c["C"], c["W"]
        st = B * (W - 1) * c["C"] * sx
        par = 4 * c["C"] * (W + 1)
        nbytes = 2 * n * sx + st * (1 + c["state"]) + par
        if train:  # the outputs' gradients in; those of the inputs, the weights and the state out
            nbytes = nbytes * 2
        return {"bytes": nbytes, "flops": n * (2 * W + 6) * (3 if train else 1)}
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    nbytes = B * L * (2 * H * P + H + 2 * G * N) * sx + 4 * B * H * P * N * (1 + c["state"]) + 12 * H
    # a token and head: decay, add to and read the state; in training the same of its adjoint, and
    # the products of both with the token's vectors
    return {"bytes": nbytes * (2 if train else 1), "flops": B * L * H * P * N * (5 if not train else 17)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_conv(c, v):
    x, w, b = v["x"], v["weight"], v["bias"]
    B, L, C = x.shape
    W = c["W"]
    s0 = v["state"] if c["state"] else x.new_zeros(B, W - 1, C)
    seen = torch.cat([s0, x], 1)
    z = b.expand(B, L, C).clone()
    for k in range(W):
        z += w[:, k] * seen[:, k:k + L]
    sg = 1 / (1 + torch.exp(-z))
    out = [z * sg if c["act"] else z, seen[:, L:]]
    if c["form"] != "train":
        return out
    dz = v["dy"] * (sg * (1 + z * (1 - sg)) if c["act"] else 1.0)
    dseen = torch.zeros_like(seen)
    dseen[:, L:] += v["dfinal"]
    dw = torch.empty_like(w)
    for k in range(W):
        dseen[:, k:k + L] += w[:, k] * dz
        dw[:, k] = (dz * seen[:, k:k + L]).sum((0, 1))
    g = {"out": out, "dx": dseen[:, W - 1:], "dweight": dw, "dbias": dz.sum((0, 1))}
    if c["state"]:
        g["dstate"] = dseen[:, :W - 1]
    return g


def _exact_scan(c, v):
    """Token by token; in training the states are kept and walked back over."""
    x, A, D = v["x"], v["A"], v["D"]
    B, L, H, P = x.shape
    rep = H // c["G"]
    raw = v["dt"] + v["dt_bias"]
    d = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    a = torch.exp(d * A)
    b, k = (v[n].repeat_interleave(rep, 2) for n in ("Bm", "Cm"))
    h = v["state"] if c["state"] else x.new_zeros(B, H, P, c["N"])
    train = c["form"] == "train"
    kept, y = [], torch.empty_like(x)
    for t in range(L):
        if train:
            kept.append(h)
        h = a[:, t, :, None, None] * h + (d[:, t, :, None] * x[:, t])[..., None] * b[:, t, :, None, :]
        y[:, t] = (h * k[:, t, :, None, :]).sum(-1)
    y += D[:, None] * x
    out = [y, h]
    if not train:
        return out
    dy, g = v["dy"], v["dfinal"].clone()
    dx, db, dk, dd, dA = torch.empty_like(x), torch.empty_like(b), torch.empty_like(k), torch.empty_like(d), 0
    for t in reversed(range(L)):
        last = h
        h = kept.pop()
        g = g + dy[:, t, :, :, None] * k[:, t, :, None, :]
        dk[:, t] = (dy[:, t, :, :, None] * last).sum(2)
        gb = (g * b[:, t, :, None, :]).sum(-1)
        da = (g * h).sum((-1, -2)) * a[:, t]
        dx[:, t] = d[:, t, :, None] * gb
        db[:, t] = (g * x[:, t, :, :, None]).sum(2) * d[:, t, :, None]
        dd[:, t] = (gb * x[:, t]).sum(-1) + da * A
        dA = dA + (da * d[:, t]).sum(0)
        g = g * a[:, t, :, None, None]
    draw_ = dd / (1 + torch.exp(-raw))
    r = {"out": out, "dx": dx + D[:, None] * dy, "ddt": draw_, "dA": dA,
         "dBm": db.unflatten(2, (c["G"], rep)).sum(3), "dCm": dk.unflatten(2, (c["G"], rep)).sum(3),
         "dD": (dy * x).sum((0, 1, 3)), "ddt_bias": draw_.sum((0, 1))}
    if c["state"]:
        r["dstate"] = g
    return r


def _exact_norm(c, v):
    x = v["x"]
    if c["gate"]:
        z = v["gate"]
        sg = 1 / (1 + torch.exp(-z))
        u = x * z * sg
    else:
        u = x
    mean = u.mean(-1, keepdim=True)
    rstd = ((u - mean).square().mean(-1, keepdim=True) + EPS) ** -0.5
    n = (u - mean) * rstd
    w, b = (v["weight"], v["bias"]) if c["affine"] else (1.0, 0.0)
    out = [n * w + b]
    if c["form"] != "train":
        return out
    dn = v["dy"] * w
    du = rstd * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
    r = {"out": out, "dx": du * z * sg if c["gate"] else du}
    if c["gate"]:
        r["dgate"] = du * x * sg * (1 + z * (1 - sg))
    if c["affine"]:
        r.update(dweight=(v["dy"] * n).sum(0), dbias=v["dy"].sum(0))
    return r


def exact(c, seed):
    if c["op"] == "scan" and c["L"] * c["B"] * c["H"] * c["P"] * c["N"] > 3e9:
        return None
    v = {k: t.double() for k, t in _inputs(c, seed).items()}
    r = {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[c["op"]](c, v)
    if c["form"] == "step":  # one token: the sequence axis goes
        r = [r[0][:, 0], r[1]]
    return r
