"""The operators of a block of the gated delta-rule layer, as timed and checked cases:
this framework's calls where `own` is true, their plain form in elementary torch
operations elsewhere.

A case is a dict of plain values whose "op" names the operator and whose "form"
says how it is called ("train": forward and the gradients of every input,
"prompt": forward alone, "step": one token on a state):

  delta  S_t = e^{g_t} S_{t-1} + u_t (x) k_t,  u_t = b_t (v_t - e^{g_t} S_{t-1} k_t),
         o_t = scale S_t q_t: a state S [P,N] per head, v [B,L,H,P], q and k
         [B,L,G,N] shared by the H/G heads of a group and, with "l2", taken at unit
         length; g <= 0 and b per token and head
  norm   r = residual + scale * silu(gate) * x / rms(x) * weight and r / rms(r) *
         next_weight, each part where the case has it: the norm after a block, its
         gate and residual scale, and the norm before the next block
  ffn    act(x Wg^T + bg) * (x Wu^T + bu)

"dtype" is the activations' type, of the feed-forward block the weights' too; the
norms' parameters and the states are fp32, the others' as the case says."""

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
        # a layer in training at the benchmark's size: 12 heads of 64, 2048 tokens
        dict(name="delta_train_b16_bf16", op="delta", form="train", B=16, L=2048, H=12, G=12, N=64, P=64, l2=True,
             state=False, dtype="bf16"),
        # the small model's heads of 32 in full precision, odd length, heads that share
        # keys, a state carried in and out
        dict(name="delta_train_b3_f32_odd", op="delta", form="train", B=3, L=777, H=4, G=2, N=32, P=32, l2=True,
             state=True, dtype="f32"),
        # wide heads in fp16, three to a key, keys of unit length already
        dict(name="delta_train_b2_f16_wide", op="delta", form="train", B=2, L=1021, H=6, G=2, N=128, P=128, l2=False,
             state=True, dtype="f16"),
        # one long prompt: few chains, so the length has to be shared out
        dict(name="delta_prompt_b1_bf16_long", op="delta", form="prompt", B=1, L=16384, H=12, G=12, N=64, P=64, l2=True,
             state=False, dtype="bf16"),
        # one token for each of 64 sequences
        dict(name="delta_step_b64_bf16", op="delta", form="step", B=64, L=1, H=12, G=12, N=64, P=64, l2=True, state=True,
             dtype="bf16"),
        # between two blocks in training: the block's output normed, scaled and added to
        # the fp32 residual, and normed for the next one
        dict(name="norm_train_b16_bf16", op="norm", form="train", R=32768, D=768, heads=1, after=True, gate=False,
             residual="f32", scale=True, next=True, dtype="bf16"),
        # the layer's own norm by heads with its gate
        dict(name="norm_heads_train_b16_bf16", op="norm", form="train", R=32768, D=64, heads=12, after=True, gate=True,
             residual=None, scale=False, next=False, dtype="bf16"),
        # between two blocks, one token for each of 64 sequences
        dict(name="norm_infer_b64_bf16", op="norm", form="prompt", R=64, D=768, heads=1, after=True, gate=False,
             residual="f32", scale=True, next=True, dtype="bf16"),
        # the feed-forward block in training at the benchmark's size
        dict(name="ffn_train_b16_bf16", op="ffn", form="train", R=32768, D=768, F=2048, act="silu", bias=False,
             dtype="bf16"),
        # odd sizes in full precision, with biases
        dict(name="ffn_train_f32_odd", op="ffn", form="train", R=2043, D=501, F=1333, act="silu", bias=True, dtype="f32"),
        # a prompt's rows in fp16 with the other activation
        dict(name="ffn_prompt_f16_odd", op="ffn", form="prompt", R=4099, D=1024, F=2731, act="gelu", bias=True,
             dtype="f16"),
        # one token for each of 64 sequences
        dict(name="ffn_infer_b64_bf16", op="ffn", form="prompt", R=64, D=768, F=2048, act="silu", bias=False,
             dtype="bf16"),
    ]


def draw(rng):
    def span(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    dt = rng.choice(["bf16", "bf16", "f32", "f16"])
    op = rng.choice(["delta", "delta", "norm", "ffn"])
    if op == "delta":
        form = rng.choice(["train", "train", "prompt", "step"])
        G = rng.choice([1, 2, 3, 4, 5])
        H, N, P = G * rng.choice([1, 1, 2]), rng.choice([16, 32, 64, 64, 80, 128]), rng.choice([32, 64, 64, 96, 128])
        B = span(1, 256 if form == "step" else 16)
        # no more than an eighth of the benchmark's tokens and heads: wide states or fp32 cost more
        L = 1 if form == "step" else span(1, max(1, min(4096, 49000 * 64 * 64 // (B * H * max(P, 32) * max(N, 32)))))
        return dict(op=op, form=form, B=B, L=L, H=H, G=G, N=N, P=P, l2=rng.random() < 0.6,
                    state=form == "step" or rng.random() < 0.5, dtype=dt)
    if op == "norm":
        heads = rng.choice([1, 1, 1, 4, 12])
        D = span(16, 128) if heads > 1 else span(32, 8192)
        D = D - D % 8 if rng.random() < 0.5 else D
        residual = rng.choice([None, "f32", dt]) if heads == 1 else None
        after = residual is None or rng.random() < 0.8
        return dict(op=op, form="train" if rng.random() < 0.6 else "prompt",
                    R=span(1, min(32768, 20000000 // (D * heads))), D=D, heads=heads, after=after,
                    gate=rng.random() < 0.5, residual=residual, scale=rng.random() < 0.5,
                    next=residual is not None and rng.random() < 0.7, dtype=dt)
    D, F = span(16, 1024), span(16, 2800)
    D = D - D % 8 if rng.random() < 0.5 else D
    F = F - F % 8 if rng.random() < 0.5 else F
    return dict(op=op, form="train" if rng.random() < 0.6 else "prompt", R=span(1, min(32768, 12000000000 // (D * F))),
                D=D, F=F, act=rng.choice(["silu", "gelu"]), bias=rng.random() < 0.5, dtype=dt)


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
        R, D, n = c["R"], c["D"], c["heads"]
        shape = (R, n, D) if n > 1 else (R, D)
        v = dict(x=r.randn(*shape).to(dt))
        if c["gate"]:  # columns of the projection
            z = r.randn(R, n * D + 24).to(dt)[:, :n * D]
            v["gate"] = z.unflatten(1, (n, D)) if n > 1 else z
        if c["residual"]:
            v["residual"] = r.randn(*shape).to(DT[c["residual"]])
        if c["after"]:
            v["weight"] = 1 + r.randn(D, std=0.1)
        if c["scale"]:
            v["scale"] = 0.5 + r.randn(D, std=0.1)
        if c["next"]:
            v["next_weight"] = 1 + r.randn(D, std=0.1)
        if train:
            v["dout"] = r.randn(*shape).to(v["residual"].dtype if c["residual"] else dt)
            if c["next"]:
                v["dnormed"] = r.randn(*shape).to(dt)
        return v
    if c["op"] == "ffn":
        R, D, F = c["R"], c["D"], c["F"]
        v = dict(x=r.randn(R, D).to(dt), w_gate=r.randn(F, D, std=D ** -0.5).to(dt),
                 w_up=r.randn(F, D, std=D ** -0.5).to(dt))
        if c["bias"]:
            v.update(b_gate=r.randn(F, std=0.1).to(dt), b_up=r.randn(F, std=0.1).to(dt))
        if train:
            v["dy"] = r.randn(R, F).to(dt)
        return v
    B, L, H, G, N, P = (c[k] for k in "BLHGNP")
    z = r.randn(B, L, 2 * G * N + H * P)
    z = z / (1 + torch.exp(-z))  # behind the convolution's SiLU
    if not c["l2"]:  # of unit length already
        qk = z[..., :2 * G * N].unflatten(-1, (2 * G, N))
        z[..., :2 * G * N] = (qk / torch.sqrt((qk * qk).sum(-1, keepdim=True) + EPS)).flatten(-2)
    z = z.to(dt)
    rate = 1 + 15 * r.rand(H)  # steps of 0.001 to 0.1 where the projection gives 0
    step = torch.exp(math.log(1e-3) + r.rand(H) * math.log(100.0))
    a = r.randn(B, L, H) + torch.log(torch.expm1(step))
    v = dict(q=z[..., :G * N].unflatten(-1, (G, N)), k=z[..., G * N:2 * G * N].unflatten(-1, (G, N)),
             v=z[..., 2 * G * N:].unflatten(-1, (H, P)), g=-rate * torch.log1p(torch.exp(a)),
             beta=1 / (1 + torch.exp(-r.randn(B, L, H))))
    if c["state"]:
        v["state"] = r.randn(B, H, P, N, std=0.3)
    if train:
        v["do"] = r.randn(B, L, H, P).to(dt)
        v["dfinal"] = r.randn(B, H, P, N, std=0.3)
    return v


_LEAVES = {"delta": ("q", "k", "v", "g", "beta", "state"),
           "norm": ("x", "weight", "residual", "gate", "scale", "next_weight"),
           "ffn": ("x", "w_gate", "w_up", "b_gate", "b_up")}


def prepare(c, seed):
    v = _inputs(c, seed)
    if c["form"] == "train":
        for k in _LEAVES[c["op"]]:
            if k in v:
                v[k] = v[k].detach().requires_grad_(True)
    elif c["form"] == "step":
        for k in ("q", "k", "v", "g", "beta"):
            v[k] = v[k][:, 0]
    return {"c": c, "v": v}


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits
# ---------------------------------------------------------------------------

CHUNK = 64


def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)


def _inverse(A):
    """(1 + A)^-1 of strictly lower triangles [.., n, n], n a power of two: of the
    blocks on the diagonal, twice as large each time."""
    n = A.shape[-1]
    lead = A.shape[:-2]
    X = torch.ones(*lead, n, 1, 1, device=A.device)  # the inverses of the diagonal's blocks
    m = 1
    while m < n:
        cut = A.reshape(*lead, n // (2 * m), 2 * m, n // (2 * m), 2 * m).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        X = X.reshape(*lead, n // (2 * m), 2, m, m)
        a, b = X[..., 0, :, :], X[..., 1, :, :]
        low = -torch.matmul(torch.matmul(b, cut[..., m:, :m].contiguous()), a.contiguous())
        X = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([low, b], -1)], -2)
        m *= 2
    return X[..., 0, :, :]


def _plain_delta(q, k, v, g, beta, state, l2):
    """(o [B,L,H,P], the last state [B,H,P,N]): everything within the chunks of all
    sequences at once, and from chunk to chunk the state alone.  Sums of log-decays in
    64 bits, since they are subtracted from each other."""
    B, L, H, P = v.shape
    G, N = k.shape[2:]
    nc = -(-L // CHUNK)
    pad = nc * CHUNK - L

    def chunks(t):  # [B,L,H,F] -> [B,H,nc,CHUNK,F], zeros behind the last token
        t = torch.cat([t, t.new_zeros(B, pad, *t.shape[2:])], 1)
        return t.reshape(B, nc, CHUNK, H, t.shape[3]).permute(0, 3, 1, 2, 4).contiguous()

    qf, kf = q.float(), k.float()
    if l2:
        qf, kf = _unit(qf), _unit(kf)
    qc, kc = (chunks(t.repeat_interleave(H // G, 2)) for t in (qf * N ** -0.5, kf))
    vc, b = chunks(v.float()), chunks(beta.float()[..., None])
    la = torch.cumsum(chunks(g[..., None])[..., 0].double(), -1)
    ones = torch.ones(CHUNK, CHUNK, device=v.device, dtype=torch.bool).tril()
    decay = torch.exp((la[..., :, None] - la[..., None, :]).masked_fill(~ones, -math.inf)).float()
    kt = kc.transpose(-1, -2).contiguous()
    A = torch.matmul(kc, kt) * decay * b * ones.tril(-1)
    M = torch.matmul(qc, kt) * decay
    head = torch.exp(la).float()[..., None]
    tail = torch.exp(la[..., -1:] - la).float()[..., None]
    end = torch.exp(la[..., -1]).float()[..., None, None]
    T = _inverse(A)
    w, u0 = torch.matmul(T, kc * b * head), torch.matmul(T, vc * b)
    kw, qw = (kc * tail).transpose(-1, -2).contiguous(), qc * head
    s = v.new_zeros(B, H, N, P, dtype=torch.float32) if state is None else state.transpose(-1, -2).contiguous()
    u, enter = [], []
    for i in range(nc):
        enter.append(s)
        u.append(u0[:, :, i] - torch.matmul(w[:, :, i], s))
        s = s * end[:, :, i] + torch.matmul(kw[:, :, i], u[-1])
    o = torch.matmul(qw, torch.stack(enter, 2)) + torch.matmul(M, torch.stack(u, 2))
    return o.permute(0, 2, 3, 1, 4).reshape(B, nc * CHUNK, H, P)[:, :L].to(v.dtype), s.transpose(-1, -2)


def _plain_delta_step(q, k, v, g, beta, state, l2):
    H, G, N = v.shape[1], k.shape[1], k.shape[2]
    qf, kf = q.float(), k.float()
    if l2:
        qf, kf = _unit(qf), _unit(kf)
    qf, kf = (t.repeat_interleave(H // G, 1)[:, :, None] for t in (qf * N ** -0.5, kf))
    s = state * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v.float() - (s * kf).sum(-1))
    s = s + u[..., None] * kf
    state.copy_(s)
    return (s * qf).sum(-1).to(v.dtype)


def _plain_norm(x, weight, residual, gate, scale, next_weight):
    n = x.float()
    if weight is not None:
        n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS) * weight
    if gate is not None:
        z = gate.float()
        n = n * (z / (1 + torch.exp(-z)))
    if scale is not None:
        n = n * scale
    if residual is None:
        return [n.to(x.dtype)]
    n = residual.float() + n
    if next_weight is None:
        return [n.to(residual.dtype)]
    y = n / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS) * next_weight
    return [n.to(residual.dtype), y.to(x.dtype)]


def _plain_ffn(x, w_gate, w_up, b_gate, b_up, act):
    xf = x.float()
    a, b = torch.matmul(xf, w_gate.float().t()), torch.matmul(xf, w_up.float().t())
    if b_gate is not None:
        a, b = a + b_gate.float(), b + b_up.float()
    a = a / (1 + torch.exp(-a)) if act == "silu" else 0.5 * a * (1 + torch.erf(a * 0.5 ** 0.5))
    return (a * b).to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _entry_points():
    sys.path[:0] = [p for p in _PATHS if p not in sys.path]
    from ttt_amd import delta, ffn, norm
    return delta, norm, ffn


def _forward(c, v):
    """The outputs of one forward pass, in a list."""
    op, form = c["op"], c["form"]
    if own:
        delta, norm, ffn = _entry_points()
        if op == "norm":
            r = norm.block_norm(v["x"], v.get("weight"), v.get("residual"), v.get("gate"), v.get("scale"),
                                v.get("next_weight"), eps=EPS)
            return list(r) if isinstance(r, tuple) else [r]
        if op == "ffn":
            return [ffn.gated_linear(v["x"], v["w_gate"], v["w_up"], v.get("b_gate"), v.get("b_up"),
                                     activation=c["act"])]
        if form == "step":
            return [delta.gated_delta_step(v["q"], v["k"], v["v"], v["g"], v["beta"], v["state"], l2_norm=c["l2"]),
                    v["state"]]
        return list(delta.gated_delta(v["q"], v["k"], v["v"], v["g"], v["beta"], initial_state=v.get("state"),
                                      l2_norm=c["l2"], return_final_state=True))
    if op == "norm":
        return _plain_norm(v["x"], v.get("weight"), v.get("residual"), v.get("gate"), v.get("scale"),
                           v.get("next_weight"))
    if op == "ffn":
        return [_plain_ffn(v["x"], v["w_gate"], v["w_up"], v.get("b_gate"), v.get("b_up"), c["act"])]
    if form == "step":
        return [_plain_delta_step(v["q"], v["k"], v["v"], v["g"], v["beta"], v["state"], c["l2"]), v["state"]]
    return list(_plain_delta(v["q"], v["k"], v["v"], v["g"], v["beta"], v.get("state"), c["l2"]))


def run(s):
    c, v = s["c"], s["v"]
    if c["form"] != "train":
        with torch.no_grad():
            return _forward(c, v)
    out = _forward(c, v)
    leaves = [k for k in _LEAVES[c["op"]] if k in v]
    grads = torch.autograd.grad(out, [v[k] for k in leaves],
                                [v[k] for k in ("do", "dfinal", "dout", "dnormed", "dy") if k in v])
    return {"out": [t.detach() for t in out], **{"d" + k: g for k, g in zip(leaves, grads)}}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _size(dt):
    return 4 if dt == "f32" else 2


def work(c):
    sx, train = _size(c["dtype"]), c["form"] == "train"
    if c["op"] == "norm":
        n = c["R"] * c["heads"] * c["D"]
        sr = _size(c["residual"]) if c["residual"] else 0
        out = n * (sr or sx) + n * sx * c["next"]
        ins = n * sx * (1 + c["gate"]) + n * sr
        par = 4 * c["D"] * (c["after"] + c["scale"] + c["next"])
        return {"bytes": ins + out + par + (ins + out + par if train else 0),
                "flops": n * (4 * c["after"] + 4 * c["next"] + 6 * c["gate"] + 2 * c["scale"]) * (3 if train else 1)}
    if c["op"] == "ffn":
        R, D, F = c["R"], c["D"], c["F"]
        one = (R * D + 2 * F * D + 2 * F * c["bias"]) * sx
        # in training the products of x once, and of the gradients with the weights and with x
        return {"bytes": one + R * F * sx + (one + R * F * sx if train else 0),
                "flops": 4 * R * D * F * (3 if train else 1)}
    B, L, H, G, N, P = (c[k] for k in "BLHGNP")
    nbytes = B * L * (2 * H * P + 2 * G * N) * sx + 8 * B * L * H + 4 * B * H * P * N * (1 + c["state"])
    # a token and head: decay the state, read it twice and add to it; in training the same of its
    # adjoint and the products of both with the token's vectors
    return {"bytes": nbytes * (2 if train else 1), "flops": B * L * H * P * N * (7 if not train else 25)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_delta(c, v):
    """Token by token; in training the states are kept and walked back over."""
    B, L, H, P = v["v"].shape
    N, rep, train = c["N"], H // c["G"], c["form"] == "train"
    x, beta, a, scale = v["v"], v["beta"], torch.exp(v["g"]), N ** -0.5
    nq, nk = (((v[n] ** 2).sum(-1, keepdim=True) + EPS) ** -0.5 if c["l2"] else 1.0 for n in ("q", "k"))
    uq, uk = v["q"] * nq, v["k"] * nk
    q, k = (t.repeat_interleave(rep, 2) for t in (uq, uk))
    s = v["state"] if c["state"] else x.new_zeros(B, H, P, N)
    o, kept = torch.empty_like(x), []
    for t in range(L):
        if train:
            kept.append(s)
        s = s * a[:, t, :, None, None]
        u = beta[:, t, :, None] * (x[:, t] - (s * k[:, t, :, None]).sum(-1))
        s = s + u[..., None] * k[:, t, :, None]
        o[:, t] = (s * q[:, t, :, None]).sum(-1) * scale
    if not train:
        return [o, s]
    last, do, ds = s, v["do"] * scale, v["dfinal"].clone()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(x)
    dg, db = torch.empty_like(a), torch.empty_like(beta)
    for t in reversed(range(L)):
        dq[:, t] = (do[:, t, ..., None] * s).sum(2)
        ds = ds + do[:, t, ..., None] * q[:, t, :, None]
        s = kept.pop()
        old, kt, bt = s * a[:, t, :, None, None], k[:, t, :, None], beta[:, t, :, None]
        miss = x[:, t] - (old * kt).sum(-1)
        du = (ds * kt).sum(-1)
        dv[:, t] = bt * du
        db[:, t] = (du * miss).sum(-1)
        dk[:, t] = (ds * (bt * miss)[..., None]).sum(2) - (dv[:, t, ..., None] * old).sum(2)
        dold = ds - dv[:, t, ..., None] * kt
        dg[:, t] = (dold * old).sum((-1, -2))
        ds = dold * a[:, t, :, None, None]
    dq, dk = (t.unflatten(2, (c["G"], rep)).sum(3) for t in (dq, dk))
    if c["l2"]:
        dq, dk = (n * (d - y * (d * y).sum(-1, keepdim=True)) for n, d, y in ((nq, dq, uq), (nk, dk, uk)))
    r = {"out": [o, last], "dq": dq, "dk": dk, "dv": dv, "dg": dg, "dbeta": db}
    if c["state"]:
        r["dstate"] = ds
    return r


def _rms_grad(dy, x, inv):
    """The gradient through x * inv, inv = (mean x^2 + eps)^-1/2."""
    return inv * dy - x * (inv ** 3 * (dy * x).mean(-1, keepdim=True))


def _exact_norm(c, v):
    x = v["x"]
    inv = ((x * x).mean(-1, keepdim=True) + EPS) ** -0.5 if c["after"] else 1.0
    w = v["weight"] if c["after"] else 1.0
    z = v["gate"] if c["gate"] else None
    sg = 1 / (1 + torch.exp(-z)) if c["gate"] else 1.0
    gate = z * sg if c["gate"] else 1.0
    sc = v["scale"] if c["scale"] else 1.0
    xn = x * inv
    r = xn * w * gate * sc + (v["residual"] if c["residual"] else 0.0)
    out = [r]
    if c["next"]:
        ri = ((r * r).mean(-1, keepdim=True) + EPS) ** -0.5
        out.append(r * ri * v["next_weight"])
    if c["form"] != "train":
        return out
    lead = tuple(range(x.dim() - 1))
    dr, res = v["dout"], {"out": out}
    if c["next"]:
        dr = dr + _rms_grad(v["dnormed"] * v["next_weight"], r, ri)
        res["dnext_weight"] = (v["dnormed"] * r * ri).sum(lead)
    if c["residual"]:
        res["dresidual"] = dr
    if c["scale"]:
        res["dscale"] = (dr * xn * w * gate).sum(lead)
    dn = dr * sc
    if c["gate"]:
        res["dgate"] = dn * xn * w * (sg * (1 + z * (1 - sg)))
    dn = dn * gate
    if c["after"]:
        res["dweight"] = (dn * xn).sum(lead)
        res["dx"] = _rms_grad(dn * w, x, inv)
    else:
        res["dx"] = dn
    return res


def _exact_ffn(c, v):
    x, wg, wu = v["x"], v["w_gate"], v["w_up"]
    a, b = x @ wg.T, x @ wu.T
    if c["bias"]:
        a, b = a + v["b_gate"], b + v["b_up"]
    if c["act"] == "silu":
        sg = 1 / (1 + torch.exp(-a))
        f, df = a * sg, sg * (1 + a * (1 - sg))
    else:
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        f, df = a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if c["form"] != "train":
        return [f * b]
    da, db = v["dy"] * b * df, v["dy"] * f
    r = {"out": [f * b], "dx": da @ wg + db @ wu, "dw_gate": da.T @ x, "dw_up": db.T @ x}
    if c["bias"]:
        r.update(db_gate=da.sum(0), db_up=db.sum(0))
    return r


def exact(c, seed):
    if c["op"] == "delta" and c["L"] * c["B"] * c["H"] * c["P"] * c["N"] > 3e9:
        return None
    v = {k: t.double() for k, t in _inputs(c, seed).items()}
    r = {"delta": _exact_delta, "norm": _exact_norm, "ffn": _exact_ffn}[c["op"]](c, v)
    if c["form"] == "step":  # one token: the sequence axis goes
        r = [r[0][:, 0], r[1]]
    return r
