"""The operators of a layer on the gated delta rule, as measured workloads.

Short convolutions of queries, keys and values are what a layer on the gated delta rule begins
with.  Behind them it normalises the queries and keys, runs the rule (chunks of tokens for a
prompt or a training batch, one token at a time to answer), normalises each head's output under a
gate, and adds the projected result to the residual stream, whose norm the next block reads.
Each case below is one pass through one of these.

``run`` computes either the operators' plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, the package's own operators on the same inputs.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    bf, f32 = "bf16", "f32"
    return [
        # One sequence generating text: the rule's step in one layer.  Nothing but latency.
        dict(name="delta_step_one", op="delta_step", dtype=bf, B=1, H=16, dk=128, dv=128, slots=0),
        # A server's decode step: 128 sequences whose states lie in a pool.
        dict(name="delta_step_pool", op="delta_step", dtype=bf, B=128, H=32, dk=128, dv=128, slots=160),
        # A few odd prompts continued from a state, on views of one fused projection, keys and
        # values of different width.
        dict(name="delta_prompt_ragged", op="delta_prompt", dtype=bf, B=3, T=777, H=5, dk=64, dv=96),
        # One long prompt: few heads, and a chain of chunks that has to be walked.
        dict(name="delta_prompt_long", op="delta_prompt", dtype=bf, B=1, T=32768, H=16, dk=128, dv=128),
        # Training, forward and backward: the four sequences of 4096 tokens and 2048 channels that
        # the package's benchmark uses.
        dict(name="delta_train", op="delta_train", dtype=bf, B=4, T=4096, H=16, dk=128, dv=128),
        # The same in 32 bits at the sizes of the package's correctness sweep (256 channels).
        dict(name="delta_train_f32", op="delta_train", dtype=f32, B=2, T=512, H=4, dk=64, dv=64),
        # One token's heads normalised under their gates.
        dict(name="gated_norm_one", op="gated_norm", dtype=bf, N=1, H=16, d=128, train=False),
        # The same for the benchmark's batch, forward and backward.
        dict(name="gated_norm_train", op="gated_norm", dtype=bf, N=16384, H=16, d=128, train=True),
        # 32 bits, odd numbers of rows and an odd width.
        dict(name="gated_norm_f32", op="gated_norm", dtype=f32, N=2331, H=5, d=99, train=True),
        # One token's residual add and norm between two blocks.
        dict(name="residual_norm_one", op="residual_norm", dtype=bf, N=1, D=2048, train=False),
        # The same for the benchmark's batch, forward and backward, with a learned scale per channel.
        dict(name="residual_norm_train", op="residual_norm", dtype=bf, N=16384, D=2048, train=True),
        # Few wide rows in 32 bits: the sums over the rows are what there is to split.
        dict(name="residual_norm_f32", op="residual_norm", dtype=f32, N=509, D=8190, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["delta_step", "delta_prompt", "delta_train", "gated_norm", "residual_norm"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if op == "delta_step":
        B = _log_int(rng, 1, 256)
        return dict(op=op, dtype=dtype, B=B, H=_log_int(rng, 1, 32 if B <= 128 else 16), dk=rng.choice([32, 64, 80, 96, 128]),
                    dv=rng.choice([32, 64, 96, 128]), slots=0 if rng.random() < 0.5 else B + _log_int(rng, 1, 32))
    if op in ("delta_prompt", "delta_train"):
        top = 1 << (14 if dtype == "f32" else 18 if op == "delta_train" else 19)  # tokens x heads
        H = _log_int(rng, 1, 32)
        T = _log_int(rng, 1, min(16384 if op == "delta_train" else 32768, top // H))
        B = _log_int(rng, 1, max(1, min(16, top // (H * T))))
        dk = rng.choice([32, 64, 72, 96, 128, 128])
        return dict(op=op, dtype=dtype, B=B, T=T, H=H, dk=dk, dv=rng.choice([32, 64, 96, 128, dk]))
    top, train = 1 << 25, rng.random() < 0.7
    if op == "gated_norm":
        H, d = _log_int(rng, 1, 32), rng.choice([32, 64, 72, 96, 99, 128, 128, 256])
        return dict(op=op, dtype=dtype, N=_log_int(rng, 1, min(65536, top // (H * d))), H=H, d=d, train=train)
    D = _log_int(rng, 64, 8192)
    return dict(op=op, dtype=dtype, N=_log_int(rng, 1, min(32768, top // D)), D=D, train=train)


# ------------------------------------------------------------------------------- inputs


def _gates(shape, H, rnd):
    """Logarithms of the decays, -A_h softplus(..) with A from 1 to 16 over the heads and steps about
    0.01, and the rates beta in (0, 1)."""
    A = torch.linspace(1, 16, H, device="cuda") if H > 1 else torch.full((1,), 4.0, device="cuda")
    step = torch.nn.functional.softplus(rnd(*shape) - 4.6)
    return -A * step, torch.sigmoid(rnd(*shape))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def unit(*shape):  # normalised rows with a direction in common, as gated activations give them
        t = rnd(*shape) + 0.3
        return t * t.square().sum(-1, keepdim=True).rsqrt()

    s = dict(case=dict(case))
    op = case["op"]
    if op == "delta_step":
        B, H, dk, dv, n = case["B"], case["H"], case["dk"], case["dv"], case["slots"] or case["B"]
        s["slots"] = torch.randperm(n, device=dev, generator=g)[:B].to(torch.int32) if case["slots"] else None
        s["q"], s["k"], s["v"] = unit(B, H, dk).to(dt), unit(B, H, dk).to(dt), rnd(B, H, dv).to(dt)
        s["log_decay"], s["beta"] = (t.to(dt) for t in _gates((B, H), H, rnd))
        s["state"] = rnd(n, H, dk, dv)  # a state that has run for a while
    elif op in ("delta_prompt", "delta_train"):
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        qkv = torch.cat([unit(B, T, H, dk).view(B, T, H * dk), unit(B, T, H, dk).view(B, T, H * dk), rnd(B, T, H * dv)], -1).to(dt)
        q, k, v = (t.unflatten(-1, (H, -1)) for t in qkv.split([H * dk, H * dk, H * dv], -1))  # views of one buffer
        s["log_decay"], s["beta"] = (t.to(dt) for t in _gates((B, T, H), H, rnd))
        s["q"], s["k"], s["v"] = q, k, v
        if op == "delta_prompt":
            s["state"] = rnd(B, H, dk, dv)
        else:
            s["do"] = rnd(B, T, H, dv).to(dt)
            for name in ("q", "k", "v"):
                s[name] = s[name].contiguous()
            for name in ("q", "k", "v", "log_decay", "beta"):
                s[name].requires_grad_()
    else:
        shape = (case["N"], case["H"], case["d"]) if op == "gated_norm" else (case["N"], case["D"])
        s["x"] = rnd(*shape).to(dt)
        s["weight"] = (1 + 0.1 * rnd(shape[-1])).to(dt)
        if op == "gated_norm":
            s["gate"] = rnd(*shape).to(dt)
        else:
            s["residual"] = (2 * rnd(*shape)).to(dt)
            s["scale"] = (0.5 + 0.1 * rnd(shape[-1])).to(dt)
        if case["train"]:
            for t in list(s.values()):
                if isinstance(t, torch.Tensor):
                    t.requires_grad_()
            s["dy"] = rnd(*shape).to(dt)
            if op == "residual_norm":
                s["dh"] = rnd(*shape).to(dt)
    return s


# --------------------------------------------------------------------------- plain forms


def _delta_step_plain(s):
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "log_decay", "beta"))
    rows = slice(None) if s["slots"] is None else s["slots"].long()
    S = s["state"][rows] * torch.exp(g)[..., None, None]
    u = (v - (k[..., None, :] @ S).squeeze(-2)) * beta[..., None]
    S = S + k[..., :, None] * u[..., None, :]
    o = (q[..., None, :] @ S).squeeze(-2) * q.shape[-1] ** -0.5
    s["state"][rows] = S
    return o.to(s["q"].dtype), s["state"]


def _delta_plain(q, k, v, g, beta, S, C=64):
    """The rule in chunks of C tokens, 32-bit tensors [B, T, H, d] and gates [B, T, H].  Within a chunk the
    updates u solve a unit lower triangular system, whose inverse is a product of powers; what the chunks
    hand on is the state S [B, H, dk, dv].  Returns o and the state after the last token."""
    B, T, H, dk = q.shape
    n = -(-T // C)
    pad = n * C - T  # (tokens behind the end: no decay, no update)
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).view(B, n, C, H, -1).permute(0, 3, 1, 2, 4) for t in (q, k, v))
    g, beta = (torch.nn.functional.pad(t, (0, 0, 0, pad)).view(B, n, C, H).permute(0, 3, 1, 2) for t in (g, beta))
    b = g.cumsum(-1)
    i = torch.arange(C, device=q.device)
    decay = torch.exp(torch.where(i[:, None] >= i, b[..., :, None] - b[..., None, :], -torch.inf))  # [B, H, n, C, C]
    kt = k.transpose(-1, -2)
    X = torch.where(i[:, None] > i, -beta[..., None] * decay * (k @ kt), 0.0)
    inv = torch.eye(C, device=q.device) + X
    for _ in range(int(math.log2(C)) - 1):
        X = X @ X
        inv = inv + inv @ X
    e = torch.exp(b)[..., None]
    w, u0 = inv @ (k * e * beta[..., None]), inv @ (v * beta[..., None])
    attn = decay * (q @ kt)
    q_in, k_out, e_out = q * e, (k * torch.exp(b[..., -1:] - b)[..., None]).transpose(-1, -2), e[..., -1:, :]
    outs = []
    for c in range(n):
        u = u0[:, :, c] - w[:, :, c] @ S
        outs.append(q_in[:, :, c] @ S + attn[:, :, c] @ u)
        S = e_out[:, :, c] * S + k_out[:, :, c] @ u
    o = torch.stack(outs, 2) * dk**-0.5
    return o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, -1)[:, :T], S


def _delta_prompt_plain(s):
    o, S = _delta_plain(*(s[n].float() for n in ("q", "k", "v", "log_decay", "beta")), s["state"])
    return o.to(s["q"].dtype), S


def _delta_train_plain(s):
    c = s["case"]
    leaves = [s[n].detach().float().requires_grad_() for n in ("q", "k", "v", "log_decay", "beta")]
    S0 = torch.zeros(c["B"], c["H"], c["dk"], c["dv"], device="cuda")
    o, _ = _delta_plain(*leaves, S0)
    grads = torch.autograd.grad(o, leaves, s["do"].float())
    return [t.detach().to(s["q"].dtype) for t in (o, *grads)]


def _gated_norm_plain(s):
    x, w, z = s["x"].detach().float(), s["weight"].detach().float(), s["gate"].detach().float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n, sig = x * r, torch.sigmoid(z)
    dt = s["x"].dtype
    y = (n * w * z * sig).to(dt)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    dn = dy * w * z * sig
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    dw = (dy * n * z * sig).sum((0, 1))
    dz = dy * n * w * sig * (1 + z * (1 - sig))
    return y, dx.to(dt), dw.to(dt), dz.to(dt)


def _residual_norm_plain(s):
    x, res, w, sc = (s[n].detach().float() for n in ("x", "residual", "weight", "scale"))
    dt = s["x"].dtype
    h = res + sc * x
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    n = h * r
    y = n * w
    if not s["case"]["train"]:
        return y.to(dt), h.to(dt)
    dy = s["dy"].float()
    dn = dy * w
    dh = s["dh"].float() + r * (dn - n * (dn * n).mean(-1, keepdim=True))
    grads = (dh * sc, dh, (dy * n).sum(0), (dh * x).sum(0))
    return [t.to(dt) for t in (y, h, *grads)]


# ------------------------------------------------------------------------- own operators


def _run_own(s):
    import dynamic_conv1d_b200 as dc

    c = s["case"]
    op = c["op"]
    if op == "delta_step":
        o = dc.gated_delta_rule_step(s["q"], s["k"], s["v"], s["state"], s["log_decay"], s["beta"], slots=s["slots"])
        return o, s["state"]
    if op == "delta_prompt":
        return dc.gated_delta_rule(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], initial_state=s["state"], return_state=True)
    if op == "delta_train":
        leaves = [s[n] for n in ("q", "k", "v", "log_decay", "beta")]
        o = dc.gated_delta_rule(*leaves)
        return [o.detach(), *torch.autograd.grad(o, leaves, s["do"])]
    if op == "gated_norm":
        y = dc.gated_rms_norm(s["x"], s["weight"], s["gate"], eps=EPS)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["gate"]), s["dy"])) if c["train"] else y
    y, h = dc.residual_rms_norm(s["x"], s["residual"], s["weight"], s["scale"], eps=EPS)
    if not c["train"]:
        return y, h
    leaves = (s["x"], s["residual"], s["weight"], s["scale"])
    return [y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"]))]


_PLAIN = {"delta_step": _delta_step_plain, "delta_prompt": _delta_prompt_plain, "delta_train": _delta_train_plain,
          "gated_norm": _gated_norm_plain, "residual_norm": _residual_norm_plain}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# -------------------------------------------------------------------------- work, oracle


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "delta_step":
        B, H, dk, dv = (case[k] for k in ("B", "H", "dk", "dv"))
        return dict(bytes=B * H * (2 * 4 * dk * dv + e * (2 * dk + 2 * dv + 2)), flops=7 * B * H * dk * dv)
    if op == "delta_prompt":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        # three products of a token with the state: what it holds for the key, the update, the output
        return dict(bytes=B * H * (e * T * (2 * dk + 2 * dv + 2) + 2 * 4 * dk * dv), flops=6 * B * T * H * dk * dv)
    if op == "delta_train":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        # q, k, v, gates and the output's gradient read, the output and five gradients written
        return dict(bytes=B * T * H * e * (4 * dk + 4 * dv + 4), flops=18 * B * T * H * dk * dv)
    n = case["N"] * (case["H"] * case["d"] if op == "gated_norm" else case["D"])
    if op == "gated_norm":
        return dict(bytes=e * n * (6 if case["train"] else 3), flops=n * (25 if case["train"] else 8))
    return dict(bytes=e * n * (8 if case["train"] else 4), flops=n * (20 if case["train"] else 7))


def _exact_rule(q, k, v, g, beta, S, do=None):
    """The rule token by token in 64 bits.  With do, also the gradients, from the last token to the first;
    the states are kept at every 64th token and computed again between them."""
    scale, T = q.shape[-1] ** -0.5, q.shape[1]
    a = torch.exp(g)[..., None, None]

    def step(t, S):
        P = S * a[:, t]
        r = v[:, t] - (k[:, t, :, None, :] @ P).squeeze(-2)
        u = r * beta[:, t, :, None]
        return P, r, u, P + k[:, t, :, :, None] * u[..., None, :]

    o, kept = torch.empty_like(v), []
    for t in range(T):
        if do is not None and t % 64 == 0:
            kept.append(S)
        S = step(t, S)[3]
        o[:, t] = (q[:, t, :, None, :] @ S).squeeze(-2) * scale
    if do is None:
        return o, S
    dq, dk, dv, dg, db = (torch.empty_like(t) for t in (q, k, v, g, beta))
    dS = torch.zeros_like(S)
    for c in reversed(range(len(kept))):
        steps, S = [], kept[c]
        for t in range(64 * c, min(T, 64 * c + 64)):
            steps.append(step(t, S))
            S = steps[-1][3]
        for t in reversed(range(64 * c, min(T, 64 * c + 64))):
            P, r, u, S = steps.pop()
            dot = do[:, t, :, :, None] * scale
            dq[:, t] = (S @ dot).squeeze(-1)
            dS = dS + q[:, t, :, :, None] * dot.transpose(-1, -2)
            du = (k[:, t, :, None, :] @ dS).squeeze(-2)
            db[:, t] = (du * r).sum(-1)
            dr = du * beta[:, t, :, None]
            dv[:, t] = dr
            dk[:, t] = (dS @ u[..., None]).squeeze(-1) - (P @ dr[..., None]).squeeze(-1)
            dS = dS - k[:, t, :, :, None] * dr[..., None, :]
            dg[:, t] = (dS * P).sum((-1, -2))
            dS = dS * a[:, t]
    return o, dq, dk, dv, dg, db


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("delta"):
        args = [s[n].detach().double() for n in ("q", "k", "v", "log_decay", "beta")]
    if op == "delta_step":
        rows = torch.arange(case["B"], device="cuda") if s["slots"] is None else s["slots"].long()
        state = s["state"].double()
        o, S = _exact_rule(*(t[:, None] for t in args), state[rows])
        state[rows] = S
        return o[:, 0], state
    if op == "delta_prompt":
        return _exact_rule(*args, s["state"].double())
    if op == "delta_train":
        S0 = torch.zeros(case["B"], case["H"], case["dk"], case["dv"], device="cuda", dtype=torch.float64)
        return list(_exact_rule(*args, S0, s["do"].double()))
    # the norms: autograd through their definitions
    names = ("x", "weight", "gate") if op == "gated_norm" else ("x", "residual", "weight", "scale")
    leaves = [s[n].detach().double().requires_grad_() for n in names]
    if op == "gated_norm":
        x, w, z = leaves
        y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w * z / (1 + torch.exp(-z))
        outs, ups = [y], ["dy"]
    else:
        x, res, w, sc = leaves
        h = res + sc * x
        outs, ups = [h / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w, h], ["dy", "dh"]
    if not case["train"]:
        return outs[0].detach() if op == "gated_norm" else [t.detach() for t in outs]
    grads = torch.autograd.grad(outs, leaves, [s[n].double() for n in ups])
    return [*(t.detach() for t in outs), *grads]
