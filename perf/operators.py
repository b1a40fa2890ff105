"""The operators that surround a dynamic short convolution in a language model, as measured workloads.

A model built on the convolutions of this package projects its activations to queries, keys and
values, convolves them (``forward_fused``), mixes tokens with linear attention whose state decays
by a factor of its own in each head, and is trained on the cross entropy of the next token.  To
answer, it runs one token at a time: one convolution step on a cache of the last W-1 inputs and
one step of the attention's recurrent state.  Each case below is one pass through one of these.

``run`` computes either the operators' plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, the package's own operators on the same inputs.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100


def listed():
    bf, f32 = "bf16", "f32"
    return [
        # One sequence generating text: the query, key and value convolutions of one layer for one
        # token.  Nothing but latency.
        dict(name="conv_step_one", op="conv_step", form="lowrank", dtype=bf, B=1, G=3, D=2048, R=15, W=4, slots=0),
        # A server's decode step on a wide layer, with the rows' caches in a pool of slots.
        dict(name="conv_step_pool", op="conv_step", form="lowrank", dtype=bf, B=256, G=3, D=4096, R=31, W=4, slots=320),
        # The headwise form for a batch of sequences: 64 heads of 32 channels.
        dict(name="conv_step_headwise", op="conv_step", form="headwise", dtype=bf, B=64, G=1, D=2048, R=64, W=4, slots=0),
        # One sequence generating text: the attention's step.
        dict(name="attn_step_one", op="attn_step", dtype=bf, B=1, H=16, dk=128, dv=128, slots=0),
        # A server's decode step: 128 sequences whose states lie in a pool.
        dict(name="attn_step_pool", op="attn_step", dtype=bf, B=128, H=32, dk=128, dv=128, slots=160),
        # A few odd prompts continued from a state, keys and values of different width.
        dict(name="attn_prompt_ragged", op="attn_prompt", dtype=bf, B=3, T=777, H=5, dk=64, dv=96),
        # One very long prompt: few heads, so the time axis is what there is to split.
        dict(name="attn_prompt_long", op="attn_prompt", dtype=bf, B=1, T=65536, H=16, dk=128, dv=128),
        # Training: the four sequences of 4096 tokens and 2048 channels that the package's benchmark
        # uses, forward and backward, on the fused output of the query/key/value convolution.
        dict(name="attn_train", op="attn_train", dtype=bf, B=4, T=4096, H=16, dk=128, dv=128),
        # The same in 32 bits at the sizes of the package's correctness sweep (256 channels).
        dict(name="attn_train_f32", op="attn_train", dtype=f32, B=2, T=512, H=4, dk=64, dv=64),
        # The loss of a small model in 32 bits, odd numbers of tokens and words.
        dict(name="loss_f32", op="loss", dtype=f32, N=1021, D=256, V=4999),
        # The loss of the benchmark's batch (4 x 4096 tokens, 2048 channels) over 50001 words.
        dict(name="loss_train", op="loss", dtype=bf, N=16384, D=2048, V=50001),
        # A short batch of a wide model over a large vocabulary: the weight's gradient dominates.
        dict(name="loss_wide", op="loss", dtype=bf, N=3001, D=4096, V=131072),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv_step", "attn_step", "attn_prompt", "attn_train", "loss"])
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    if op == "conv_step":
        B, W = _log_int(rng, 1, 512), rng.choice([2, 3, 4, 4, 4, 6, 8])
        slots = 0 if rng.random() < 0.5 else B + _log_int(rng, 1, 64)
        if rng.random() < 0.5:
            D = 8 * _log_int(rng, 8, 512)
            return dict(op=op, form="lowrank", dtype=dtype, B=B, G=rng.choice([1, 3]), D=D, R=rng.choice([7, 15, 31]), W=W, slots=slots)
        hs, H = rng.choice([1, 2, 8, 16, 32, 64, 128]), _log_int(rng, 4, 64)
        return dict(op=op, form="headwise", dtype=dtype, B=B, G=1, D=hs * H, R=H, W=W, slots=slots)
    if op == "attn_step":
        B = _log_int(rng, 1, 256)
        return dict(op=op, dtype=dtype, B=B, H=_log_int(rng, 1, 32), dk=rng.choice([32, 64, 96, 128]),
                    dv=rng.choice([32, 64, 128]), slots=0 if rng.random() < 0.5 else B + _log_int(rng, 1, 32))
    if op in ("attn_prompt", "attn_train"):
        top = 1 << 14 if dtype == "f32" else 1 << 20  # tokens x heads
        H = _log_int(rng, 1, 32)
        T = _log_int(rng, 1, min(65536, top // H))
        B = _log_int(rng, 1, max(1, min(16, top // (H * T))))
        dk = rng.choice([32, 64, 80, 128, 128])
        dv = dk if op == "attn_train" else rng.choice([32, 64, 96, 128])
        return dict(op=op, dtype=dtype, B=B, T=T, H=H, dk=dk, dv=dv)
    D, V = 8 * _log_int(rng, 8, 512), _log_int(rng, 500, 20000 if dtype == "f32" else 131072)
    top = 2e10 if dtype == "f32" else 1.6e12  # N * D * V
    return dict(op=op, dtype=dtype, N=_log_int(rng, 1, max(1, min(16384, int(top / (D * V))))), D=D, V=V)


# ------------------------------------------------------------------------------- inputs


def _decays(H, device):
    """Log of the heads' decay factors: 1 - 2^-5 in the first head, 1 - 2^-12 in the last."""
    e = torch.linspace(5, 12, H, device=device, dtype=torch.float64) if H > 1 else torch.full((1,), 7.0, device=device, dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dt)

    s = dict(case=dict(case))
    op = case["op"]
    if op in ("conv_step", "attn_step"):
        B, n = case["B"], case["slots"] or case["B"]
        s["slots"] = torch.randperm(n, device=dev, generator=g)[:B].to(torch.int32) if case["slots"] else None
    if op == "conv_step":
        G, D, W = case["G"], case["D"], case["W"]
        s["x"] = rnd(B, G * D)
        s["cache"] = rnd(n, W - 1, G * D)
        if case["form"] == "lowrank":
            R = case["R"]
            s["z"] = rnd(B, G * R, scale=R**-0.5)
            s["U"] = rnd(G, R, W * D, scale=0.5)
            s["static_w"] = rnd(G, W, D, scale=W**-0.5)
        else:
            s["weight"] = rnd(B, case["R"], W, scale=0.5)
            s["static_w"] = rnd(W, D, scale=W**-0.5)
    elif op == "attn_step":
        H, dk, dv = case["H"], case["dk"], case["dv"]
        s["q"], s["k"], s["v"] = rnd(B, H, dk), rnd(B, H, dk), rnd(B, H, dv)
        s["log_decay"] = _decays(H, dev)
        # a state that has run for a while: about 32 tokens' worth of products
        s["state"] = torch.randn(n, H, dk, dv, device=dev, generator=g) * 32**0.5
    elif op == "attn_prompt":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        s["q"], s["k"], s["v"] = rnd(B, T, H, dk), rnd(B, T, H, dk), rnd(B, T, H, dv)
        s["log_decay"] = _decays(H, dev)
        s["state"] = torch.randn(B, H, dk, dv, device=dev, generator=g) * 32**0.5
    elif op == "attn_train":
        B, T, H, d = (case[k] for k in ("B", "T", "H", "dk"))
        s["qkv"] = rnd(B, T, 3 * H * d).requires_grad_()
        s["do"] = rnd(B, T, H * d)
        s["log_decay"] = _decays(H, dev)
    else:
        N, D, V = case["N"], case["D"], case["V"]
        s["hidden"] = rnd(N, D).requires_grad_()
        s["weight"] = rnd(V, D, scale=2.0 * D**-0.5).requires_grad_()
        t = torch.randint(0, V, (N,), device=dev, generator=g)
        # one token in twenty is padding; the first never is, so that there is something to learn
        pad = torch.rand(N, device=dev, generator=g) < 0.05
        pad[0] = False
        s["target"] = torch.where(pad, torch.full_like(t, IGNORE), t)
    return s


# --------------------------------------------------------------------------- plain forms


def _conv_step_plain(s):
    c = s["case"]
    B, G, D, W = (c[k] for k in ("B", "G", "D", "W"))
    rows = slice(None) if s["slots"] is None else s["slots"].long()
    window = torch.cat([s["cache"][rows], s["x"][:, None]], dim=1)  # oldest input first
    if c["form"] == "lowrank":
        z = s["z"].float().view(B, G, -1).transpose(0, 1)
        w = (z @ s["U"].float()).view(G, B, W, D) + s["static_w"].float()[:, None]
        w = w.permute(1, 2, 0, 3).reshape(B, W, G * D)
    else:
        hs = D // c["R"]
        w = s["weight"].float().transpose(1, 2)[..., None].expand(B, W, c["R"], hs).reshape(B, W, D) + s["static_w"].float()
    y = (w * window.float().flip(1)).sum(1) + s["x"].float()
    s["cache"][rows] = window[:, 1:]
    return y.to(s["x"].dtype), s["cache"]


def _attn_step_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    rows = slice(None) if s["slots"] is None else s["slots"].long()
    S = s["state"][rows] * torch.exp(s["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
    o = (q[..., None, :] @ S).squeeze(-2) * q.shape[-1] ** -0.5
    s["state"][rows] = S
    return o.to(s["q"].dtype), s["state"]


def _attn_plain(q, k, v, log_decay, S0, C):
    """Linear attention with decay in chunks of C tokens, 32-bit tensors [B, T, H, d]: the products
    within each chunk under a mask of decays, and a state handed from chunk to chunk by one product
    with the chunks' own matrix of decays.  Returns o and the state after the last token."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    n = -(-T // C)
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, 0, 0, n * C - T)).view(B, n, C, H, -1).permute(0, 3, 1, 2, 4) for t in (q, k, v))
    i = torch.arange(C, device=q.device, dtype=torch.float32)
    lam = log_decay[:, None, None]
    mask = torch.where(i[:, None] >= i, torch.exp(lam * (i[:, None] - i).clamp(min=0)), 0.0)  # [H, C, C]
    intra = ((q @ k.transpose(-1, -2)) * mask[None, :, None]) @ v
    # tokens of the last chunk that are there
    last = T - (n - 1) * C
    local = (k * torch.exp(lam * (C - 1 - i[:, None]))[None, :, None]).transpose(-1, -2) @ v  # [B, H, n, dk, dv]
    j = torch.arange(n + 1, device=q.device, dtype=torch.float32)
    carry = torch.where(j[:, None] > j[:-1], torch.exp(lam * C * (j[:, None] - 1 - j[:-1]).clamp(min=0)), 0.0)  # [H, n+1, n]
    states = (carry @ local.reshape(B, H, n, dk * dv)).view(B, H, n + 1, dk, dv)
    states = states + torch.exp(log_decay[:, None] * C * j)[None, :, :, None, None] * S0[:, :, None]
    inter = (q @ states[:, :, :-1]) * torch.exp(lam * (i[:, None] + 1))[None, :, None]
    # the state at the last token itself: from the start of its chunk
    k_last = k[:, :, -1, :last] * torch.exp(lam * (last - 1 - i[:last, None]))
    final = states[:, :, -2] * torch.exp(lam * last) + k_last.transpose(-1, -2) @ v[:, :, -1, :last]
    o = (intra + inter) * dk**-0.5
    return o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, dv)[:, :T], final


def _attn_prompt_plain(s):
    c = s["case"]
    C = 64 if c["T"] <= 4096 else 256
    o, S = _attn_plain(s["q"].float(), s["k"].float(), s["v"].float(), s["log_decay"], s["state"], C)
    return o.to(s["q"].dtype), S


def _attn_train_plain(s):
    c = s["case"]
    B, T, H, d = (c[k] for k in ("B", "T", "H", "dk"))
    x = s["qkv"].detach().float().requires_grad_()
    q, k, v = x.view(B, T, 3, H, d).unbind(2)
    S0 = torch.zeros(B, H, d, d, device=x.device)
    o, _ = _attn_plain(q, k, v, s["log_decay"], S0, 64 if T <= 4096 else 256)
    o = o.reshape(B, T, H * d)
    (dx,) = torch.autograd.grad(o, x, s["do"].float())
    return o.detach().to(s["qkv"].dtype), dx.to(s["qkv"].dtype)


def _loss_plain(s):
    h, w, t = s["hidden"].detach().float(), s["weight"].detach().float(), s["target"]
    keep = t != IGNORE
    n = keep.sum()
    at = t.clamp(min=0)[:, None]
    p = h @ w.T
    top = p.amax(1, keepdim=True)
    lse = torch.log(torch.exp(p - top).sum(1, keepdim=True)) + top
    loss = torch.where(keep, (lse - p.gather(1, at)).squeeze(1), 0.0).sum() / n
    p = torch.exp(p - lse)
    p.scatter_add_(1, at, torch.full_like(lse, -1.0))
    p *= (keep / n)[:, None]
    return loss, (p @ w).to(s["hidden"].dtype), (p.T @ h).to(s["weight"].dtype)


# ------------------------------------------------------------------------- own operators


def _run_own(s):
    import dynamic_conv1d_b200 as dc

    c = s["case"]
    op = c["op"]
    if op == "conv_step":
        if c["form"] == "lowrank":
            y = dc.lowrank_dynamic_convolution_grouped_step(s["x"], s["z"], s["U"], s["cache"], s["static_w"], residual=True, slots=s["slots"])
        else:
            y = dc.headwise_dynamic_convolution_step(s["x"], s["weight"], s["cache"], s["static_w"], residual=True, slots=s["slots"])
        return y, s["cache"]
    if op == "attn_step":
        o = dc.decay_linear_attention_step(s["q"], s["k"], s["v"], s["state"], s["log_decay"], slots=s["slots"])
        return o, s["state"]
    if op == "attn_prompt":
        return dc.decay_linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"], return_state=True)
    if op == "attn_train":
        o = dc.decay_linear_attention_fused(s["qkv"], s["log_decay"])
        (dx,) = torch.autograd.grad(o, s["qkv"], s["do"])
        return o.detach(), dx
    loss = dc.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE)
    dh, dw = torch.autograd.grad(loss, (s["hidden"], s["weight"]))
    return loss.detach(), dh, dw


_PLAIN = {"conv_step": _conv_step_plain, "attn_step": _attn_step_plain, "attn_prompt": _attn_prompt_plain,
          "attn_train": _attn_train_plain, "loss": _loss_plain}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# -------------------------------------------------------------------------- work, oracle


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "conv_step":
        B, G, D, W, R = (case[k] for k in ("B", "G", "D", "W", "R"))
        C = G * D
        io = B * C * 2 + B * (W - 1) * C * 2  # input, output, the rows' caches read and written
        if case["form"] == "lowrank":
            return dict(bytes=e * (io + B * G * R + G * R * W * D + W * C), flops=2 * B * C * W * (R + 1))
        return dict(bytes=e * (io + B * R * W + W * D), flops=2 * B * C * W)
    if op == "attn_step":
        B, H, dk, dv = (case[k] for k in ("B", "H", "dk", "dv"))
        return dict(bytes=B * H * (2 * 4 * dk * dv + e * (2 * dk + 2 * dv)), flops=5 * B * H * dk * dv)
    if op == "attn_prompt":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        return dict(bytes=B * H * (e * T * (2 * dk + 2 * dv) + 2 * 4 * dk * dv), flops=4 * B * T * H * dk * dv)
    if op == "attn_train":
        B, T, H, d = (case[k] for k in ("B", "T", "H", "dk"))
        # q, k, v and the output's gradient read, the output and three gradients written
        return dict(bytes=B * T * H * d * e * 8, flops=16 * B * T * H * d * d)
    N, D, V = (case[k] for k in ("N", "D", "V"))
    return dict(bytes=e * 2 * (N * D + V * D) + 8 * N, flops=6 * N * D * V)


def _exact_conv_step(s):
    c = s["case"]
    B, G, D, W = (c[k] for k in ("B", "G", "D", "W"))
    x, cache = s["x"].double(), s["cache"].double()
    rows = torch.arange(B, device=x.device) if s["slots"] is None else s["slots"].long()
    y, past = x.clone(), [x] + [cache[rows, W - 2 - j] for j in range(W - 1)]
    for w in range(W):
        if c["form"] == "lowrank":
            taps = torch.cat([s["z"].double()[:, g * c["R"]:(g + 1) * c["R"]] @ s["U"][g].double()[:, w * D:(w + 1) * D]
                              + s["static_w"][g, w].double() for g in range(G)], dim=1)
        else:
            taps = s["weight"].double()[:, :, w].repeat_interleave(D // c["R"], 1) + s["static_w"][w].double()
        y += taps * past[w]
    for j in range(W - 1):
        cache[rows, j] = past[W - 2 - j]
    return y, cache


def _exact_recurrence(q, k, v, log_decay, S):
    """o_t = scale * q_t S_t with S_t = decay * S_{t-1} + k_t (outer) v_t, token by token in 64 bits."""
    decay = torch.exp(log_decay.double())[:, None, None]
    o = torch.empty(*q.shape[:-1], v.shape[-1], device=q.device, dtype=torch.float64)
    for t in range(q.shape[1]):
        S.mul_(decay).addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        o[:, t] = (q[:, t, :, None, :] @ S).squeeze(-2)
    return o * q.shape[-1] ** -0.5


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv_step":
        return _exact_conv_step(s)
    if op == "attn_step":
        rows = torch.arange(case["B"], device="cuda") if s["slots"] is None else s["slots"].long()
        state = s["state"].double()
        S = state[rows]
        o = _exact_recurrence(*(s[k].double()[:, None] for k in ("q", "k", "v")), s["log_decay"], S)
        state[rows] = S
        return o[:, 0], state
    if op == "attn_prompt":
        S = s["state"].double()
        return _exact_recurrence(*(s[k].double() for k in ("q", "k", "v")), s["log_decay"], S), S
    if op == "attn_train":
        B, T, H, d = (case[k] for k in ("B", "T", "H", "dk"))
        q, k, v = s["qkv"].detach().double().view(B, T, 3, H, d).unbind(2)
        do = s["do"].double().view(B, T, H, d)
        zero = lambda: torch.zeros(B, H, d, d, device="cuda", dtype=torch.float64)  # noqa: E731
        o = _exact_recurrence(q, k, v, s["log_decay"], zero())
        # the gradients are the same recurrence with the tensors' parts exchanged:
        # dq_t = (sum_{j<=t} decay^(t-j) (do_t . v_j) k_j), and dk, dv run from the end
        back = lambda *t: [x.flip(1) for x in t]  # noqa: E731
        dq = _exact_recurrence(do, v, k, s["log_decay"], zero())
        dk = _exact_recurrence(*back(v, do, q), s["log_decay"], zero()).flip(1)
        dv = _exact_recurrence(*back(k, q, do), s["log_decay"], zero()).flip(1)
        return o.reshape(B, T, H * d), torch.stack([dq, dk, dv], dim=2).reshape(B, T, 3 * H * d)
    h, w, t = s["hidden"].detach().double(), s["weight"].detach().double(), s["target"]
    valid = torch.nonzero(t != IGNORE).squeeze(1)
    hv, tv = h[valid], t[valid]
    logits = hv @ w.T
    lse = torch.logsumexp(logits, dim=1)
    pick = torch.arange(len(valid), device="cuda")
    loss = (lse - logits[pick, tv]).mean()
    d = logits.sub_(lse[:, None]).exp_()
    d[pick, tv] -= 1.0
    d /= len(valid)
    dh = torch.zeros_like(h)
    dh[valid] = d @ w
    return loss, dh, d.T @ hv
