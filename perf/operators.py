"""Cases of the sequence operators that sit in front of the MPC solve: linear
attention with a decay per head (prompts, training, single tokens), the
residual addition with its root-mean-square norm, and the gated linear layer.

They are what a learned policy around the differentiable solver runs: an
encoder reads every environment's history of states and controls and emits the
solve's cost parameters.  Training runs whole histories of a batch of
environments forward and backward; the closed loop feeds one token per
environment and control tick.

``own`` selects who computes: the plain form (elementary torch operations in 32
bits, rounded once) or the package's operators.
"""
import math

import torch

own = False

CHUNK = 64  # tokens per step of the plain chunked form

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def _attention(name, batch, T, heads, kv_heads, dk, dv, dtype, lengths=False, state=False, train=False):
    return {"name": name, "op": "attention_train" if train else "attention", "batch": batch, "T": T, "heads": heads,
            "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype, "lengths": lengths, "state": state}


def _step(name, batch, heads, kv_heads, dk, dv, dtype):
    return {"name": name, "op": "step", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv,
            "dtype": dtype}


def _norm(name, rows, d, dtype, train=False):
    return {"name": name, "op": "norm_train" if train else "norm", "rows": rows, "d": d, "dtype": dtype}


def _gated(name, rows, d, f, dtype, activation="silu", train=False):
    return {"name": name, "op": "gated_train" if train else "gated", "rows": rows, "d": d, "f": f, "dtype": dtype,
            "activation": activation}


def listed():
    return [
        # One control tick of 64 environments, 32-bit: a launch's latency.
        _step("step_b64_f32", 64, 4, 4, 32, 32, "f32"),
        # One control tick of a full simulation batch: the states' bytes.
        _step("step_b16384_bf16", 16384, 4, 2, 64, 64, "bf16"),
        # Histories of one horizon length, of different lengths per environment; the state goes on into the closed loop.
        _attention("prompt_b1024_t61_bf16", 1024, 61, 4, 4, 64, 64, "bf16", lengths=True, state=True),
        # Two long logs continued from a state, key / value heads shared: few rows, a long axis.
        _attention("prompt_b2_t32749_bf16", 2, 32749, 8, 2, 128, 128, "bf16", state=True),
        # Training on short horizons in 32 bits, odd head sizes.
        _attention("train_b256_t51_f32", 256, 51, 4, 4, 32, 24, "f32", train=True),
        # Training on rollouts of different lengths, key / value heads shared.
        _attention("train_b1024_t301_bf16", 1024, 301, 8, 4, 64, 64, "bf16", lengths=True, train=True),
        # The norm of a small model's tokens, odd width, 32-bit.
        _norm("norm_r16384_d250_f32", 16384, 250, "f32"),
        # Training's norm over every token of the rollouts.
        _norm("norm_train_r308224_d512_bf16", 308224, 512, "bf16", train=True),
        # One control tick through the feed-forward of a small model: latency.
        _gated("gated_r64_d128_f341_f32", 64, 128, 341, "f32"),
        # A simulation batch's tick through a wider model.
        _gated("gated_r16384_d512_f1365_bf16", 16384, 512, 1365, "bf16"),
        # Training a small model in 32 bits, the other activation.
        _gated("gated_train_r15616_d128_f341_f32", 15616, 128, 341, "f32", "gelu", train=True),
        # Training the wider model over every token of the rollouts.
        _gated("gated_train_r308224_d512_f1365_bf16", 308224, 512, 1365, "bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "attention", "attention", "attention_train", "attention_train", "norm", "norm_train", "gated",
                     "gated_train"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "step":
        kv = rng.choice([1, 2, 4, 8])
        case = _step("", _log_int(rng, 1, 16384), kv * rng.choice([1, 1, 2, 4]), kv, rng.choice([16, 24, 32, 48, 64, 96, 128]),
                     rng.choice([16, 20, 32, 50, 64, 80, 128]), dtype)
        while case["batch"] * case["heads"] * case["dk"] * case["dv"] > 16384 * 4 * 64 * 64:
            case["batch"] = (case["batch"] + 1) // 2
    elif op in ("attention", "attention_train"):
        kv = rng.choice([1, 2, 4, 8])
        train = op == "attention_train"
        case = _attention("", _log_int(rng, 1, 4096), _log_int(rng, 1, 1024 if train else 32768),
                          kv * rng.choice([1, 1, 2, 4]), kv, rng.choice([16, 24, 32, 48, 64, 96, 128]),
                          rng.choice([16, 20, 32, 50, 64, 80, 128]), dtype, rng.random() < 0.5, rng.random() < 0.5, train)
        limit = (1024 * 301 * 8 * 64 * 64) if train else (2 * 32768 * 8 * 128 * 128)
        while case["batch"] * case["T"] * case["heads"] * case["dk"] * case["dv"] > limit:
            key = "batch" if case["batch"] > 1 else "T"
            case[key] = (case[key] + 1) // 2
    elif op in ("norm", "norm_train"):
        case = _norm("", _log_int(rng, 1, 308224), _log_int(rng, 16, 4096), dtype, op == "norm_train")
        while case["rows"] * case["d"] * _SIZE[dtype] > 308224 * 512 * 2:
            case["rows"] = (case["rows"] + 1) // 2
    else:
        train = op == "gated_train"
        case = _gated("", _log_int(rng, 1, 308224), _log_int(rng, 16, 1024), _log_int(rng, 32, 4096), dtype,
                      rng.choice(["silu", "gelu"]), train)
        limit = (308224 if train else 65536) * 512 * 1365 // (8 if dtype == "f32" else 1)
        while case["rows"] * case["d"] * case["f"] > limit or case["rows"] * case["f"] > 308224 * 1365:
            case["rows"] = (case["rows"] + 1) // 2
    del case["name"]
    return case


def work(case):
    """Each input read once, each output written once; the products of the
    recurrence (state update and read-out, their adjoints) and of the layers."""
    w = _SIZE[case["dtype"]]
    op = case["op"]
    if op == "step":
        B, H, G, dk, dv = (case[k] for k in ("batch", "heads", "kv_heads", "dk", "dv"))
        return {"bytes": 2 * 4 * B * H * dk * dv + w * B * (H * (dk + dv) + G * (dk + dv)) + 4 * H,
                "flops": 5 * B * H * dk * dv}
    if op in ("attention", "attention_train"):
        B, T, H, G, dk, dv = (case[k] for k in ("batch", "T", "heads", "kv_heads", "dk", "dv"))
        tokens = B * T  # lengths are drawn over 0..T: half the tokens on average
        if case["lengths"]:
            tokens = B * T // 2
        qk, vo = w * H * dk, w * H * dv
        kv = w * G * (dk + dv)
        st = 4 * B * H * dk * dv
        padded_o = B * T * vo
        if op == "attention":
            return {"bytes": tokens * (qk + kv) + padded_o + (2 * st if case["state"] else 0),
                    "flops": 4 * tokens * H * dk * dv}
        return {"bytes": tokens * (qk + kv) + padded_o + tokens * (qk + vo + kv) + B * T * (qk + kv)
                + (2 * st if case["state"] else 0),
                "flops": 14 * tokens * H * dk * dv}
    if op == "norm":
        n = case["rows"] * case["d"]
        return {"bytes": 4 * w * n + w * case["d"], "flops": 6 * n}
    if op == "norm_train":
        n = case["rows"] * case["d"]
        return {"bytes": (4 + 4) * w * n + 2 * w * case["d"], "flops": 18 * n}
    N, d, f = case["rows"], case["d"], case["f"]
    if op == "gated":
        return {"bytes": w * (N * d + 2 * d * f + N * f), "flops": 4 * N * d * f + 6 * N * f}
    return {"bytes": w * (N * d + 2 * d * f + N * f) + w * (N * f + N * d + 2 * d * f + N * d + 2 * d * f),
            "flops": 12 * N * d * f + 20 * N * f}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _decay(heads):
    """log of 1 - 2^-i, i spread over 2..7 across the heads: memories of 4 to 128 tokens."""
    i = 2.0 + 5.0 * torch.arange(heads, dtype=torch.float64) / max(heads - 1, 1)
    return torch.log1p(-torch.exp2(-i)).float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        x = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
        return (x.mul_(std) if std != 1.0 else x).to(dtype)

    op = case["op"]
    s = {"case": case}
    if op == "step":
        B, H, G, dk, dv = (case[k] for k in ("batch", "heads", "kv_heads", "dk", "dv"))
        s.update(q=normal(B, H, dk), k=normal(B, G, dk), v=normal(B, G, dv), log_decay=_decay(H),
                 state=normal(B, H, dk, dv, std=2.0, dtype=torch.float32))
        s["state_out"] = torch.empty_like(s["state"])
    elif op in ("attention", "attention_train"):
        B, T, H, G, dk, dv = (case[k] for k in ("batch", "T", "heads", "kv_heads", "dk", "dv"))
        s.update(q=normal(B, T, H, dk), k=normal(B, T, G, dk), v=normal(B, T, G, dv), log_decay=_decay(H))
        s["initial"] = normal(B, H, dk, dv, std=2.0, dtype=torch.float32) if case["state"] else None
        s["lengths"] = None
        if case["lengths"]:
            s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        if op == "attention_train":
            s["do"] = normal(B, T, H, dv)
            for key in ("q", "k", "v", "log_decay", "initial"):
                if s[key] is not None:
                    s[key].requires_grad_(True)
    elif op in ("norm", "norm_train"):
        N, d = case["rows"], case["d"]
        s.update(x=normal(N, d), residual=normal(N, d, std=2.0), weight=(1.0 + normal(d, std=0.1, dtype=torch.float32)).to(dt))
        if op == "norm_train":
            s.update(dy=normal(N, d), ds=normal(N, d))
            for key in ("x", "residual", "weight"):
                s[key].requires_grad_(True)
    else:
        N, d, f = case["rows"], case["d"], case["f"]
        s.update(x=normal(N, d), w_gate=normal(f, d, std=d ** -0.5), w_up=normal(f, d, std=d ** -0.5))
        if op == "gated_train":
            s["dh"] = normal(N, f)
            for key in ("x", "w_gate", "w_up"):
                s[key].requires_grad_(True)
    return s


# --------------------------------------------------------------------------
# Plain forms
# --------------------------------------------------------------------------
def _plain_attention(q, k, v, log_decay, initial, lengths):
    """Chunks of CHUNK tokens: the masked product within a chunk, the state before it."""
    dt = q.dtype
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    rep = H // k.shape[2]
    q = q.float() * dk ** -0.5
    k, v, g = k.float().repeat_interleave(rep, 2), v.float().repeat_interleave(rep, 2), log_decay
    S = torch.zeros(B, H, dk, dv, device=q.device) if initial is None else initial
    if lengths is not None:
        alive = (torch.arange(T, device=q.device)[None, :] < lengths[:, None]).float()
        q, k, v = (x * alive[:, :, None, None] for x in (q, k, v))
    out = []
    for t0 in range(0, T, CHUNK):
        qc, kc, vc = (x[:, t0:t0 + CHUNK].transpose(1, 2) for x in (q, k, v))  # (B, H, C, D)
        C = qc.shape[2]
        pos = torch.arange(C, device=q.device)
        lag = (pos[:, None] - pos[None, :]).float()
        mask = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), torch.zeros((), device=q.device))
        o = (qc @ kc.transpose(2, 3) * mask) @ vc
        o = o + torch.exp(g[:, None] * (pos + 1))[..., None] * (qc @ S)
        out.append(o.transpose(1, 2))
        if lengths is None:
            left = torch.full((B, 1), C, device=q.device)
        else:
            left = (lengths - t0).clamp(0, C)[:, None]
        lag_end = (left[:, None, :] - 1 - pos[None, None, :]).clamp(min=0).float()  # (B, 1, C)
        kd = kc * torch.exp(g[None, :, None] * lag_end)[..., None]
        S = torch.exp(g[None, :] * left)[..., None, None] * S + kd.transpose(2, 3) @ vc
    return torch.cat(out, 1).to(dt), S


def _plain_step(q, k, v, log_decay, state):
    rep = q.shape[1] // k.shape[1]
    kf, vf = k.float().repeat_interleave(rep, 1), v.float().repeat_interleave(rep, 1)
    S = torch.exp(log_decay)[None, :, None, None] * state + kf[..., None] * vf[:, :, None, :]
    o = ((q.float() * q.shape[-1] ** -0.5)[..., None] * S).sum(2)
    return o.to(q.dtype), S


def _plain_norm(x, residual, weight):
    s = x.float() + residual.float()
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-6) * weight.float()
    return y.to(x.dtype), s.to(x.dtype)


def _plain_act(g, activation):
    if activation == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.erf(g * 2 ** -0.5))


def _plain_gated(x, w_gate, w_up, activation):
    xf = x.float()
    return (_plain_act(xf @ w_gate.float().t(), activation) * (xf @ w_up.float().t())).to(x.dtype)


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from turbompc_b200 import sequence
    if op == "step":
        if own:
            o = sequence.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"],
                                               state_out=s["state_out"])
            return [o, s["state_out"]]
        return list(_plain_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]))
    if op in ("attention", "attention_train"):
        if own:
            o, S = sequence.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial"],
                                             lengths=s["lengths"], return_state=True)
        else:
            o, S = _plain_attention(s["q"], s["k"], s["v"], s["log_decay"], s["initial"], s["lengths"])
        if op == "attention":
            return [o, S]
        leaves = [s[key] for key in ("q", "k", "v", "log_decay", "initial") if s[key] is not None]
        return [o.detach(), *torch.autograd.grad(o, leaves, s["do"])]
    if op in ("norm", "norm_train"):
        fn = sequence.add_rms_norm if own else _plain_norm
        y, r = fn(s["x"], s["residual"], s["weight"])
        if op == "norm":
            return [y, r]
        return [y.detach(), r.detach(),
                *torch.autograd.grad([y, r], [s["x"], s["residual"], s["weight"]], [s["dy"], s["ds"]])]
    if own:
        h = sequence.gated_linear(s["x"], s["w_gate"], s["w_up"], activation=case["activation"])
    else:
        h = _plain_gated(s["x"], s["w_gate"], s["w_up"], case["activation"])
    if op == "gated":
        return [h]
    return [h.detach(), *torch.autograd.grad(h, [s["x"], s["w_gate"], s["w_up"]], s["dh"])]


# --------------------------------------------------------------------------
# Exact values (64 bits, token by token, gradients by the adjoint recurrences)
# --------------------------------------------------------------------------
def _exact_attention(s, train):
    c = s["case"]
    B, T, H, G, dk, dv = (c[k] for k in ("batch", "T", "heads", "kv_heads", "dk", "dv"))
    rep, scale = H // G, dk ** -0.5
    lam = torch.exp(s["log_decay"].detach().double())[None, :, None, None]
    o_all = torch.empty(B, T, H, dv, dtype=torch.float64, device="cuda")
    S_all = torch.empty(B, H, dk, dv, dtype=torch.float64, device="cuda")
    per = (T if train else 4) * H * dk * dv * 8
    block = max(1, min(B, int(12e9) // per))
    grads = []
    for b0 in range(0, B, block):
        sl = slice(b0, min(B, b0 + block))
        q, k, v = (s[key].detach()[sl].double() for key in ("q", "k", "v"))
        nb = q.shape[0]
        on = torch.ones(nb, T, dtype=torch.bool, device="cuda")
        if s["lengths"] is not None:
            on = torch.arange(T, device="cuda")[None, :] < s["lengths"][sl][:, None]
        S = torch.zeros(nb, H, dk, dv, dtype=torch.float64, device="cuda")
        if s["initial"] is not None:
            S = s["initial"].detach()[sl].double()
        kept = []
        for t in range(T):
            live = on[:, t, None, None, None]
            kt, vt = (x[:, t, :, None, :].expand(nb, G, rep, x.shape[-1]).reshape(nb, H, -1) for x in (k, v))
            if train:
                kept.append(S)  # the state before token t
            S = torch.where(live, lam * S + kt[:, :, :, None] * vt[:, :, None, :], S)
            o_all[sl, t] = torch.where(live[..., 0], scale * torch.einsum("bhk,bhkv->bhv", q[:, t], S), 0.0)
        S_all[sl] = S
        if not train:
            continue
        do = s["do"][sl].double()
        dq = torch.zeros_like(q)
        dk_, dv_ = torch.zeros_like(k), torch.zeros_like(v)
        dg = torch.zeros(H, dtype=torch.float64, device="cuda")
        dS = torch.zeros_like(S)
        after = S
        for t in range(T - 1, -1, -1):
            live = on[:, t, None, None, None]
            before = kept.pop()
            kt, vt = (x[:, t, :, None, :].expand(nb, G, rep, x.shape[-1]).reshape(nb, H, -1) for x in (k, v))
            dot = do[:, t] * on[:, t, None, None]
            dq[:, t] = scale * torch.einsum("bhkv,bhv->bhk", after, dot)
            dS = dS + scale * q[:, t, :, :, None] * dot[:, :, None, :]
            zero = dS * live
            dk_[:, t] = torch.einsum("bhkv,bhv->bhk", zero, vt).view(nb, G, rep, dk).sum(2)
            dv_[:, t] = torch.einsum("bhkv,bhk->bhv", zero, kt).view(nb, G, rep, dv).sum(2)
            dg += (zero * lam * before).sum((0, 2, 3))
            dS = torch.where(live, lam * dS, dS)
            after = before
        grads.append((dq, dk_, dv_, dg, dS))
    if not train:
        return [o_all, S_all]
    cat = [torch.cat([g[i] for g in grads]) for i in (0, 1, 2)]
    out = [o_all, *cat, sum(g[3] for g in grads)]
    if s["initial"] is not None:
        out.append(torch.cat([g[4] for g in grads]))
    return out


def _exact_norm(s, train):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    t = x + s["residual"].detach().double()
    r = 1.0 / torch.sqrt(t.pow(2).sum(-1, keepdim=True) / t.shape[-1] + 1e-6)
    out = [t * r * w, t]
    if train:
        dy, ds = s["dy"].double(), s["ds"].double()
        p = dy * w
        dt = ds + r * p - t * r.pow(3) * (p * t).sum(-1, keepdim=True) / t.shape[-1]
        out += [dt, dt, (dy * t * r).sum(0)]
    return out


def _exact_gated(s, train):
    x, wg, wu = (s[key].detach().double() for key in ("x", "w_gate", "w_up"))
    g, u = torch.mm(x, wg.T), torch.mm(x, wu.T)
    if s["case"]["activation"] == "silu":
        sig = torch.sigmoid(g)
        a, da = g * sig, sig * (1 + g * (1 - sig))
        del sig
    else:
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        a, da = g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        del cdf
    out = [a * u]
    if train:
        dh = s["dh"].double()
        du = dh * a
        dg = dh.mul_(u).mul_(da)
        del a, da, g, u
        out += [torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.T, x), torch.mm(du.T, x)]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "step":
        B, H, G, dk, dv = (case[k] for k in ("batch", "heads", "kv_heads", "dk", "dv"))
        k, v = (s[key].double()[:, :, None].expand(B, G, H // G, s[key].shape[-1]).reshape(B, H, -1) for key in ("k", "v"))
        S = torch.exp(s["log_decay"].double()).view(1, H, 1, 1) * s["state"].double()
        S += torch.einsum("bhk,bhv->bhkv", k, v)
        return [torch.einsum("bhk,bhkv->bhv", s["q"].double(), S) / math.sqrt(dk), S]
    if op in ("attention", "attention_train"):
        return _exact_attention(s, op == "attention_train")
    if op in ("norm", "norm_train"):
        return _exact_norm(s, op == "norm_train")
    return _exact_gated(s, op == "gated_train")
