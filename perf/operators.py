"""The sequence-policy operators as measured work: the gated linear recurrence, token log-probs and
entropies from logits, the clipped policy loss with its gradients and the preference loss with its
gradients.

`listed()` and `draw()` give the cases, `prepare()` a case's inputs on the GPU, `run()` one pass (the
package's operators where `own` is true, elementary torch operations in 32 bits otherwise), `exact()`
the same outputs in 64 bits from the definitions, and `work()` the bytes and operations that a pass
cannot do without.
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100


def _ops():
    return importlib.import_module("cuda-optimization-benchmark_b200").ops


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One token for each of 64 sequences being generated, their states in a pool of 80 slots.
        {"name": "recurrence step", "op": "rec_step", "B": 64, "H": 2048, "slots": 80, "dtype": "bf16",
         "form": "sigmoid"},
        # Training on packed documents of odd sizes: gate and input are halves of one projection.
        {"name": "recurrence ragged train", "op": "rec_train", "B": 3, "T": 1003, "H": 770, "dtype": "fp16",
         "form": "decay", "reset": True, "time_first": False},
        # Training at an ordinary size: a layer of 2048 channels over 8 sequences of 4096 steps.
        {"name": "recurrence train", "op": "rec_train", "B": 8, "T": 4096, "H": 2048, "dtype": "bf16",
         "form": "sigmoid", "reset": False, "time_first": False},
        # Reading one long sequence in before generating from it.
        {"name": "recurrence long read", "op": "rec_fwd", "B": 1, "T": 65539, "H": 1024, "dtype": "fp32",
         "form": "decay", "reset": False, "time_first": False},
        # Scoring one new token of each of 16 sequences.
        {"name": "logprob 16 rows", "op": "lp_fwd", "B": 16, "T": 1, "V": 32768, "dtype": "bf16", "shift": False,
         "entropy": True, "temperature": 0.7},
        # Training on next tokens (logits[:, :-1] against token[:, 1:]) with an odd vocabulary.
        {"name": "logprob odd vocabulary train", "op": "lp_train", "B": 4, "T": 511, "V": 50001, "dtype": "bf16",
         "shift": True, "entropy": True, "temperature": 1.0},
        # Training with a large vocabulary, no entropy term.
        {"name": "logprob large train", "op": "lp_train", "B": 8, "T": 512, "V": 131072, "dtype": "bf16",
         "shift": False, "entropy": False, "temperature": 1.0},
        # A small update: 16 short answers against a reference policy.
        {"name": "policy small", "op": "policy", "B": 16, "T": 256, "ref": True, "entropy": False, "kl": "k3",
         "reduction": "token_mean", "dual": 0.0, "adv_rows": True},
        # Long answers of odd length, every sequence weighted alike, dual clipping.
        {"name": "policy ragged", "op": "policy", "B": 61, "T": 4099, "ref": True, "entropy": False, "kl": "k2",
         "reduction": "sequence_mean", "dual": 3.0, "adv_rows": True},
        # The RL batch of the repository's benchmark, 4096 trajectories of 1000 steps, with an entropy bonus.
        {"name": "policy batch", "op": "policy", "B": 4096, "T": 1000, "ref": False, "entropy": True, "kl": "k1",
         "reduction": "token_mean", "dual": 0.0, "adv_rows": False},
        # A few pairs of odd lengths.
        {"name": "preference small", "op": "pref", "B": 4, "Tc": 700, "Tr": 523, "ref": True, "form": "sigmoid",
         "average": False, "smoothing": 0.1},
        # A large batch of long pairs.
        {"name": "preference large", "op": "pref", "B": 512, "Tc": 8192, "Tr": 8192, "ref": True, "form": "sigmoid",
         "average": False, "smoothing": 0.0},
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rec_step", "rec_train", "rec_train", "rec_fwd", "lp_fwd", "lp_train", "policy", "policy",
                     "pref", "pref"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    form = rng.choice(["decay", "sigmoid"])
    if op == "rec_step":
        B = _log_int(rng, 1, 1024)
        return {"op": op, "B": B, "H": _log_int(rng, 64, 8192), "slots": B + rng.randint(0, 64), "dtype": dtype,
                "form": form}
    if op in ("rec_train", "rec_fwd"):
        H = _log_int(rng, 33, 4096)
        B = _log_int(rng, 1, 32)
        most = (1 << 25) // (B * H)
        T = _log_int(rng, 1, max(1, min(65536, most)))
        return {"op": op, "B": B, "T": T, "H": H, "dtype": dtype, "form": form, "reset": rng.random() < 0.5,
                "time_first": rng.random() < 0.3}
    if op in ("lp_fwd", "lp_train"):
        V = _log_int(rng, 2, 200000)
        B = _log_int(rng, 1, 16)
        T = _log_int(rng, 1, max(1, min(2048, (1 << 27) // (B * V))))
        return {"op": op, "B": B, "T": T, "V": V, "dtype": dtype, "shift": rng.random() < 0.5,
                "entropy": rng.random() < 0.5, "temperature": rng.choice([0.6, 1.0, 1.3])}
    if op == "policy":
        B = _log_int(rng, 1, 4096)
        T = _log_int(rng, 1, max(1, min(32768, (1 << 22) // B)))
        return {"op": op, "B": B, "T": T, "ref": rng.random() < 0.6, "entropy": rng.random() < 0.5,
                "kl": rng.choice(["k1", "k2", "k3"]),
                "reduction": rng.choice(["token_mean", "sequence_mean", "sum"]), "dual": rng.choice([0.0, 3.0]),
                "adv_rows": rng.random() < 0.5}
    B = _log_int(rng, 1, 512)
    most = min(131072, (1 << 22) // B)
    return {"op": "pref", "B": B, "Tc": _log_int(rng, 1, most), "Tr": _log_int(rng, 1, most),
            "ref": rng.random() < 0.7, "form": rng.choice(["sigmoid", "hinge", "ipo"]),
            "average": rng.random() < 0.4, "smoothing": rng.choice([0.0, 0.1])}


# ------------------------------------------------------------------------------------- the inputs
def _lengths_mask(B, T, g):
    """Answers of random lengths behind prompts of random lengths; about one row in 16 is empty."""
    start = (torch.rand(B, generator=g, device="cuda") * 0.2 * T).floor()
    length = (torch.rand(B, generator=g, device="cuda") * (T - start)).ceil()
    length = torch.where(torch.rand(B, generator=g, device="cuda") < 0.06, torch.zeros_like(length), length)
    t = torch.arange(T, device="cuda", dtype=torch.float32)
    return (t >= start[:, None]) & (t < (start + length)[:, None])


def _recurrence_inputs(case, g):
    B, T, H = case["B"], case.get("T", 1), case["H"]
    dt = DTYPES[case["dtype"]]
    # One projection [B, T, 2H] (or time first) whose halves are the gate and the input.
    shape = (T, B, 2 * H) if case.get("time_first") else (B, T, 2 * H)
    proj = torch.randn(shape, generator=g, device="cuda")
    proj[..., :H] = proj[..., :H] * 1.5 + 2.0
    if case["form"] == "decay":
        proj[..., :H] = torch.sigmoid(proj[..., :H])
    proj = proj.to(dt)
    if case.get("time_first"):
        proj = proj.transpose(0, 1)
    return proj[..., :H], proj[..., H:]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "rec_step":
        B, H, S = case["B"], case["H"], case["slots"]
        gate, x = _recurrence_inputs(case, g)
        s["gate"], s["x"] = gate[:, 0], x[:, 0]
        s["pool"] = torch.randn(S, H, generator=g, device="cuda")
        s["slots"] = torch.randperm(S, generator=g, device="cuda")[:B].to(torch.int32)
        s["next"] = s["pool"].clone()
    elif op in ("rec_train", "rec_fwd"):
        B, T, H = case["B"], case["T"], case["H"]
        s["gate"], s["x"] = _recurrence_inputs(case, g)
        s["state"] = torch.randn(B, H, generator=g, device="cuda")
        s["reset"] = (torch.rand(B, T, generator=g, device="cuda") < 0.01) if case["reset"] else None
        if op == "rec_train":
            s["grad"] = torch.randn(B, T, H, generator=g, device="cuda").to(DTYPES[case["dtype"]])
            s["grad_final"] = torch.randn(B, H, generator=g, device="cuda")
    elif op in ("lp_fwd", "lp_train"):
        B, T, V = case["B"], case["T"], case["V"]
        Tf = T + 1 if case["shift"] else T
        logits = torch.empty(B, Tf, V, device="cuda", dtype=DTYPES[case["dtype"]])
        for b in range(B):  # a sequence at a time keeps the 32-bit copy small
            logits[b] = torch.randn(Tf, V, generator=g, device="cuda") * 2.5
        token = torch.randint(0, V, (B, Tf), generator=g, device="cuda")
        token = torch.where(torch.rand(B, Tf, generator=g, device="cuda") < 0.1, torch.full_like(token, IGNORE), token)
        s["logits"] = logits[:, :-1] if case["shift"] else logits
        s["token"] = token[:, 1:] if case["shift"] else token
        if op == "lp_train":
            s["grad"] = torch.randn(B, T, generator=g, device="cuda")
            s["grad_ent"] = torch.randn(B, T, generator=g, device="cuda") * 0.3 if case["entropy"] else None
    elif op == "policy":
        B, T = case["B"], case["T"]
        s["cur"] = -(torch.randn(B, T, generator=g, device="cuda") * 0.5 - 1.0).abs()
        s["old"] = s["cur"] + 0.1 * torch.randn(B, T, generator=g, device="cuda")
        s["ref"] = s["cur"] + 0.2 * torch.randn(B, T, generator=g, device="cuda") if case["ref"] else None
        s["ent"] = 2.0 * torch.rand(B, T, generator=g, device="cuda") if case["entropy"] else None
        s["adv"] = torch.randn(*((B,) if case["adv_rows"] else (B, T)), generator=g, device="cuda")
        s["mask"] = _lengths_mask(B, T, g)
    else:
        B, Tc, Tr = case["B"], case["Tc"], case["Tr"]
        for k, T in (("c", Tc), ("r", Tr)):
            s["lp_" + k] = -(torch.randn(B, T, generator=g, device="cuda") * 0.5 - 1.0).abs()
            s["ref_" + k] = s["lp_" + k] + 0.05 * torch.randn(B, T, generator=g, device="cuda") if case["ref"] else None
            s["mask_" + k] = _lengths_mask(B, T, g)
    return s


POLICY = {"clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.05, "entropy_coef": 0.01, "scale": 0.5}
PREF = {"beta": 0.1}


def _policy_options(c):
    return {"clip_low": POLICY["clip_low"], "clip_high": POLICY["clip_high"],
            "dual_clip": c["dual"] if c["dual"] else None, "kl_coef": POLICY["kl_coef"] if c["ref"] else 0.0,
            "kl_form": c["kl"], "entropy_coef": POLICY["entropy_coef"] if c["entropy"] else 0.0,
            "reduction": c["reduction"], "scale": POLICY["scale"]}


# ------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ops, c = _ops(), s["case"]
    op = c["op"]
    if op == "rec_step":
        h = ops.linear_recurrence_step(s["gate"], s["x"], s["pool"], slots=s["slots"], form=c["form"],
                                       state_out=s["next"])
        return {"h": h, "state": s["next"]}
    if op == "rec_fwd":
        h, final = ops.linear_recurrence(s["gate"], s["x"], s["state"], reset=s["reset"], form=c["form"])
        return {"h": h, "final": final}
    if op == "rec_train":
        h, final, ck = ops.linear_recurrence_train(s["gate"], s["x"], s["state"], reset=s["reset"], form=c["form"])
        gg, gx, gs = ops.linear_recurrence_backward(s["gate"], s["x"], ck, s["grad"], s["grad_final"],
                                                    reset=s["reset"], form=c["form"])
        return {"h": h, "final": final, "grad_gate": gg, "grad_x": gx, "grad_state": gs}
    if op == "lp_fwd":
        lp, ent = ops.token_logprob(s["logits"], s["token"], c["temperature"], entropy=c["entropy"])
        return {"log_prob": lp, "entropy": ent} if c["entropy"] else {"log_prob": lp}
    if op == "lp_train":
        lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"], c["temperature"], entropy=c["entropy"])
        gl = ops.token_logprob_backward(s["logits"], s["token"], stats, s["grad"], s["grad_ent"], c["temperature"])
        return {"log_prob": lp, "entropy": ent, "grad_logits": gl} if c["entropy"] else \
            {"log_prob": lp, "grad_logits": gl}
    if op == "policy":
        out, grad, grad_ent = ops.policy_loss_grad(s["cur"], s["old"], s["adv"], mask=s["mask"],
                                                   ref_log_prob=s["ref"], entropy=s["ent"], **_policy_options(c))
        return {"out": out, "grad": grad, "grad_entropy": grad_ent} if c["entropy"] else {"out": out, "grad": grad}
    out, rc, rr, gc, gr = ops.preference_loss_grad(
        s["lp_c"], s["lp_r"], s["ref_c"], s["ref_r"], s["mask_c"], s["mask_r"], beta=PREF["beta"], form=c["form"],
        label_smoothing=c["smoothing"] if c["form"] == "sigmoid" else 0.0, average=c["average"])
    return {"out": out, "reward_chosen": rc, "reward_rejected": rr, "grad_chosen": gc, "grad_rejected": gr}


def _scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1 from h = 0, by doubling."""
    k, T = 1, b.shape[1]
    while k < T:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _coefficients(c, gate, x):
    if c["form"] == "decay":
        return gate.float(), x.float()
    f = 1 / (1 + torch.exp(-gate.float()))
    return f, (1 - f) * x.float()


def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op == "rec_step":
        a, b = _coefficients(c, s["gate"], s["x"])
        idx = s["slots"].long()
        h = a * s["pool"][idx] + b
        nxt = s["pool"].clone()
        nxt[idx] = h
        return {"h": h.to(s["x"].dtype), "state": nxt}
    if op in ("rec_fwd", "rec_train"):
        a, b = _coefficients(c, s["gate"], s["x"])
        keep = a if s["reset"] is None else a * (~s["reset"]).unsqueeze(-1)
        b0 = b.clone()
        b0[:, 0] += keep[:, 0] * s["state"]
        h = _scan(keep, b0)
        dt = s["x"].dtype
        if op == "rec_fwd":
            return {"h": h.to(dt), "final": h[:, -1].clone()}
        d = s["grad"].float()
        d[:, -1] += s["grad_final"]
        nxt = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
        g = _scan(nxt.flip(1), d.flip(1)).flip(1)
        prev = torch.cat([s["state"].unsqueeze(1), h[:, :-1]], 1)
        if s["reset"] is not None:
            prev = prev * (~s["reset"]).unsqueeze(-1)
        if c["form"] == "decay":
            gg, gx = g * prev, g
        else:
            gg, gx = g * (prev - s["x"].float()) * a * (1 - a), (1 - a) * g
        return {"h": h.to(dt), "final": h[:, -1].clone(), "grad_gate": gg.to(dt), "grad_x": gx.to(dt),
                "grad_state": keep[:, 0] * g[:, 0]}
    if op in ("lp_fwd", "lp_train"):
        x, tok = s["logits"], s["token"]
        inv = 1.0 / c["temperature"]
        on = tok >= 0
        at = torch.where(on, tok, torch.zeros_like(tok)).unsqueeze(-1)
        z = x.float()
        z = (z - z.amax(-1, keepdim=True)) * inv
        e = torch.exp(z)
        total = e.sum(-1, keepdim=True)
        log_total = torch.log(total)
        zero = torch.zeros((), device=z.device)
        lp = torch.where(on, (z.gather(-1, at) - log_total).squeeze(-1), zero)
        out = {"log_prob": lp}
        if c["entropy"]:
            ent = (log_total - (e * z).sum(-1, keepdim=True) / total)
            out["entropy"] = torch.where(on, ent.squeeze(-1), zero)
        if op == "lp_train":
            p = e / total
            del e
            gl = p * (-s["grad"].unsqueeze(-1))
            gl.scatter_add_(-1, at, s["grad"].unsqueeze(-1))
            if c["entropy"]:
                gl -= s["grad_ent"].unsqueeze(-1) * p * (z - log_total + ent)
            out["grad_logits"] = (gl * (inv * on.unsqueeze(-1))).to(x.dtype)
        return out
    if op == "policy":
        o, m = _policy_options(c), s["mask"]
        cur, A = s["cur"], s["adv"] if s["adv"].dim() == 2 else s["adv"].unsqueeze(1)
        A = A.expand_as(cur)
        wide = cur.double() - s["old"].double()  # decisions at the borders need the exact difference
        high, low = wide > math.log1p(o["clip_high"]), wide < math.log1p(-o["clip_low"])
        d = wide.float()
        r = torch.exp(d)
        clipped = ((A > 0) & high) | ((A < 0) & low)
        bound = torch.where(high, 1 + o["clip_high"], 1 - o["clip_low"])
        pg = -torch.where(clipped, bound, r) * A
        if o["dual_clip"]:
            dual = (A < 0) & (wide > math.log(o["dual_clip"]))
            pg = torch.where(dual, -o["dual_clip"] * A, pg)
            clipped = clipped | dual
        dpg = torch.where(clipped, torch.zeros_like(r), -r * A)
        n_row = m.sum(1)
        if o["reduction"] == "token_mean":
            w = torch.full_like(cur, o["scale"]) / m.sum().clamp(min=1)
        elif o["reduction"] == "sequence_mean":
            w = (o["scale"] / ((n_row > 0).sum().clamp(min=1) * n_row.clamp(min=1).double())).float()
            w = w.unsqueeze(1).expand_as(cur)
        else:
            w = torch.full_like(cur, o["scale"])
        w = w * m
        zero = torch.zeros((), device=cur.device, dtype=torch.float64)
        kl, ent, grad = zero, zero, dpg
        if s["ref"] is not None:
            q = s["ref"].double() - cur.double()
            if o["kl_form"] == "k1":
                k, dk = -q, torch.ones_like(cur)
            elif o["kl_form"] == "k2":
                k, dk = 0.5 * q * q, -q.float()
            else:
                k, dk = torch.expm1(q) - q, -torch.expm1(q.float())
            kl = (k * w).sum()
            grad = grad + o["kl_coef"] * dk
        if s["ent"] is not None:
            ent = (s["ent"] * w).sum(dtype=torch.float64)
        pol = (pg * w).sum(dtype=torch.float64)
        n = m.sum().clamp(min=1)
        # The mean of (r - 1) - d loses its digits in 32 bits where d is small.
        appr = ((torch.expm1(wide) - wide) * m).sum() / n
        out = torch.stack([pol + o["kl_coef"] * kl - o["entropy_coef"] * ent, pol, kl, ent,
                           ((high | low) & m).sum() / n.double(), appr, torch.where(m, r, torch.zeros_like(r)).amax().double(),
                           (r * m).sum(dtype=torch.float64) / n]).float()
        res = {"out": out, "grad": grad * w}
        if s["ent"] is not None:
            res["grad_entropy"] = -o["entropy_coef"] * w
        return res
    # preference
    def total(k):
        m = s["mask_" + k]
        n = m.sum(1).clamp(min=1)
        v = s["lp_" + k].double()
        t = (v * m).sum(1)  # long sums whose difference is what counts
        u = (s["ref_" + k].double() * m).sum(1) if s["ref_" + k] is not None else torch.zeros_like(t)
        return ((t - u) / n, 1.0 / n) if c["average"] else (t - u, torch.ones_like(t))
    (tc, nc), (tr, nr) = total("c"), total("r")
    beta, B, form = PREF["beta"], c["B"], c["form"]
    z = beta * (tc - tr)
    if form == "sigmoid":
        e = c["smoothing"]
        loss = (1 - e) * _softplus(-z) + e * _softplus(z)
        dz = (1 - e) * -(1 / (1 + torch.exp(z))) + e * (1 / (1 + torch.exp(-z)))
    elif form == "hinge":
        loss, dz = (1 - z).clamp(min=0), torch.where(z < 1, -1.0, 0.0).double()
    else:
        u = z / beta - 1 / (2 * beta)
        loss, dz = u * u, 2 * u / beta
    k = beta * dz / B
    out = torch.stack([loss.mean(), (z > 0).double().mean(), z.mean()]).float()
    return {"out": out, "reward_chosen": (beta * tc).float(), "reward_rejected": (beta * tr).float(),
            "grad_chosen": (k * nc).float().unsqueeze(1) * s["mask_c"],
            "grad_rejected": (-k * nr).float().unsqueeze(1) * s["mask_r"]}


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


# ------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op in ("rec_step", "rec_fwd", "rec_train"):
        gate, x = s["gate"].to(f64), s["x"].to(f64)
        f = gate if case["form"] == "decay" else torch.sigmoid(gate)
        b = x if case["form"] == "decay" else (1 - f) * x
        if op == "rec_step":
            h = torch.empty_like(b)
            pool = s["pool"].to(f64)
            for i, slot in enumerate(s["slots"].tolist()):
                h[i] = f[i] * pool[slot] + b[i]
                pool[slot] = h[i]
            return {"h": h, "state": pool}
        B, T, H = b.shape
        live = torch.ones(B, T, 1, dtype=f64, device="cuda") if s["reset"] is None else \
            (1.0 - s["reset"].to(f64)).unsqueeze(-1)
        h = torch.empty_like(b)
        cur = s["state"].to(f64)
        prev = torch.empty_like(b) if op == "rec_train" else None
        for t in range(T):
            before = cur * live[:, t]
            if prev is not None:
                prev[:, t] = before
            cur = f[:, t] * before + b[:, t]
            h[:, t] = cur
        res = {"h": h, "final": cur}
        if op == "rec_fwd":
            return res
        gx, gg = torch.empty_like(b), torch.empty_like(b)
        acc = s["grad_final"].to(f64)
        dh = s["grad"].to(f64)
        for t in range(T - 1, -1, -1):
            acc = acc + dh[:, t]
            if case["form"] == "decay":
                gx[:, t], gg[:, t] = acc, acc * prev[:, t]
            else:
                gx[:, t] = acc * (1 - f[:, t])
                gg[:, t] = acc * (prev[:, t] - x[:, t]) * f[:, t] * (1 - f[:, t])
            acc = acc * f[:, t] * live[:, t]
        res.update(grad_gate=gg, grad_x=gx, grad_state=acc)
        return res
    if op in ("lp_fwd", "lp_train"):
        B, T, V = s["logits"].shape
        rows = max(1, (1 << 27) // V)  # rows at a time: 1 GiB of 64-bit values
        tok = s["token"].reshape(-1)
        lps, ents, grads = [], [], []
        flat = s["logits"].reshape(-1, V)
        for r0 in range(0, B * T, rows):
            z = flat[r0:r0 + rows].to(f64) / case["temperature"]
            tk = tok[r0:r0 + rows]
            logp = z - torch.logsumexp(z, -1, keepdim=True)
            p = logp.exp()
            ent = -(p * logp).sum(-1)
            sel = torch.arange(len(tk), device="cuda")
            dead = tk < 0
            lp = logp[sel, tk.clamp(min=0)]
            lps.append(lp.masked_fill(dead, 0.0))
            ents.append(ent.masked_fill(dead, 0.0))
            if op == "lp_train":
                g = s["grad"].reshape(-1)[r0:r0 + rows].to(f64)
                d = -p * g[:, None]
                d[sel, tk.clamp(min=0)] += g
                if case["entropy"]:
                    d -= s["grad_ent"].reshape(-1)[r0:r0 + rows].to(f64)[:, None] * p * (logp + ent[:, None])
                d /= case["temperature"]
                d[dead] = 0.0
                grads.append(d.float() if case["dtype"] != "fp32" else d)
        res = {"log_prob": torch.cat(lps).view(B, T)}
        if case["entropy"]:
            res["entropy"] = torch.cat(ents).view(B, T)
        if op == "lp_train":
            res["grad_logits"] = torch.cat(grads).view(B, T, V)
        return res
    if op == "policy":
        return _exact_policy(case, s)
    return _exact_preference(case, s)


def _np(t):
    return None if t is None else t.cpu().numpy().astype(np.float64 if t.dtype != torch.bool else bool)


def _exact_policy(case, s):
    o = _policy_options(case)
    cur, old, m = _np(s["cur"]), _np(s["old"]), _np(s["mask"])
    A = _np(s["adv"])
    A = np.broadcast_to(A if A.ndim == 2 else A[:, None], cur.shape)
    d = cur - old
    ratio = np.exp(d)
    lo, hi = 1 - o["clip_low"], 1 + o["clip_high"]
    held = np.minimum(np.maximum(ratio, lo), hi)
    gain = np.minimum(ratio * A, held * A)
    through = ratio * A <= held * A
    if o["dual_clip"]:
        floor = o["dual_clip"] * A
        cut = (A < 0) & (gain < floor)
        gain, through = np.where(cut, floor, gain), through & ~cut
    slope = np.where(through, ratio * A, 0.0)
    counts = m.sum(1)
    if o["reduction"] == "token_mean":
        w = np.full(cur.shape, 1.0 / max(1, counts.sum()))
    elif o["reduction"] == "sequence_mean":
        w = np.broadcast_to((1.0 / (max(1, (counts > 0).sum()) * np.maximum(1, counts)))[:, None], cur.shape)
    else:
        w = np.ones(cur.shape)
    w = np.where(m, w * o["scale"], 0.0)
    grad, kl, ent = -slope, 0.0, 0.0
    if s["ref"] is not None:
        q = _np(s["ref"]) - cur
        form = o["kl_form"]
        k = {"k1": lambda: -q, "k2": lambda: q * q / 2, "k3": lambda: np.expm1(q) - q}[form]()
        dk = {"k1": lambda: np.ones_like(q), "k2": lambda: -q, "k3": lambda: 1 - np.exp(q)}[form]()
        kl = float((w * k).sum())
        grad = grad + o["kl_coef"] * dk
    if s["ent"] is not None:
        ent = float((w * _np(s["ent"])).sum())
    pol = -float((w * gain).sum())
    n = max(1, counts.sum())
    got = ratio[m]
    out = np.array([pol + o["kl_coef"] * kl - o["entropy_coef"] * ent, pol, kl, ent,
                    ((held != ratio) & m).sum() / n, (np.expm1(d) - d)[m].sum() / n, got.max() if got.size else 0.0,
                    got.sum() / n])
    res = {"out": out, "grad": grad * w}
    if s["ent"] is not None:
        res["grad_entropy"] = -o["entropy_coef"] * w
    return res


def _exact_preference(case, s):
    beta, B = PREF["beta"], case["B"]
    side = {}
    for k in "cr":
        m = _np(s["mask_" + k])
        gap = _np(s["lp_" + k]) - (_np(s["ref_" + k]) if s["ref_" + k] is not None else 0.0)
        n = np.maximum(1, m.sum(1)) if case["average"] else np.ones(B)
        side[k] = (np.where(m, gap, 0.0).sum(1) / n, m / n[:, None])
    z = beta * (side["c"][0] - side["r"][0])
    if case["form"] == "sigmoid":
        e = case["smoothing"]
        loss = (1 - e) * np.logaddexp(0, -z) + e * np.logaddexp(0, z)
        dz = e - 0.5 * (1 - np.tanh(z / 2))  # e - sigmoid(-z)
    elif case["form"] == "hinge":
        loss, dz = np.maximum(0, 1 - z), -(z < 1).astype(np.float64)
    else:
        u = z / beta - 0.5 / beta
        loss, dz = u ** 2, 2 * u / beta
    slope = (beta * dz / B)[:, None]
    return {"out": np.array([loss.mean(), (z > 0).mean(), z.mean()]), "reward_chosen": beta * side["c"][0],
            "reward_rejected": beta * side["r"][0], "grad_chosen": slope * side["c"][1],
            "grad_rejected": -slope * side["r"][1]}


# ------------------------------------------------------------------------- bytes and operations
def work(case):
    op = case["op"]
    if op == "rec_step":
        e = SIZE[case["dtype"]]
        n = case["B"] * case["H"]
        return {"bytes": n * (3 * e + 8) + 4 * case["B"], "flops": 4 * n}
    if op in ("rec_fwd", "rec_train"):
        e = SIZE[case["dtype"]]
        rows = case["B"] * case["H"]
        n = rows * case["T"]
        extra = case["B"] * case["T"] if case["reset"] else 0
        if op == "rec_fwd":
            return {"bytes": 3 * e * n + 8 * rows + extra, "flops": 4 * n}
        # gate, input and gradient read; h and both gradients written
        return {"bytes": 6 * e * n + 16 * rows + extra, "flops": 12 * n}
    if op in ("lp_fwd", "lp_train"):
        rows = case["B"] * case["T"]
        n = rows * case["V"]
        e = SIZE[case["dtype"]]
        both = op == "lp_train"
        return {"bytes": n * e * (2 if both else 1) + rows * (8 + 4 + (4 if case["entropy"] else 0) +
                                                               (8 if both else 0)),
                "flops": n * (10 if both else 5)}
    if op == "policy":
        n = case["B"] * case["T"]
        streams = 2 + (1 if case["ref"] else 0) + (1 if case["entropy"] else 0) + (0 if case["adv_rows"] else 1)
        return {"bytes": n * (4 * streams + 1 + 4 + (4 if case["entropy"] else 0)) +
                (4 * case["B"] if case["adv_rows"] else 0) + 32, "flops": 20 * n}
    n = case["B"] * (case["Tc"] + case["Tr"])
    return {"bytes": n * (4 * (2 if case["ref"] else 1) + 1 + 4) + 8 * case["B"] + 12, "flops": 4 * n}
