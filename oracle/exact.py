"""numpy restatement of each task's correctness oracle `reference_exact` (test infrastructure).

fp64 for pow_abs_sqrt_mean, ppo_clip, reward_to_go and efficient_kan; the fp32 step order for
leaky (whose oracle is the fp32 reference itself); fp64 then one rounding to bf16 for fp8_linear.
Each function cites the reference lines it restates.  Inputs are the dicts built by
`oracle.inputs` (torch CPU tensors or numpy arrays); outputs are numpy arrays keyed like the
reference's output names.
"""
import math

import numpy as np

TOLERANCE = {  # tasks/<task>/tests/task.json "tolerance"
    "pow_abs_sqrt_mean": (1e-3, 1e-3),
    "ppo_clip": (1e-5, 1e-4),
    "reward_to_go": (1e-5, 1e-5),
    "leaky": (1e-6, 1e-5),
    "efficient_kan": (1e-5, 1e-5),
    "fp8_linear": (1e-2, 1e-2),
}


def _np(t):
    if hasattr(t, "detach"):
        t = t.detach().cpu()
        if str(t.dtype) == "torch.float8_e4m3fn":
            return t.view(__import__("torch").uint8).numpy()
        if str(t.dtype) == "torch.bfloat16":
            return t.view(__import__("torch").int16).numpy().view(np.uint16)
        return t.numpy()
    return np.asarray(t)


# -------------------------------------------------------------------------------- robust-L1
def pow_abs_sqrt_mean(inp):
    """tasks/pow_abs_sqrt_mean/reference.py:22-24,31-32: mean(sqrt(|a-b|^2 + 0.001*0.001)) in fp64."""
    a = _np(inp["inp"]).astype(np.float64).ravel()
    b = _np(inp["target"]).astype(np.float64).ravel()
    d = np.abs(a - b)
    v = np.sqrt(d * d + (0.001 * 0.001))
    return {"output": np.array(v.mean() if v.size else np.nan)}


# ------------------------------------------------------------------------------------- PPO
def _logsumexp(v):
    m = np.max(v)
    return m + math.log(np.sum(np.exp(v - m)))


def ppo_clip(inp, entropy=None):
    """tasks/ppo_clip/reference.py:27-35,42-45 in fp64, eps first rounded to fp32 (:43).

    With `entropy`, a 7th value (its mean) is appended: the extended form's diagnostic.
    """
    cur = _np(inp["current_log_prob"]).astype(np.float64).ravel()
    old = _np(inp["old_log_prob"]).astype(np.float64).ravel()
    adv = _np(inp["advantage"]).astype(np.float64).ravel()
    eps = float(np.float32(inp["clip_epsilon"]))
    lw = cur - old
    ratio = np.exp(lw)
    lwc = np.clip(lw, math.log1p(-eps), math.log1p(eps))
    gain = np.minimum(ratio * adv, np.exp(lwc) * adv)
    n = lw.size
    ess = math.exp(2.0 * _logsumexp(lw) - _logsumexp(2.0 * lw)) / n
    out = [-gain.mean(), (lwc != lw).astype(np.float64).mean(), ((ratio - 1.0) - lw).mean(), ess, ratio.max(),
           ratio.mean()]
    if entropy is not None:
        out.append(_np(entropy).astype(np.float64).mean())
    return {"output": np.array(out)}


# ---------------------------------------------------------------------------- reward-to-go
def reward_to_go(inp):
    """tasks/reward_to_go/reference.py:34-42: fp64 backward loop, nxt = r + gamma*keep*nxt."""
    r = _np(inp["reward"]).astype(np.float64)
    keep = (~_np(inp["done"]).astype(bool)).astype(np.float64)
    gamma = float(inp["gamma"])
    out = np.empty_like(r)
    nxt = np.zeros(r.shape[0])
    for t in range(r.shape[1] - 1, -1, -1):
        nxt = r[:, t] + gamma * keep[:, t] * nxt
        out[:, t] = nxt
    return {"output": out}


# ---------------------------------------------------------------------------------------- LIF
def leaky(inp):
    """tasks/leaky/reference.py:26-40: the fp32 loop, one rounding per product and sum."""
    x = _np(inp["input_current"]).astype(np.float32)
    T, B, H = x.shape
    beta = np.clip(_np(inp["beta"]).astype(np.float32), np.float32(0), np.float32(1)).reshape(1, H)
    th = _np(inp["threshold"]).astype(np.float32).reshape(1, H)
    mem = _np(inp["mem0"]).astype(np.float32).copy()
    spikes = np.empty_like(x)
    for t in range(T):
        reset = (mem >= th).astype(np.float32)
        mem = (beta * mem + x[t]) - reset * th
        spikes[t] = (mem >= th).astype(np.float32)
    return {"spikes": spikes, "final_mem": mem}


# ---------------------------------------------------------------------------------------- KAN
def kan_bases(x, grid, k_order):
    """Cox-de Boor bases; tasks/efficient_kan/reference.py:33-39 (indicator, then K rounds)."""
    xe = x[:, :, None]
    bases = ((xe >= grid[None, :, :-1]) & (xe < grid[None, :, 1:])).astype(x.dtype)
    for k in range(1, k_order + 1):
        left = (xe - grid[None, :, :-(k + 1)]) / (grid[None, :, k:-1] - grid[None, :, :-(k + 1)])
        right = (grid[None, :, k + 1:] - xe) / (grid[None, :, k + 1:] - grid[None, :, 1:-k])
        bases = left * bases[:, :, :-1] + right * bases[:, :, 1:]
    return bases


def efficient_kan(inp, rows=None):
    """tasks/efficient_kan/reference.py:42-46,54-57 in fp64.  `rows` limits the batch rows."""
    x = _np(inp["x"]).astype(np.float64)
    if rows is not None:
        x = x[rows]
    grid = _np(inp["grid"]).astype(np.float64)
    wb = _np(inp["base_weight"]).astype(np.float64)
    sw = _np(inp["spline_weight"]).astype(np.float64)
    sc = _np(inp["spline_scaler"]).astype(np.float64)
    bases = kan_bases(x, grid, int(inp["spline_order"]))
    silu = x / (1.0 + np.exp(-x))
    w = (sw * sc[:, :, None]).reshape(wb.shape[0], -1)
    out = silu @ wb.T + bases.reshape(x.shape[0], -1) @ w.T
    return {"out": out}


# ---------------------------------------------------------------------------------- FP8 linear
def e4m3_table():
    """Value of every E4M3 (fn variant) byte: 1 sign, 4 exponent (bias 7), 3 mantissa bits;
    exponent 0 is subnormal, S.1111.111 is NaN, no infinities."""
    vals = np.empty(256, dtype=np.float64)
    for b in range(256):
        s = -1.0 if b & 0x80 else 1.0
        e = (b >> 3) & 0xF
        m = b & 0x7
        if e == 0xF and m == 0x7:
            vals[b] = np.nan
        elif e == 0:
            vals[b] = s * (m / 8.0) * 2.0 ** -6
        else:
            vals[b] = s * (1.0 + m / 8.0) * 2.0 ** (e - 7)
    return vals


def f32_to_bf16_bits(v32):
    """Round fp32 values to bf16 (round to nearest, ties to even); returns uint16 bits."""
    u = np.ascontiguousarray(v32, dtype=np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(v32)
    rounded = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    out = rounded.astype(np.uint16)
    out[nan] = 0x7FC0
    return out


def bf16_bits_to_f64(b):
    return (np.asarray(b, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def fp8_linear(inp, rows=None):
    """tasks/fp8_linear/reference.py:34-37,44-45: (q_x/sx) @ (q_w/sw)^T + bias in fp64, then one
    conversion to bf16.  The conversion goes through fp32 (fp64 -> fp32 -> bf16, each round to
    nearest even), which is how the reference's `.to(torch.bfloat16)` of an fp64 tensor rounds.
    Returns bf16 bits (uint16) and the fp64 values before rounding."""
    tab = e4m3_table()
    xq = _np(inp["x_fp8"]).astype(np.uint8)
    if rows is not None:
        xq = xq[rows]
    x = tab[xq]
    x /= float(inp["scale_x"])
    w = tab[_np(inp["w_fp8"]).astype(np.uint8)]
    w /= float(inp["scale_w"])
    bias = bf16_bits_to_f64(_np(inp["bias"]))
    y = x @ w.T
    del w
    y += bias[None, :]
    return {"output": f32_to_bf16_bits(y.astype(np.float32)), "output_f64": y}


TASKS = {
    "pow_abs_sqrt_mean": pow_abs_sqrt_mean,
    "ppo_clip": ppo_clip,
    "reward_to_go": reward_to_go,
    "leaky": leaky,
    "efficient_kan": efficient_kan,
    "fp8_linear": fp8_linear,
}


def within(out, ref, atol, rtol):
    """Reference pass rule per element: |o - r| <= atol + rtol*|r|, NaN matches NaN
    (graders/child.py:150-175).  Returns (number of bad elements, worst |o-r|/(atol+rtol|r|))."""
    o = np.asarray(out, dtype=np.float64)
    r = np.asarray(ref, dtype=np.float64)
    both_nan = np.isnan(o) & np.isnan(r)
    err = np.abs(o - r)
    lim = atol + rtol * np.abs(r)
    ok = (err <= lim) | both_nan
    ratio = np.where(both_nan, 0.0, err / lim)
    worst = float(np.nanmax(ratio)) if ratio.size else 0.0
    return int((~ok).sum()), worst


def gae(inp):
    """Generalised advantage estimation in fp64 (no reference implementation in the reference
    repository: the published algorithm of Schulman et al. 2016 in the form of TorchRL's
    generalized_advantage_estimate, with separate done and terminated flags):
    delta = r + gamma * next_value * (1 - terminated) - value; A[t] = delta[t] + gamma * lambda *
    (1 - done[t]) * A[t + 1], A past the last step 0; value_target = A + value.  gamma and lambda
    are taken as the fp32 values the kernel receives."""
    r = _np(inp["reward"]).astype(np.float64)
    v = _np(inp["value"]).astype(np.float64)
    nv = _np(inp["next_value"]).astype(np.float64)
    done = _np(inp["done"]).astype(bool)
    term = _np(inp["terminated"]).astype(bool)
    g = float(np.float32(inp["gamma"]))
    lam = float(np.float32(inp["lmbda"]))
    delta = r + g * nv * (~term) - v
    adv = np.zeros_like(delta)
    a = np.zeros(delta.shape[0])
    for t in range(delta.shape[1] - 1, -1, -1):
        a = delta[:, t] + g * lam * (~done[:, t]) * a
        adv[:, t] = a
    return {"advantage": adv, "value_target": adv + v}


def atan_surrogate_grad(u, alpha):
    """Derivative of the arctangent spike surrogate (Fang et al., "Incorporating Learnable
    Membrane Time Constant to Enhance Learning of Spiking Neural Networks", 2021; snnTorch's
    default surrogate for Leaky): d spike / d u = (alpha / 2) / (1 + (pi / 2 * alpha * u)^2)."""
    return (alpha / 2.0) / (1.0 + (math.pi / 2.0 * alpha * u) ** 2)


def leaky_backward(inp, grad_spikes, grad_final_mem=None, alpha=2.0):
    """Surrogate-gradient backward of the leaky layer (no reference implementation in the reference
    repository: snnTorch's Leaky, the layer tasks/leaky restates, trained through its arctangent
    surrogate with the reset detached).  The forward is the reference's own fp32 loop
    (tasks/leaky/reference.py:26-40, `leaky` above), so every reset and spike decision is the
    reference's; the backward is then fp64 over those fp32 membrane values:

        u[t] = mem[t] - th,   s'[t] = atan_surrogate_grad(u[t]),   r[t] = (mem[t-1] >= th)
        g[t] = grad_spikes[t] * s'[t] + beta * g[t+1]         (beta * g[T] := grad_final_mem)
        grad_x[t] = g[t];   grad_mem0 = beta * g[0]
        grad_beta[h] = [0 <= beta_raw[h] <= 1] * sum_{b,t} g[t] * mem[t-1]
        grad_threshold[h] = -sum_{b,t} (grad_spikes[t] * s'[t] + r[t] * g[t])

    with mem[-1] = mem0 and beta the clamped value the forward uses."""
    x = _np(inp["input_current"]).astype(np.float32)
    T, B, H = x.shape
    braw = _np(inp["beta"]).astype(np.float32)
    beta32 = np.clip(braw, np.float32(0), np.float32(1)).reshape(1, H)
    th32 = _np(inp["threshold"]).astype(np.float32).reshape(1, H)
    mem = _np(inp["mem0"]).astype(np.float32).copy()
    mems = np.empty((T + 1, B, H), dtype=np.float32)
    mems[0] = mem
    for t in range(T):
        reset = (mem >= th32).astype(np.float32)
        mem = (beta32 * mem + x[t]) - reset * th32
        mems[t + 1] = mem
    gs = _np(grad_spikes).astype(np.float64).reshape(T, B, H)
    c = (np.zeros((B, H)) if grad_final_mem is None
         else _np(grad_final_mem).astype(np.float64).reshape(B, H))
    beta = beta32.astype(np.float64)
    th = th32.astype(np.float64)
    gx = np.empty((T, B, H))
    gb = np.zeros((B, H))
    gt = np.zeros((B, H))
    gb_abs = np.zeros((B, H))
    gt_abs = np.zeros((B, H))
    for t in range(T - 1, -1, -1):
        gsp = gs[t] * atan_surrogate_grad(mems[t + 1].astype(np.float64) - th, alpha)
        g = gsp + c
        gx[t] = g
        prev = mems[t].astype(np.float64)
        gb += g * prev
        gb_abs += np.abs(g * prev)
        term = gsp + (prev >= th) * g
        gt -= term
        gt_abs += np.abs(term)
        c = beta * g
    mask = ((braw >= 0) & (braw <= 1)).astype(np.float64)
    # *_abs: the sums of the terms' magnitudes, the scale of a summation's rounding error.
    return {"grad_input": gx, "grad_mem0": c, "grad_beta": mask * gb.sum(axis=0),
            "grad_threshold": gt.sum(axis=0), "grad_beta_abs": gb_abs.sum(axis=0),
            "grad_threshold_abs": gt_abs.sum(axis=0), "spikes": (mems[1:] >= th32).astype(np.float32),
            "final_mem": mems[T], "checkpoints": mems[0:T:16]}


def pack_done_bits(done):
    """Done flags [B, T] -> uint32 words [B, ceil(T/32)]: bit t % 32 of word [b, t // 32] is
    done[b, t], bits past T zero (the bit layout beside the reference's one-bool-per-step ABI)."""
    d = _np(done).astype(bool)
    B, T = d.shape
    W = (T + 31) // 32
    padded = np.zeros((B, W * 32), dtype=np.uint64)
    padded[:, :T] = d
    weights = np.left_shift(np.uint64(1), np.arange(32, dtype=np.uint64))
    return (padded.reshape(B, W, 32) * weights).sum(axis=2).astype(np.uint32)


def efficient_kan_backward(inp, grad_out, rows=None):
    """Backward of the KAN layer in fp64 (no reference implementation in the reference repository:
    the gradients of tasks/efficient_kan/reference.py:33-46, the KANLinear forward, that torch
    autograd forms through it).  With W_spl = spline_weight * spline_scaler and the bases B_c(x)
    and their derivatives from forward-mode differentiation of the same Cox-de Boor recurrence:

        grad_x[b,i]      = silu'(x) * (G @ W_base)[b,i] + sum_c B'_c(x[b,i]) * (G @ W_spl)[b,i,c]
        grad_W_base      = G^T @ silu(x)
        grad_W_spl       = G^T @ B(x)                       ([O, I, C])
        grad_sw          = grad_W_spl * spline_scaler;  grad_scaler = sum_c grad_W_spl * sw

    `rows` limits grad_x to a subset of batch rows (the weight gradients always use every row).
    *_abs: the same sums over the terms' magnitudes (the scale of a summation's rounding error)."""
    x = _np(inp["x"]).astype(np.float64)
    g = _np(inp["grid"]).astype(np.float64)
    wb = _np(inp["base_weight"]).astype(np.float64)
    sw = _np(inp["spline_weight"]).astype(np.float64)
    sc = _np(inp["spline_scaler"]).astype(np.float64)
    G = _np(grad_out).astype(np.float64)
    K = int(inp["spline_order"])
    B, I = x.shape
    O = wb.shape[0]
    C = sw.shape[2]
    xe = x[:, :, None]
    bases = ((xe >= g[None, :, :-1]) & (xe < g[None, :, 1:])).astype(np.float64)
    dbases = np.zeros_like(bases)
    for k in range(1, K + 1):
        dl = 1.0 / (g[None, :, k:-1] - g[None, :, :-(k + 1)])
        dr = -1.0 / (g[None, :, k + 1:] - g[None, :, 1:-k])
        left = (xe - g[None, :, :-(k + 1)]) * dl
        right = (g[None, :, k + 1:] - xe) * -dr
        nb = left * bases[:, :, :-1] + right * bases[:, :, 1:]
        dbases = dl * bases[:, :, :-1] + left * dbases[:, :, :-1] + dr * bases[:, :, 1:] + right * dbases[:, :, 1:]
        bases = nb
    s = 1.0 / (1.0 + np.exp(-x))
    silu = x * s
    dsilu = s * (1.0 + x * (1.0 - s))
    wspl = (sw * sc[:, :, None]).reshape(O, I * C)
    xr = slice(None) if rows is None else rows
    Gr = G[xr]
    ga_base = Gr @ wb
    ga_spl = (Gr @ wspl).reshape(-1, I, C)
    ga_base_abs = np.abs(Gr) @ np.abs(wb)
    ga_spl_abs = (np.abs(Gr) @ np.abs(wspl)).reshape(-1, I, C)
    grad_x = ga_base * dsilu[xr] + (ga_spl * dbases[xr]).sum(axis=2)
    grad_x_abs = ga_base_abs * np.abs(dsilu[xr]) + (ga_spl_abs * np.abs(dbases[xr])).sum(axis=2)
    gw_base = G.T @ silu
    gw_base_abs = np.abs(G).T @ np.abs(silu)
    bflat = bases.reshape(B, I * C)
    gw_spl = (G.T @ bflat).reshape(O, I, C)
    gw_spl_abs = (np.abs(G).T @ np.abs(bflat)).reshape(O, I, C)  # bases can be negative on unordered knots
    return {"grad_x": grad_x, "grad_base_weight": gw_base, "grad_spline_weight": gw_spl * sc[:, :, None],
            "grad_spline_scaler": (gw_spl * sw).sum(axis=2),
            "grad_x_abs": grad_x_abs, "grad_base_weight_abs": gw_base_abs,
            "grad_spline_weight_abs": gw_spl_abs * np.abs(sc[:, :, None]),
            "grad_spline_scaler_abs": (gw_spl_abs * np.abs(sw)).sum(axis=2)}


# ------------------------------------------------------------------- gated linear recurrence
def _f64(t):
    if hasattr(t, "detach"):
        t = t.detach().cpu()
        return t.numpy() if str(t.dtype) == "torch.bool" else t.double().numpy()
    t = np.asarray(t)
    return t if t.dtype == bool else t.astype(np.float64)


U32 = 2.0 ** -24  # half a step of fp32, relative


def linear_recurrence(gate, x, state=None, reset=None, form="decay", grad_h=None, grad_final=None):
    """The gated linear recurrence in fp64, step by step: h[t] = a h[t-1] + v (decay: a = gate, v = x;
    sigmoid: a = s(gate), v = (1 - a) x; reset drops h[t-1]) and, with grad_h, its gradients.  Returns
    (values, errors): errors[k] bounds the error of values[k] when every step is done in fp32, in any
    association of the scan.

    The bound: a step's result carries the error of the state it starts from, times |a|, and at most 16
    roundings relative to M, the recurrence of the absolute values (a sigmoid: exp 4, its argument's
    scaling 2, sum, reciprocal and product 4; a map's composition 2, the final fma 1, the step's own
    products 3).  A sigmoid below 2^-125 may be off by that much (the smallest normal fp32 value is 2^-126, and
    what lies below it may be flushed to 0), and so may 1 - a.  The backward's recurrence is bounded the
    same way."""
    low = 2.0 ** -125 if form == "sigmoid" else 0.0
    gate, x = _f64(gate), _f64(x)
    B, T, H = x.shape
    keep = np.ones((B, T, 1)) if reset is None else 1.0 - _f64(reset).astype(np.float64)[:, :, None]
    live = keep > 0
    if form == "decay":
        a, na, v = gate, np.ones_like(gate), x
    else:
        e = np.exp(-np.abs(gate))
        a = np.where(gate >= 0, 1.0, e) / (1.0 + e)
        na = np.where(gate >= 0, e, 1.0) / (1.0 + e)
        v = na * x
    cur = np.zeros((B, H)) if state is None else _f64(state).copy()
    mag, err = np.abs(cur), np.zeros((B, H))
    h, prev, eh, eprev = (np.empty_like(x) for _ in range(4))
    for t in range(T):
        prev[:, t] = np.where(live[:, t], cur, 0.0)
        eprev[:, t] = err * keep[:, t]
        cur = a[:, t] * prev[:, t] + v[:, t]
        mag = np.abs(a[:, t]) * np.where(live[:, t], mag, 0.0) + np.abs(v[:, t])
        err = np.abs(a[:, t]) * eprev[:, t] + 16 * U32 * mag + low * (np.abs(prev[:, t]) + np.abs(x[:, t]))
        h[:, t], eh[:, t] = cur, err
    val = {"h": h, "final": cur.copy()}
    bound = {"h": eh, "final": err.copy()}
    if grad_h is None:
        return val, bound
    dh = _f64(grad_h)
    acc = np.zeros((B, H)) if grad_final is None else _f64(grad_final).copy()
    mag, err = np.abs(acc), np.zeros((B, H))
    gg, gx, egg, egx = (np.empty_like(x) for _ in range(4))
    for t in range(T - 1, -1, -1):
        g = dh[:, t] + acc
        mag = mag + np.abs(dh[:, t])
        err = err + 16 * U32 * mag
        if form == "decay":
            gg[:, t] = g * prev[:, t]
            egg[:, t] = err * np.abs(prev[:, t]) + np.abs(g) * eprev[:, t] + 4 * U32 * np.abs(gg[:, t])
        else:
            d, s = prev[:, t] - x[:, t], a[:, t] * na[:, t]
            gg[:, t] = g * d * s
            egg[:, t] = (err * np.abs(d) + np.abs(g) * (eprev[:, t] + U32 * np.abs(d)) + 24 * U32 * np.abs(g * d)) * s + low * np.abs(g * d)
        gx[:, t] = na[:, t] * g
        egx[:, t] = na[:, t] * (err + 16 * U32 * np.abs(g)) + low * np.abs(g)
        acc = a[:, t] * g * keep[:, t]
        mag = np.abs(a[:, t]) * mag * keep[:, t]
        err = np.abs(a[:, t]) * err * keep[:, t] + 16 * U32 * mag + low * np.abs(g)
    val.update(grad_gate=gg, grad_x=gx, grad_state=acc)
    bound.update(grad_gate=egg, grad_x=egx, grad_state=err)
    return val, bound


# ------------------------------------------------------------------------- token log-probs
def token_logprob(logits, token, temperature=1.0, grad_log_prob=None, grad_entropy=None):
    """log softmax(logits / temperature)[token] and the entropy in fp64 (0 where token < 0), with the gradient
    of the logits where gradients are given.  Returns (values, errors) as linear_recurrence.

    The bound: exp has a relative error of 4 u and its argument d one of 3 u |d| (difference, scaling by a
    rounded 1 / temperature).  A sum of V terms is taken in at least 128 interleaved chains (a warp, two sets of
    pairs) that meet in a tree: ceil(V / 128) + 16 roundings, so K = ceil(V / 128) + 32 roundings cover log S
    and p beside the |d| part."""
    x, tok = _f64(logits), np.asarray(token.cpu() if hasattr(token, "cpu") else token)
    V = x.shape[-1]
    K = -(-V // 128) + 32
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = (x - x.max(-1, keepdims=True)) / temperature
        e = np.exp(d)
        log_s = np.log(e.sum(-1, keepdims=True))
        logp = d - log_s
        p = np.exp(logp)
        plogp = np.where(p > 0, p * logp, 0.0)
        pd = np.where(p > 0, p * np.abs(d), 0.0).sum(-1)
    ent = -plogp.sum(-1)
    on = tok >= 0
    at = np.clip(tok, 0, V - 1)
    lp = np.take_along_axis(logp, at[..., None], -1)[..., 0]
    dt = np.abs(np.take_along_axis(d, at[..., None], -1)[..., 0])
    base = K * U32 * (1 + np.abs(log_s[..., 0])) + 4 * U32 * pd
    val = {"log_prob": np.where(on, lp, 0.0), "entropy": np.where(on, ent, 0.0)}
    bound = {"log_prob": np.where(np.isfinite(dt), base + 4 * U32 * dt, 0.0) * on,
             "entropy": (base * (1 + pd) + K * U32 * pd) * on}
    if grad_log_prob is None:
        return val, bound
    gl = _f64(grad_log_prob)[..., None]
    ge = np.zeros_like(gl) if grad_entropy is None else _f64(grad_entropy)[..., None]
    hot = np.zeros_like(x)
    np.put_along_axis(hot, at[..., None], 1.0, -1)
    with np.errstate(invalid="ignore"):
        pl = np.where(p > 0, p * (logp + ent[..., None]), 0.0)
        g = (gl * (hot - p) - ge * pl) / temperature
        rel = K * U32 + base[..., None] + 4 * U32 * np.where(p > 0, np.abs(d), 0.0)
        size = np.abs(gl) * p + np.abs(ge) * p * (np.where(p > 0, np.abs(logp), 0.0) + np.abs(ent[..., None]))
        eg = (size * rel + np.abs(ge) * p * (bound["entropy"][..., None] + base[..., None]) +
              4 * U32 * np.abs(gl) * hot) / temperature
    val["grad_logits"] = np.where(on[..., None], g, 0.0)
    bound["grad_logits"] = np.where(on[..., None], eg, 0.0)
    return val, bound


# ------------------------------------------------------------------- policy and preference losses
def policy_loss(log_prob, old_log_prob, advantage, mask=None, ref_log_prob=None, entropy=None, clip_low=0.2,
                clip_high=0.2, dual_clip=None, kl_coef=0.0, kl_form="k3", entropy_coef=0.0, reduction="token_mean",
                scale=1.0):
    """The clipped policy loss with KL and entropy terms and its gradients in fp64.  Returns (values, errors).

    The bound: a token's terms (ratio, KL, gradient) carry at most 16 roundings of fp32 relative to their
    sizes (exp of a rounded difference: 4 + |d|), sums are in fp64, each output is rounded once."""
    cur, old, adv = _f64(log_prob), _f64(log_prob if old_log_prob is None else old_log_prob), _f64(advantage)
    adv = np.broadcast_to(adv if adv.ndim == 2 else adv[:, None], cur.shape)
    m = np.ones(cur.shape, bool) if mask is None else _f64(mask)
    cur, old, adv = (np.where(m, v, 0.0) for v in (cur, old, adv))
    d = cur - old
    r = np.exp(d)
    held = np.clip(r, 1.0 - clip_low, 1.0 + clip_high)
    gain = np.minimum(r * adv, held * adv)
    free = r * adv <= held * adv
    if dual_clip is not None:
        cut = (adv < 0) & (gain < dual_clip * adv)
        gain, free = np.where(cut, dual_clip * adv, gain), free & ~cut
    n_row = m.sum(1)
    n = max(1, int(m.sum()))
    if reduction == "token_mean":
        w = np.full(cur.shape, scale / n)
    elif reduction == "sequence_mean":
        w = np.broadcast_to((scale / (max(1, int((n_row > 0).sum())) * np.maximum(1, n_row)))[:, None], cur.shape)
    else:
        w = np.full(cur.shape, float(scale))
    w = np.where(m, w, 0.0)
    slope = np.where(free, -r * adv, 0.0)
    size = np.abs(slope) * (1 + np.abs(d))
    kl, kabs, ent, eabs = 0.0, 0.0, 0.0, 0.0
    if ref_log_prob is not None:
        q = np.where(m, _f64(ref_log_prob), 0.0) - cur
        k, dk = {"k1": (-q, np.ones_like(q)), "k2": (0.5 * q * q, -q),
                 "k3": (np.expm1(q) - q, -np.expm1(q))}[kl_form]
        kl, kabs = (w * k).sum(), (np.abs(w * k) * (1 + np.abs(q))).sum()
        slope = slope + kl_coef * dk
        size = size + np.abs(kl_coef) * np.abs(dk) * (1 + np.abs(q))
    if entropy is not None:
        h = np.where(m, _f64(entropy), 0.0)
        ent, eabs = (w * h).sum(), np.abs(w * h).sum()
    pol, pabs = -(w * gain).sum(), (np.abs(w * gain) * (1 + np.abs(d))).sum()
    out = np.array([pol + kl_coef * kl - entropy_coef * ent, pol, kl, ent, ((held != r) & m).sum() / n,
                    np.where(m, np.expm1(d) - d, 0.0).sum() / n, np.where(m, r, 0.0).max(initial=0.0),
                    np.where(m, r, 0.0).sum() / n])
    size_out = np.array([pabs + abs(kl_coef) * kabs + abs(entropy_coef) * eabs, pabs, kabs, eabs, out[4],
                         out[5] * (1 + np.abs(d).max(initial=0.0)), out[6] * (1 + np.abs(d).max(initial=0.0)),
                         out[7] * (1 + np.abs(d).max(initial=0.0))])
    val = {"out": out, "grad": w * slope, "grad_entropy": -w * entropy_coef}
    bound = {"out": 16 * U32 * size_out, "grad": 16 * U32 * np.abs(w) * size,
             "grad_entropy": 4 * U32 * np.abs(w * entropy_coef)}
    return val, bound


def preference_loss(chosen, rejected, ref_chosen=None, ref_rejected=None, chosen_mask=None, rejected_mask=None,
                    beta=0.1, form="sigmoid", label_smoothing=0.0, margin=0.0, average=False):
    """The preference loss and its gradients in fp64.  Returns (values, errors): everything up to the outputs
    is in fp64 in the kernel too, so 4 roundings of fp32 cover each output."""
    def side(lp, ref, mask):
        lp = _f64(lp)
        m = np.ones(lp.shape, bool) if mask is None else _f64(mask)
        gap = np.where(m, lp, 0.0) - (0.0 if ref is None else np.where(m, _f64(ref), 0.0))
        n = np.maximum(1, m.sum(1)) if average else np.ones(lp.shape[0])
        return gap.sum(1) / n, m / n[:, None], np.abs(gap).sum(1) / n
    (c, mc, ac), (r, mr, ar) = side(chosen, ref_chosen, chosen_mask), side(rejected, ref_rejected, rejected_mask)
    B = max(1, len(c))
    gap = beta * (c - r)
    z = gap - margin
    if form == "sigmoid":
        loss = (1 - label_smoothing) * np.logaddexp(0, -z) + label_smoothing * np.logaddexp(0, z)
        dz = label_smoothing - np.exp(-np.logaddexp(0, z))
    elif form == "hinge":
        loss, dz = np.maximum(0.0, 1 - z), np.where(z < 1, -1.0, 0.0)
    else:
        loss, dz = ((z - 0.5) / beta) ** 2, 2 * (z - 0.5) / beta ** 2
    k = (beta * dz / B)[:, None]
    val = {"out": np.array([loss.sum(), (c > r).sum(), gap.sum()]) / B, "reward_chosen": beta * c,
           "reward_rejected": beta * r, "grad_chosen": k * mc, "grad_rejected": -k * mr}
    # fp64 sums are off by up to 2^-40 of their terms' sizes, which the losses' slopes carry on.
    lost = 2.0 ** -40 * beta * (ac + ar)
    bound = {n: 4 * U32 * np.abs(v) for n, v in val.items()}
    bound["out"] = bound["out"] + np.array([(np.abs(dz) * lost).sum(), 0.0, lost.sum()]) / B
    bound["reward_chosen"] = bound["reward_chosen"] + lost
    bound["reward_rejected"] = bound["reward_rejected"] + lost
    curve = {"sigmoid": 0.25, "hinge": 0.0, "ipo": 2 / beta ** 2}[form]
    slip = (beta * curve * lost / B)[:, None]
    bound["grad_chosen"] = bound["grad_chosen"] + slip * mc
    bound["grad_rejected"] = bound["grad_rejected"] + slip * mr
    return val, bound
