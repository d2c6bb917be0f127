"""The clipped policy loss with KL and entropy terms, and its gradients.

The oracle (oracle.exact.policy_loss) is fp64; on the CPU its gradients are checked against differences.
GPU: reductions, KL forms, masks with empty rows and non-finite values behind them, strides, ratios on the
borders, broadcast advantages, repeats, captures.
"""
import math

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import exact
from sequence_policy import captured, load_ops, near, same_bits


@pytest.fixture(scope="module")
def ops():
    return load_ops()


def make(B, T, seed, ref=True, ent=True, rows=False, mask=0.7, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    cur = -(torch.randn(B, T, generator=g) * 0.5 - 1).abs()
    s = {"log_prob": cur, "old_log_prob": cur + 0.25 * torch.randn(B, T, generator=g),
         "advantage": torch.randn(*((B,) if rows else (B, T)), generator=g),
         "mask": torch.rand(B, T, generator=g) < mask if mask is not None else None,
         "ref_log_prob": cur + 0.3 * torch.randn(B, T, generator=g) if ref else None,
         "entropy": 2 * torch.rand(B, T, generator=g) if ent else None}
    if s["mask"] is not None and B > 2:
        s["mask"][B // 2] = False
    return {k: v.to(device) if v is not None else None for k, v in s.items()}


FULL = dict(clip_low=0.2, clip_high=0.28, kl_coef=0.07, entropy_coef=0.02, scale=0.5)


def check(ops, s, **o):
    out, grad, ge = ops.policy_loss_grad(**s, **o)
    alone = ops.policy_loss(**s, **o)
    torch.cuda.synchronize()
    assert same_bits(out, alone)
    want, err = exact.policy_loss(**s, **o)
    near(out, want["out"], err["out"], "outputs")
    near(grad, want["grad"], err["grad"], "grad")
    if s["entropy"] is not None:
        near(ge, want["grad_entropy"], err["grad_entropy"], "grad_entropy")
    else:
        assert ge is None
    if s["mask"] is not None:
        assert not grad[~s["mask"]].any()
    return out, grad


# --------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
@pytest.mark.parametrize("kl_form", ["k1", "k2", "k3"])
@pytest.mark.parametrize("dual", [None, 1.5])
def test_oracle_gradients_against_differences(reduction, kl_form, dual):
    s = {k: None if v is None else v.numpy().astype(bool if v.dtype == torch.bool else np.float64)
         for k, v in make(3, 5, seed=1, device="cpu").items()}
    s["old_log_prob"] = s["log_prob"] + (s["old_log_prob"] - s["log_prob"]) * 3
    o = dict(FULL, reduction=reduction, kl_form=kl_form, dual_clip=dual)
    want = exact.policy_loss(**s, **o)[0]
    for name, g in (("log_prob", "grad"), ("entropy", "grad_entropy")):
        for at in np.ndindex(3, 5):
            up, dn = dict(s), dict(s)
            up[name], dn[name] = s[name].copy(), s[name].copy()
            up[name][at] += 1e-6
            dn[name][at] -= 1e-6
            d = (exact.policy_loss(**up, **o)[0]["out"][0] - exact.policy_loss(**dn, **o)[0]["out"][0]) / 2e-6
            assert abs(d - want[g][at]) < 1e-8, (name, at)


def test_refusals_on_the_cpu():
    ops = pkg().ops
    x = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="CUDA"):
        ops.policy_loss(x, x, x)
    lib = pkg().load()
    st = (pkg()._native.c_i64 * 7)(3, 3, 3, 1, 0, 0, 0)
    P = 4096  # never dereferenced: each call is refused before any CUDA call

    def call(B=2, T=3, low=0.2, high=0.2, dual=0.0, form=2, red=0, cur=P, out=P, strides=st, ge=None, ws=P,
             size=1 << 30):
        return lib.b200_policy_loss_async(cur, P, P, None, None, None, strides, B, T, low, high, dual, 0.0, form, 0.0,
                                          red, 1.0, out, None, ge, ws, size, None)

    for bad in (dict(B=-1), dict(T=-1), dict(low=1.0), dict(low=-0.1), dict(high=-0.1), dict(high=float("nan")),
                dict(dual=0.5), dict(form=3), dict(red=-1), dict(red=3), dict(cur=None), dict(out=None),
                dict(strides=None), dict(ge=P), dict(strides=(pkg()._native.c_i64 * 7)(3, 3, 3, 2, 0, 0, 0))):
        assert call(**bad) == 1, bad
    need = lib.b200_policy_loss_workspace_bytes(100, 3000)  # (few tokens need none)
    assert call(B=100, T=3000, ws=None) == 4 and call(B=100, T=3000, size=need - 1) == 4
    assert lib.b200_policy_loss_workspace_bytes(-1, 3) == -1


# --------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("B,T", [(1, 1), (1, 3), (3, 1), (4, 33), (5, 257), (2, 4096), (1, 50_001), (300, 20), (64, 1000)])
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
def test_against_oracle(ops, B, T, reduction):
    check(ops, make(B, T, seed=B * 31 + T), reduction=reduction, **FULL)


@pytest.mark.gpu
@pytest.mark.parametrize("kl_form", ["k1", "k2", "k3"])
@pytest.mark.parametrize("dual", [None, 1.3])
@pytest.mark.parametrize("rows", [False, True])
def test_forms(ops, kl_form, dual, rows):
    check(ops, make(7, 300, seed=3, rows=rows), kl_form=kl_form, dual_clip=dual, **FULL)


@pytest.mark.gpu
@pytest.mark.parametrize("ref", [False, True])
@pytest.mark.parametrize("ent", [False, True])
@pytest.mark.parametrize("mask", [None, 0.5])
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
def test_optional_inputs(ops, ref, ent, mask, reduction):
    o = dict(FULL, kl_coef=FULL["kl_coef"] if ref else 0.0, entropy_coef=FULL["entropy_coef"] if ent else 0.0)
    check(ops, make(6, 131, seed=4, ref=ref, ent=ent, mask=mask), reduction=reduction, **o)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
def test_large(ops, reduction):
    """More tokens than the GPU holds at once, with lengths from none to all."""
    s = make(2000, 2300, seed=8, rows=True)
    n = torch.randint(0, 2301, (2000,), device="cuda")
    s["mask"] = torch.arange(2300, device="cuda") < n[:, None]
    check(ops, s, reduction=reduction, **FULL)


@pytest.mark.gpu
def test_on_policy(ops):
    """Without old log-probs the ratio is 1 and the gradient is the policy gradient."""
    s = make(4, 65, seed=2, ref=False, ent=False)
    s["old_log_prob"] = None
    out, grad = check(ops, s)
    assert out[4] == 0 and out[5] == 0 and out[6] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
@pytest.mark.parametrize("B,T", [(3, 40), (700, 3000)])
def test_nothing_left(ops, reduction, B, T):
    s = make(B, T, seed=6)
    s["mask"][:] = False
    s["log_prob"][:] = float("nan")
    out, grad, ge = ops.policy_loss_grad(**s, reduction=reduction, **FULL)
    torch.cuda.synchronize()
    assert not out.any() and not grad.any() and not ge.any()


@pytest.mark.gpu
@pytest.mark.parametrize("B,T", [(0, 4), (4, 0)])
def test_empty(ops, B, T):
    z = torch.zeros(B, T, device="cuda")
    out, grad, ge = ops.policy_loss_grad(z, z, z, entropy=z)
    torch.cuda.synchronize()
    assert not out.any() and grad.shape == (B, T) and ge.shape == (B, T)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min])
def test_what_masked_tokens_hold_does_not_count(ops, bad):
    s = make(5, 200, seed=7)
    want = ops.policy_loss_grad(**s, reduction="sequence_mean", **FULL)
    for k in ("log_prob", "old_log_prob", "ref_log_prob", "entropy", "advantage"):
        s[k] = torch.where(s["mask"], s[k], torch.full_like(s[k], bad))
    got = ops.policy_loss_grad(**s, reduction="sequence_mean", **FULL)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_ratios_at_the_borders(ops):
    """Differences next to log(1 + clip_high), log(1 - clip_low) and log(dual): which side each falls on is
    decided as in exact arithmetic."""
    rng = np.random.default_rng(0)
    n = 4000
    old = (-np.abs(rng.normal(size=n) * 3)).astype(np.float32)
    edge = rng.choice([math.log1p(0.28), math.log1p(-0.2), math.log(3.0)], size=n)
    cur = (old.astype(np.float64) + edge).astype(np.float32)
    step = np.spacing(cur) * rng.integers(-2, 3, size=n).astype(np.float32)
    cur = (cur + step).astype(np.float32)
    s = {"log_prob": torch.from_numpy(cur)[None].cuda(), "old_log_prob": torch.from_numpy(old)[None].cuda(),
         "advantage": torch.from_numpy(rng.normal(size=n).astype(np.float32))[None].cuda(), "mask": None,
         "ref_log_prob": None, "entropy": None}
    d = cur.astype(np.float64) - old
    assert (np.abs(d - edge) < 1e-6).mean() > 0.9
    check(ops, s, clip_low=0.2, clip_high=0.28, dual_clip=3.0, reduction="sum")


@pytest.mark.gpu
def test_far_ratios(ops):
    """Ratios that overflow fp32: clipped ones stay finite, zero advantages give zero."""
    s = {"log_prob": torch.tensor([[100.0, 100.0, -200.0, -200.0, 100.0]], device="cuda"),
         "old_log_prob": torch.zeros(1, 5, device="cuda"),
         "advantage": torch.tensor([[1.0, -1.0, 1.0, -1.0, 0.0]], device="cuda"), "mask": None, "ref_log_prob": None,
         "entropy": None}
    out, grad, _ = ops.policy_loss_grad(**s, dual_clip=2.0, reduction="sum")
    torch.cuda.synchronize()
    assert not grad.any() and abs(float(out[0]) - (-1.2 + 2.0 + 0.8)) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("T", [61, 64, 1025])
def test_strided_rows(ops, T):
    """Answers cut out of longer rows, at odd offsets."""
    s = make(5, T, seed=T)
    cut = {}
    for i, (k, v) in enumerate(s.items()):
        wide = torch.zeros(5, T + 40 + i, dtype=v.dtype, device="cuda")
        cut[k] = wide[:, 3 * i + 1:3 * i + 1 + T]
        cut[k].copy_(v)
    check(ops, cut, **FULL)
    cut["advantage"] = s["advantage"][:, 0][:, None].expand(5, 8)[:, 0]
    check(ops, cut, **FULL)
    one = dict(s, ref_log_prob=s["ref_log_prob"][:1].expand(5, T))
    check(ops, one, **FULL)


@pytest.mark.gpu
def test_scratch_serves_other_sizes(ops):
    for k, (B, T) in enumerate([(500, 900), (2, 3), (3000, 1500), (1, 1), (70, 5000), (500, 900)]):
        check(ops, make(B, T, seed=k), reduction=["token_mean", "sequence_mean"][k % 2], **FULL)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T", [(8, 100), (900, 1100)])
def test_repeats_streams_and_captures(ops, B, T):
    sets = [make(B, T, seed=k) for k in (1, 2, 3)]
    calls = [lambda s=s: ops.policy_loss_grad(**s, reduction="sequence_mean", **FULL) for s in sets]
    want = [[t.clone() for t in c()] for c in calls]
    (ga, oa), (gb, ob) = captured(calls[0]), captured(calls[1])
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(6):
        torch.cuda.synchronize()
        for t in (*oa, *ob):
            t.fill_(5)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            ga.replay()
        with torch.cuda.stream(b):
            gb.replay()
        now = calls[2]()
        torch.cuda.synchronize()
        for got, w in ((oa, want[0]), (ob, want[1]), (now, want[2])):
            assert all(same_bits(x, y) for x, y in zip(got, w))


@pytest.mark.gpu
def test_threads_share_a_stream(ops):
    """Calls of several threads on one stream, of more than one launch each, do not mix."""
    import threading
    sets = [make(700, 900, seed=k) for k in range(4)]
    call = lambda s: ops.policy_loss_grad(**s, reduction="sequence_mean", **FULL)  # noqa: E731
    want = [[t.clone() for t in call(s)] for s in sets]
    got = [[] for _ in sets]

    def work(k):
        for _ in range(30):
            got[k].append(call(sets[k]))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(4):
        assert len(got[k]) == 30 and all(same_bits(a, b) for c in got[k] for a, b in zip(c, want[k]))


@pytest.mark.gpu
def test_row_strides_beyond_32_bits(ops):
    s = make(2, 3000, seed=12)
    gap = 2**31 + 4
    store = torch.empty(gap + 5 * 3000, device="cuda")
    for i, k in enumerate(("log_prob", "old_log_prob", "advantage", "ref_log_prob", "entropy")):
        v = store.as_strided((2, 3000), (gap, 1), i * 3000)
        v.copy_(s[k])
        s[k] = v
    check(ops, s, **FULL)


@pytest.mark.gpu
def test_autograd(ops):
    s = make(4, 50, seed=5)
    lp, ent = s["log_prob"].clone().requires_grad_(), s["entropy"].clone().requires_grad_()
    loss, out = ops.PolicyLossFunction.apply(lp, ent, s["old_log_prob"], s["advantage"], s["mask"], s["ref_log_prob"],
                                             dict(FULL, kl_form="k3"))
    (3.0 * loss).backward()
    want, err = exact.policy_loss(**s, **FULL)
    near(lp.grad, 3 * want["grad"], 4 * err["grad"] + 4 * exact.U32 * np.abs(want["grad"]))
    near(ent.grad, 3 * want["grad_entropy"], 4 * err["grad_entropy"] + 4 * exact.U32 * np.abs(want["grad_entropy"]))
    assert not out.requires_grad and float(out[0]) == float(loss)
    lp.grad = None
    ops.PolicyLossFunction.apply(lp, None, s["old_log_prob"], s["advantage"])[0].backward()
    want, err = exact.policy_loss(s["log_prob"], s["old_log_prob"], s["advantage"])
    near(lp.grad, want["grad"], err["grad"])


@pytest.mark.gpu
def test_refusals(ops):
    x, m = torch.zeros(2, 3, device="cuda"), torch.ones(2, 3, dtype=torch.bool, device="cuda")
    for bad in (lambda: ops.policy_loss(x.half(), x, x), lambda: ops.policy_loss(x, x[:, :2], x),
                lambda: ops.policy_loss(x, x, x[:, 0, None]), lambda: ops.policy_loss(x, x, x[0]),
                lambda: ops.policy_loss(x, x, x, mask=x), lambda: ops.policy_loss(x.t(), x.t(), x.t()),
                lambda: ops.policy_loss(x, x, x, kl_coef=0.1), lambda: ops.policy_loss(x, x, x, entropy_coef=0.1),
                lambda: ops.policy_loss(x, x, x, kl_form="k4"), lambda: ops.policy_loss(x, x, x, reduction="mean"),
                lambda: ops.policy_loss(x, x, x, clip_low=1.0), lambda: ops.policy_loss(x, x, x, clip_high=-1),
                lambda: ops.policy_loss(x, x, x, dual_clip=1.0),
                lambda: ops.policy_loss(x, x, x, scale=float("nan")), lambda: ops.policy_loss(x, x, x, m.cpu()),
                lambda: ops.PolicyLossFunction.apply(x, None, x, x.clone().requires_grad_()),
                lambda: ops.PolicyLossFunction.apply(x, None, x, x, None, None, {"clip": 0.2})):
        with pytest.raises((ValueError, TypeError)):
            bad()
