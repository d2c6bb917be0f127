"""The preference loss over pairs of answers, and its gradients.

The oracle (oracle.exact.preference_loss) is fp64; on the CPU its gradients are checked against differences.
GPU: forms, masks with empty answers, answers of different lengths (none among them), strides, one long pair, many short ones,
repeats, captures.
"""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import exact
from sequence_policy import captured, load_ops, near, same_bits


@pytest.fixture(scope="module")
def ops():
    return load_ops()


def make(B, Tc, Tr, seed, ref=True, mask=0.7, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    s = {}
    for k, T in (("chosen", Tc), ("rejected", Tr)):
        s[k] = -(torch.randn(B, T, generator=g) * 0.5 - 1).abs()
        s["ref_" + k] = s[k] + 0.1 * torch.randn(B, T, generator=g) if ref else None
        s[k + "_mask"] = torch.rand(B, T, generator=g) < mask if mask is not None else None
        if mask is not None and B > 2:
            s[k + "_mask"][B // 2 if k == "chosen" else 0] = False
    return {k: v.to(device) if v is not None else None for k, v in s.items()}


def check(ops, s, **o):
    got = ops.preference_loss_grad(**s, **o)
    alone = ops.preference_loss(**s, **o)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(alone, got))
    want, err = exact.preference_loss(**s, **o)
    for k, v in zip(("out", "reward_chosen", "reward_rejected", "grad_chosen", "grad_rejected"), got):
        near(v, want[k], err[k], k)
    return got


# --------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("form,e", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [False, True])
def test_oracle_gradients_against_differences(form, e, average):
    s = {k: v.numpy().astype(bool if v.dtype == torch.bool else np.float64)
         for k, v in make(3, 4, 5, seed=1, device="cpu").items()}
    o = dict(beta=0.5, form=form, label_smoothing=e, margin=0.1, average=average)
    want = exact.preference_loss(**s, **o)[0]
    for name in ("chosen", "rejected"):
        for at in np.ndindex(s[name].shape):
            up, dn = dict(s), dict(s)
            up[name], dn[name] = s[name].copy(), s[name].copy()
            up[name][at] += 1e-6
            dn[name][at] -= 1e-6
            d = (exact.preference_loss(**up, **o)[0]["out"][0] - exact.preference_loss(**dn, **o)[0]["out"][0]) / 2e-6
            assert abs(d - want["grad_" + name][at]) < 1e-8, (name, at)


def test_refusals_on_the_cpu():
    ops = pkg().ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.preference_loss(torch.zeros(2, 3), torch.zeros(2, 3))
    lib = pkg().load()
    st = (pkg()._native.c_i64 * 6)(3, 3, 3, 3, 3, 3)
    P = 4096  # never dereferenced: each call is refused before any CUDA call

    def call(B=2, Tc=3, beta=0.1, form=0, e=0.0, c=P, rc=None, rr=None, out=P, w=P, ws=P, size=1 << 30, strides=st):
        return lib.b200_preference_loss_async(c, P, rc, rr, None, None, strides, B, Tc, 3, beta, form, e, 0.0, 0, out,
                                              w, P, None, None, ws, size, None)

    for bad in (dict(B=-1), dict(Tc=-1), dict(beta=0.0), dict(beta=float("nan")), dict(form=3), dict(e=0.6),
                dict(e=-0.1), dict(form=1, e=0.1), dict(c=None), dict(rc=P), dict(rr=P), dict(out=None), dict(w=None),
                dict(strides=None)):
        assert call(**bad) == 1, bad
    assert call(ws=None) == 4 and call(size=lib.b200_preference_loss_workspace_bytes(2) - 1) == 4
    assert lib.b200_preference_loss_workspace_bytes(-1) == -1


# --------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("B,Tc,Tr", [(1, 1, 1), (2, 3, 1), (4, 33, 70), (3, 257, 256), (5, 1000, 515), (1, 70_001, 300),
                                     (2, 20_000, 40_003), (600, 9, 12), (200, 700, 800)])
@pytest.mark.parametrize("form", ["sigmoid", "hinge", "ipo"])
def test_against_oracle(ops, B, Tc, Tr, form):
    check(ops, make(B, Tc, Tr, seed=B + Tc), form=form)


@pytest.mark.gpu
@pytest.mark.parametrize("form,e", [("sigmoid", 0.0), ("sigmoid", 0.3), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("ref", [False, True])
@pytest.mark.parametrize("mask", [None, 0.5])
def test_options(ops, form, e, average, ref, mask):
    check(ops, make(7, 120, 131, seed=5, ref=ref, mask=mask), beta=0.7, form=form, label_smoothing=e, margin=0.25,
          average=average)


@pytest.mark.gpu
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("Tc,Tr", [(0, 5), (5, 0), (0, 0), (40, 40)])
def test_answers_without_tokens(ops, average, Tc, Tr):
    s = make(3, Tc, Tr, seed=3)
    s["chosen_mask"][:] = False
    s["rejected_mask"][:] = False
    s["chosen"][:] = float("nan")
    out, rc, rr, gc, gr = ops.preference_loss_grad(**s, average=average)
    torch.cuda.synchronize()
    assert abs(float(out[0]) - np.log(2)) < 1e-6 and out[1] == 0 and out[2] == 0
    assert not rc.any() and not rr.any() and not gc.any() and not gr.any()


@pytest.mark.gpu
def test_no_pairs(ops):
    z = torch.zeros(0, 4, device="cuda")
    out, rc, rr, gc, gr = ops.preference_loss_grad(z, z)
    torch.cuda.synchronize()
    assert not out.any() and rc.shape == (0,) and gc.shape == (0, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min])
def test_what_masked_tokens_hold_does_not_count(ops, bad):
    s = make(4, 300, 211, seed=9)
    want = ops.preference_loss_grad(**s)
    for k in ("chosen", "rejected"):
        for n in (k, "ref_" + k):
            s[n] = torch.where(s[k + "_mask"], s[n], torch.full_like(s[n], bad))
    got = ops.preference_loss_grad(**s)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_far_margins(ops):
    """Margins at which exp overflows in fp32 and in fp64."""
    lp = torch.zeros(4, 2, device="cuda")
    c, r = lp.clone(), lp.clone()
    c[:, 0] = torch.tensor([-200.0, -2000.0, 300.0, 3000.0])
    for form in ("sigmoid", "hinge"):
        check(ops, {"chosen": c, "rejected": r, "ref_chosen": None, "ref_rejected": None, "chosen_mask": None,
                    "rejected_mask": None}, beta=1.0, form=form)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [64, 77, 4097])
def test_halves_of_one_batch_and_strided_rows(ops, T):
    s = make(3, T, T, seed=T)
    both = {k: torch.cat([s[a], s[b]]) for k, a, b in
            (("lp", "chosen", "rejected"), ("ref", "ref_chosen", "ref_rejected"), ("m", "chosen_mask", "rejected_mask"))}
    wide = {k: torch.zeros(6, T + 9, dtype=v.dtype, device="cuda") for k, v in both.items()}
    for i, (k, v) in enumerate(both.items()):
        wide[k][:, i + 1:i + 1 + T] = v
        both[k] = wide[k][:, i + 1:i + 1 + T]
    cut = {"chosen": both["lp"][:3], "rejected": both["lp"][3:], "ref_chosen": both["ref"][:3],
           "ref_rejected": both["ref"][3:], "chosen_mask": both["m"][:3], "rejected_mask": both["m"][3:]}
    a, b = check(ops, cut), check(ops, s)
    assert all(same_bits(x, y) for x, y in zip(a[3:], b[3:]))


@pytest.mark.gpu
def test_scratch_serves_other_sizes(ops):
    for k, (B, Tc, Tr) in enumerate([(300, 100, 90), (2, 30_000, 10), (900, 5, 6), (1, 1, 1), (300, 100, 90)]):
        check(ops, make(B, Tc, Tr, seed=k))


@pytest.mark.gpu
@pytest.mark.parametrize("B,T", [(3, 9000), (500, 400)])
def test_repeats_streams_and_captures(ops, B, T):
    sets = [make(B, T, T + 1, seed=k) for k in (1, 2, 3)]
    calls = [lambda s=s: ops.preference_loss_grad(**s) for s in sets]
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
def test_autograd(ops):
    s = make(4, 50, 60, seed=5)
    c, r = s["chosen"].clone().requires_grad_(), s["rejected"].clone().requires_grad_()
    loss, out, rc, rr = ops.PreferenceLossFunction.apply(c, r, s["ref_chosen"], s["ref_rejected"], s["chosen_mask"],
                                                         s["rejected_mask"], {"beta": 0.3})
    (2.0 * loss).backward()
    want, err = exact.preference_loss(**s, beta=0.3)
    for t, k in ((c, "grad_chosen"), (r, "grad_rejected")):
        near(t.grad, 2 * want[k], 2 * err[k] + 4 * exact.U32 * np.abs(want[k]))
    assert not rc.requires_grad and float(out[0]) == float(loss)


@pytest.mark.gpu
def test_refusals(ops):
    x, m = torch.zeros(2, 3, device="cuda"), torch.ones(2, 3, dtype=torch.bool, device="cuda")
    for bad in (lambda: ops.preference_loss(x.half(), x), lambda: ops.preference_loss(x, x[:1]),
                lambda: ops.preference_loss(x, x, x), lambda: ops.preference_loss(x, x, x, x[:, :2]),
                lambda: ops.preference_loss(x, x, chosen_mask=x), lambda: ops.preference_loss(x, x, chosen_mask=m[:, :2]),
                lambda: ops.preference_loss(x.t(), x.t()), lambda: ops.preference_loss(x, x, beta=0.0),
                lambda: ops.preference_loss(x, x, form="other"), lambda: ops.preference_loss(x, x, label_smoothing=0.7),
                lambda: ops.preference_loss(x, x, form="ipo", label_smoothing=0.1),
                lambda: ops.preference_loss(x, x, margin=float("inf")),
                lambda: ops.PreferenceLossFunction.apply(x, x, x.clone().requires_grad_(), x),
                lambda: ops.PreferenceLossFunction.apply(x, x, None, None, None, None, {"tau": 1})):
        with pytest.raises((ValueError, TypeError)):
            bad()
