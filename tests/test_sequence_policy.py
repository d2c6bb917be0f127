"""The sequence-policy operators run together, as a training step uses them: a recurrent layer, its head's
token log-probs, then the policy loss or the preference loss, and the gradients back to the projections.

The whole step is held against the same step in fp64 (torch autograd over elementary operations)."""
import pytest
import torch

from conftest import pkg
from sequence_policy import captured, load_ops, same_bits


@pytest.fixture(scope="module")
def ops():
    return load_ops()


def layer(x, w_in, state):
    """The recurrence in elementary operations, any dtype."""
    gate, v = (x @ w_in).chunk(2, -1)
    f = torch.sigmoid(gate)
    h, hs = state, []
    for t in range(x.shape[1]):
        h = f[:, t] * h + (1 - f[:, t]) * v[:, t]
        hs.append(h)
    return torch.stack(hs, 1)


def make(B, T, D, H, V, seed):
    g = torch.Generator().manual_seed(seed)
    return {"x": torch.randn(B, T, D, generator=g).cuda(), "w_in": (torch.randn(D, 2 * H, generator=g) / D ** 0.5).cuda(),
            "w_out": (torch.randn(H, V, generator=g) / H ** 0.5 * 2).cuda(), "state": torch.randn(B, H, generator=g).cuda(),
            "token": torch.randint(0, V, (B, T), generator=g).cuda(),
            "mask": (torch.rand(B, T, generator=g) < 0.8).cuda(), "adv": torch.randn(B, generator=g).cuda(),
            "noise": 0.2 * torch.randn(2, B, T, generator=g).cuda()}


OPTIONS = dict(clip_low=0.2, clip_high=0.2, kl_coef=0.1, kl_form="k3", entropy_coef=0.02, reduction="sequence_mean")


def plain_log_probs(s, w_in, w_out):
    logits = layer(s["x"].to(w_in.dtype), w_in, s["state"].to(w_in.dtype)) @ w_out
    logp = logits.log_softmax(-1)
    return logp.gather(-1, s["token"][..., None])[..., 0], -(logp.exp() * logp).sum(-1)


def own_log_probs(ops, s, w_in, w_out):
    gate, v = (s["x"] @ w_in).chunk(2, -1)
    h, _ = ops.LinearRecurrenceFunction.apply(gate, v, s["state"], None, "sigmoid")
    return ops.TokenLogProbFunction.apply(h @ w_out, s["token"], 1.0)


def leaves(s, dtype):
    return [s[k].to(dtype).clone().requires_grad_() for k in ("w_in", "w_out")]


def compare(got, want):
    """Gradients of an fp32 step against fp64.  The matrix products (K <= 256 terms in fp32) and the 200 steps of
    the recurrence each lose at most some hundred roundings of 2^-24: 2^-24 * 1000 relative to the
    largest gradient."""
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 1000 * 2.0 ** -24 * b.abs().max(), (a.double() - b).abs().max() / b.abs().max()


def test_calls_go_to_the_tensors_device(monkeypatch):
    """A call on tensors of another device than the current one makes that device current for the launch, and takes
    that device's stream (a stand-in for the devices: no GPU here)."""
    from conftest import pkg
    ops = pkg().ops
    current, seen = [0], []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", device)
    call = lambda *a: seen.append((current[0], a)) or 0  # noqa: E731
    ops._run("x", call, 1, 7)
    ops._run("x", call, 0, 8)
    assert seen == [(1, (7, 101)), (0, (8, 100))] and current == [0]


@pytest.fixture(autouse=True)
def full_precision_products():
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = before


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,V", [(3, 200, 211), (5, 37, 1000)])
def test_policy_step(ops, B, T, V):
    s = make(B, T, 48, 64, V, seed=B)
    w64 = leaves(s, torch.float64)
    lp64, ent64 = plain_log_probs(s, *w64)
    old, ref = (lp64.detach() + s["noise"][0]).float(), (lp64.detach() + s["noise"][1]).float()
    r = (lp64 - old).exp()
    adv = s["adv"].double()[:, None]
    gain = torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
    q = ref - lp64
    per = -gain + 0.1 * (q.exp() - q - 1) - 0.02 * ent64
    m = s["mask"].double()
    loss64 = ((per * m).sum(1) / m.sum(1)).mean()
    want = torch.autograd.grad(loss64, w64)

    w = leaves(s, torch.float32)
    lp, ent = own_log_probs(ops, s, *w)
    loss, out = ops.PolicyLossFunction.apply(lp, ent, old, s["adv"], s["mask"], ref, OPTIONS)
    got = torch.autograd.grad(loss, w)
    # a token whose ratio rounds across a border would change its gradient: none may sit that near
    d = (lp64 - old).detach()
    border = torch.tensor([0.8, 1.2], device="cuda", dtype=torch.float64).log()
    assert (d[..., None] - border).abs().min() > 1e-5
    assert abs(float(loss) - float(loss64)) <= 1000 * 2.0 ** -24 * float(per.abs().max())
    compare(got, want)


@pytest.mark.gpu
def test_preference_step(ops):
    s = make(6, 90, 48, 64, 300, seed=9)
    w64 = leaves(s, torch.float64)
    lp64, _ = plain_log_probs(s, *w64)
    ref = (lp64.detach() + s["noise"][0]).float()
    t = ((lp64 - ref) * s["mask"]).sum(1)
    loss64 = torch.nn.functional.softplus(-0.3 * (t[:3] - t[3:])).mean()
    want = torch.autograd.grad(loss64, w64)
    w = leaves(s, torch.float32)
    lp, _ = own_log_probs(ops, s, *w)
    m = s["mask"]
    loss = ops.PreferenceLossFunction.apply(lp[:3], lp[3:], ref[:3], ref[3:], m[:3], m[3:], {"beta": 0.3})[0]
    got = torch.autograd.grad(loss, w)
    assert abs(float(loss) - float(loss64)) <= 1000 * 2.0 ** -24
    compare(got, want)


@pytest.mark.gpu
def test_captured_training_step(ops):
    """Forward, loss and gradients in one CUDA graph, through the functional forms."""
    s = make(4, 150, 48, 64, 500, seed=2)
    old = torch.full((4, 150), -6.0, device="cuda") + s["noise"][0]

    def step():
        proj = s["x"] @ s["w_in"]
        gate, v = proj.chunk(2, -1)
        h, final, ck = ops.linear_recurrence_train(gate, v, s["state"], form="sigmoid")
        logits = h @ s["w_out"]
        lp, ent, stats = ops.token_logprob_train(logits, s["token"])
        out, g, ge = ops.policy_loss_grad(lp, old, s["adv"], s["mask"], entropy=ent, entropy_coef=0.02)
        gl = ops.token_logprob_backward(logits, s["token"], stats, g, ge, out=logits)
        gh = gl @ s["w_out"].t()
        gg, gv, _ = ops.linear_recurrence_backward(gate, v, ck, gh, form="sigmoid")
        d = torch.cat([gg, gv], -1)
        return out, s["x"].flatten(0, 1).t() @ d.flatten(0, 1), h.flatten(0, 1).t() @ gl.flatten(0, 1)

    for _ in range(2):
        want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (2, 3):
        fresh = make(4, 150, 48, 64, 500, seed=seed)
        for k in ("x", "state"):
            s[k].copy_(fresh[k])
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)


def test_options_held_in_tensors_are_read_every_call():
    ops = pkg().ops
    v = torch.tensor(0.5)
    policy = lambda: ops._policy_options(0.2, 0.2, None, v, "k3", 0.0, "sum", 1.0, True, False)[3]
    preference = lambda: ops._preference_options(v, "sigmoid", 0.0, 0.0)[0]
    assert (policy(), preference()) == (0.5, 0.5)
    v.fill_(0.25)
    assert (policy(), preference()) == (0.25, 0.25)


def everything(ops, s, dtype):
    """Every operator once: all outputs."""
    x, gate, reset = s["x"].to(dtype), s["gate"].to(dtype), s["reset"]
    h, final, ckpt = ops.linear_recurrence_train(gate, x, s["state"], reset, "sigmoid")
    out = [h, final, ckpt, *ops.linear_recurrence(gate.transpose(0, 1).contiguous().transpose(0, 1), x, form="sigmoid")]
    out += ops.linear_recurrence_backward(gate, x, ckpt, h, final, reset, "sigmoid")
    pool, after = s["state"].clone(), torch.zeros_like(s["state"])
    out += [ops.linear_recurrence_step(gate[:, 0], x[:, 0], pool, s["slots"]), pool,
            ops.linear_recurrence_step(gate[:, 1], x[:, 1], pool, None, "sigmoid", state_out=after), after]
    lp, ent, stats = ops.token_logprob_train(h, s["token"], 0.7)
    out += [lp, ent, stats, *ops.token_logprob(h[:, 1:], s["token"][:, 1:]), ops.token_logprob(h[0], s["token"][0], 2.0, False)[0],
            ops.token_logprob_backward(h, s["token"], stats, lp, ent, 0.7)]
    out += ops.policy_loss_grad(lp, s["old"], s["adv"], s["mask"], s["old"], ent, kl_coef=0.1, entropy_coef=0.01)
    out += [ops.policy_loss(lp, None, lp, reduction="sum", dual_clip=3.0)]
    out += ops.preference_loss_grad(lp, lp[:, 5:], s["old"], s["old"][:, 5:], s["mask"], None, average=True)
    out += ops.preference_loss(lp, s["old"], form="hinge", margin=0.5)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_both_ways_of_a_call_agree(ops, monkeypatch, dtype):
    """What the module _calls returns has the bits of the call through ctypes, also while it is captured."""
    B, T, H = 3, 300, 200
    g = torch.Generator().manual_seed(5)
    s = {"x": torch.randn(B, T, H, generator=g).cuda(), "gate": torch.rand(B, T, H, generator=g).cuda(),
         "reset": (torch.rand(B, T, generator=g) < 0.02).cuda(), "state": torch.randn(B, H, generator=g).cuda(),
         "slots": torch.tensor([2, 0, 2], dtype=torch.int32).cuda(), "token": torch.randint(-1, H, (B, T), generator=g).cuda(),
         "old": -torch.rand(B, T, generator=g).cuda() * 8, "adv": torch.randn(B, generator=g).cuda(),
         "mask": (torch.rand(B, T, generator=g) < 0.8).cuda()}
    native = pkg()._native
    assert native.calls() is not None
    short = everything(ops, s, dtype)
    graph, during = captured(lambda: everything(ops, s, dtype))
    graph.replay()
    monkeypatch.setattr(native, "calls", lambda: None)
    long = everything(ops, s, dtype)
    assert len(short) == len(long) == len(during)
    for a, b, c in zip(short, long, during):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
        assert same_bits(a, b) and same_bits(c, b)


@pytest.mark.gpu
def test_calls_leave_what_they_cannot_take(ops):
    """The short way returns None for wrong arguments, and the checks in front of the long way say what is wrong."""
    calls = pkg()._native.calls()
    x = torch.zeros(2, 3, 4).cuda()
    for bad in (x.double(), x.cpu(), x[0], x.transpose(1, 2), torch.zeros(0, 3, 4).cuda(), None, 3, x.to_sparse()):
        assert calls.recurrence(x, bad, None, None, 0, False) is None
        assert calls.recurrence(bad, x, None, None, 0, False) is None
        assert calls.recurrence(x, x, bad, None, 0, False) is None or bad is None
        assert calls.recurrence(x, x, None, bad, 0, False) is None or bad is None
    for form in (-1, "decay", None, 1.0, 2 ** 70):
        assert calls.recurrence(x, x, None, None, form, False) is None
    with pytest.raises(ValueError, match="form"):
        ops.linear_recurrence(x, x, form="other")
    with pytest.raises(ValueError, match="last dimension"):
        ops.linear_recurrence(x.transpose(1, 2), x.transpose(1, 2))
