"""Gated linear recurrence: forward, backward and the single-token step.

The oracle (oracle.exact.linear_recurrence) steps through time in fp64 and bounds the error of an fp32
evaluation in any association; on the CPU its gradients are checked against differences.  GPU: every
type, both forms, odd sizes, strides and layouts, resets, one step to many tiles, a long narrow
sequence, the same bits on every call, captured and replayed calls, other streams.
"""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import exact
from sequence_policy import captured, load_ops, near, same_bits

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


@pytest.fixture(scope="module")
def ops():
    return load_ops()


def make(B, T, H, dtype, form, seed, reset_p=None, state=True, device="cuda"):
    """gate and x as halves of one projection [B, T, 2H]."""
    g = torch.Generator().manual_seed(seed)
    proj = torch.randn(B, T, 2 * H, generator=g)
    proj[..., :H] = proj[..., :H] * 1.5 + 1.5
    if form == "decay":
        proj[..., :H] = torch.tanh(proj[..., :H])  # in (-1, 1): negative gates too
    proj = proj.to(device=device, dtype=dtype)
    s = {"gate": proj[..., :H], "x": proj[..., H:]}
    s["state"] = torch.randn(B, H, generator=g).to(device) if state else None
    s["reset"] = (torch.rand(B, T, generator=g) < reset_p).to(device) if reset_p is not None else None
    s["grad_h"] = torch.randn(B, T, H, generator=g).to(device=device, dtype=dtype)
    s["grad_final"] = torch.randn(B, H, generator=g).to(device) if state else None
    return s


def check(ops, s, form):
    h, final, ck = ops.linear_recurrence_train(s["gate"], s["x"], s["state"], s["reset"], form)
    gg, gx, gs = ops.linear_recurrence_backward(s["gate"], s["x"], ck, s["grad_h"], s["grad_final"], s["reset"], form)
    h2, final2 = ops.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], form)
    torch.cuda.synchronize()
    assert same_bits(h, h2) and same_bits(final, final2)
    want, err = exact.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], form, s["grad_h"], s["grad_final"])
    got = {"h": h, "final": final, "grad_gate": gg, "grad_x": gx, "grad_state": gs}
    for k, v in got.items():
        near(v, want[k], err[k], k)


# --------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_oracle_gradients_against_differences(form):
    rng = np.random.default_rng(3)
    B, T, H = 2, 7, 3
    gate, x = rng.normal(size=(B, T, H)), rng.normal(size=(B, T, H))
    state, dh, df = rng.normal(size=(B, H)), rng.normal(size=(B, T, H)), rng.normal(size=(B, H))
    reset = rng.random((B, T)) < 0.2

    def loss(gate, x, state):
        v, _ = exact.linear_recurrence(gate, x, state, reset, form)
        return (v["h"] * dh).sum() + (v["final"] * df).sum()

    got, _ = exact.linear_recurrence(gate, x, state, reset, form, dh, df)
    for name, k in (("grad_gate", 0), ("grad_x", 1), ("grad_state", 2)):
        args = [gate, x, state]
        for at in np.ndindex(args[k].shape):
            up, dn = [a.copy() for a in args], [a.copy() for a in args]
            up[k][at] += 1e-6
            dn[k][at] -= 1e-6
            assert abs((loss(*up) - loss(*dn)) / 2e-6 - got[name][at]) < 1e-7, (name, at)


def test_refusals_on_the_cpu():
    ops = pkg().ops
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_recurrence(x, x)
    with pytest.raises(ValueError, match="form"):
        ops.linear_recurrence(x, x, form="other")
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_recurrence_step(x[0], x[0], torch.zeros(3, 4))


def test_status_codes_without_a_gpu():
    lib = pkg().load()
    st = (pkg()._native.c_i64 * 12)()
    P = 4096  # never dereferenced: each call is refused before any CUDA call
    assert lib.b200_linear_recurrence_async(P, P, 0, 0, st, None, None, -1, 4, 4, P, None, None, None, 0, None) == 1
    assert lib.b200_linear_recurrence_async(P, P, 9, 0, st, None, None, 1, 4, 4, P, None, None, P, 1 << 30, None) == 1
    assert lib.b200_linear_recurrence_async(P, P, 0, 7, st, None, None, 1, 4, 4, P, None, None, P, 1 << 30, None) == 1
    assert lib.b200_linear_recurrence_async(P, None, 0, 0, st, None, None, 1, 4, 4, P, None, None, P, 1 << 30, None) == 1
    assert lib.b200_linear_recurrence_async(P, P, 0, 0, None, None, None, 1, 4, 4, P, None, None, P, 1 << 30, None) == 1
    assert lib.b200_linear_recurrence_async(P, P, 0, 0, st, None, None, 0, 4, 4, P, None, None, None, 0, None) == 0
    assert lib.b200_linear_recurrence_backward_async(P, P, 0, 0, st, None, None, P, None, 1, 4, 4, P, P, None, P,
                                                     1 << 30, None) == 1
    assert lib.b200_linear_recurrence_step_async(P, P, 0, 0, st, P, P, None, 1, 2, 4, P, None) == 1  # too few states
    assert lib.b200_linear_recurrence_step_async(P, P, 0, 0, st, None, P, None, 2, 2, 4, P, None) == 1
    assert lib.b200_linear_recurrence_workspace_bytes(-1, 1, 1) == -1
    assert lib.b200_linear_recurrence_checkpoint_bytes(1, -1, 1) == -1


# --------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 3, 5), (1, 127, 64), (3, 128, 66), (2, 129, 33), (1, 255, 128),
                                   (2, 300, 70), (5, 515, 130), (1, 2049, 8), (2, 260, 193)])
def test_against_oracle(ops, dtype, form, B, T, H):
    check(ops, make(B, T, H, dtype, form, seed=T * 7 + H), form)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("p", [0.0, 0.02, 0.5, 1.0])
def test_resets(ops, dtype, form, p):
    check(ops, make(2, 400, 72, dtype, form, seed=11, reset_p=p), form)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 130, 700])
def test_no_state_and_no_final_gradient(ops, T):
    check(ops, make(2, T, 40, torch.float32, "sigmoid", seed=5, state=False), "sigmoid")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20_000, 66_001])
def test_long_narrow(ops, T):
    check(ops, make(1, T, 32, torch.float32, "decay", seed=T, reset_p=1e-4), "decay")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_long_narrow_16_bits(ops, dtype, form):
    """Several blocks of records, each brought in more than one round where a lane has two channels, with resets."""
    check(ops, make(2, 6011, 72, dtype, form, seed=77, reset_p=1e-3), form)


@pytest.mark.gpu
def test_many_channels(ops):
    check(ops, make(16, 260, 1030, torch.bfloat16, "sigmoid", seed=6, reset_p=0.01), "sigmoid")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["time_first", "odd_rows", "odd_start", "channels_slice"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts(ops, layout, dtype):
    B, T, H = 3, 270, 72
    s = make(B, T, H, dtype, "sigmoid", seed=21, reset_p=0.01)

    def lay(t):
        if layout == "time_first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "odd_rows":  # rows of H + 1 elements: every other row starts off alignment
            w = torch.empty(B, T, H + 1, dtype=t.dtype, device="cuda")[..., :H]
        elif layout == "odd_start":
            w = torch.empty(B * T * H + 3, dtype=t.dtype, device="cuda")[3:].view(B, T, H)
        else:
            w = torch.empty(B, T, 3 * H + 5, dtype=t.dtype, device="cuda")[..., H + 2:2 * H + 2]
        w.copy_(t)
        return w

    for k in ("gate", "x", "grad_h"):
        s[k] = lay(s[k])
    if layout == "time_first":
        s["reset"] = s["reset"].t().contiguous().t()
    check(ops, s, "sigmoid")
    h, _ = ops.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], "sigmoid")
    if layout == "time_first":
        assert h.transpose(0, 1).is_contiguous()
    # an output of the caller's, in the caller's layout, with what lies around it left as it was
    big = torch.full((B + 2, T, H + 4), 7.0, dtype=dtype, device="cuda")
    out = big[1:-1, :, 2:-2]
    got, _ = ops.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], "sigmoid", out=out)
    torch.cuda.synchronize()
    assert got is out and same_bits(out, h)
    big[1:-1, :, 2:-2] = 7.0
    assert torch.equal(big, torch.full_like(big, 7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("H", [64, 65])
def test_strides_beyond_32_bits(ops, H):
    """A batch stride of more than 2^31 elements, by tensor loads (H = 64) and by copies."""
    gap = 2**31 + 64
    s = make(2, 200, H, torch.bfloat16, "sigmoid", seed=H)
    store = torch.empty(gap + 3 * 200 * H, dtype=torch.bfloat16, device="cuda")
    for k, k0 in (("gate", 0), ("x", 200 * H), ("grad_h", 2 * 200 * H)):
        v = store.as_strided((2, 200, H), (gap, H, 1), k0)
        v.copy_(s[k])
        s[k] = v
    check(ops, s, "sigmoid")


@pytest.mark.gpu
def test_broadcast_inputs(ops):
    """A gate shared by all sequences and steps (strides 0)."""
    s = make(3, 200, 48, torch.float32, "sigmoid", seed=2)
    s["gate"] = s["gate"][:1, :1].expand(3, 200, 48)
    check(ops, s, "sigmoid")


@pytest.mark.gpu
def test_extreme_gates(ops):
    """Gates whose sigmoid is 0 or 1 in fp32, and decays of 0 and +-1."""
    s = make(2, 300, 64, torch.float32, "sigmoid", seed=8)
    g = s["gate"].clone()
    g[:, ::3] = 200.0
    g[:, 1::5] = -200.0
    s["gate"] = g
    check(ops, s, "sigmoid")
    d = make(2, 300, 64, torch.float32, "decay", seed=9)
    g = torch.where(torch.rand(2, 300, 64, device="cuda") < 0.5, 1.0, -1.0)
    g[:, ::7] = 0.0
    d["gate"] = g
    check(ops, d, "decay")


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_reset_drops_non_finite_states(ops, bad):
    """What a document leaves behind, infinities and NaN included, does not reach the next one."""
    s = make(2, 600, 40, torch.float32, "decay", seed=4, reset_p=0.0)
    s["x"] = s["x"].clone()
    s["x"][0, 250] = bad
    s["state"][1] = bad
    s["reset"][0, 300] = True
    s["reset"][1, 0] = True
    h, final = ops.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], "decay")
    torch.cuda.synchronize()
    assert torch.isfinite(h[0, :250]).all() and torch.isfinite(h[0, 300:]).all() and torch.isfinite(h[1]).all()
    assert not torch.isfinite(h[0, 250]).any() and torch.isfinite(final).all()
    s["x"][0, 250] = 0.0
    want, err = exact.linear_recurrence(s["gate"], s["x"], None, s["reset"], "decay")
    near(h[0, 300:], want["h"][0, 300:], err["h"][0, 300:])
    near(h[1], want["h"][1], err["h"][1])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H", [(0, 5, 4), (2, 5, 0), (2, 0, 4)])
def test_empty(ops, B, T, H):
    g = torch.zeros(B, T, H, device="cuda")
    state = torch.randn(B, H, device="cuda")
    h, final, ck = ops.linear_recurrence_train(g, g, state)
    gg, gx, gs = ops.linear_recurrence_backward(g, g, ck, g, state)
    torch.cuda.synchronize()
    assert h.shape == (B, T, H) and torch.equal(final, state) and torch.equal(gs, state)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("B,H", [(1, 1), (5, 33), (64, 2048), (300, 72)])
def test_step(ops, dtype, form, B, H):
    s = make(B, 1, H, dtype, form, seed=B + H)
    gate, x = s["gate"][:, 0], s["x"][:, 0]
    S = B + 5
    pool = torch.randn(S, H, device="cuda")
    slots = torch.randperm(S, device="cuda")[:B].to(torch.int32)
    before = pool.clone()
    h = ops.linear_recurrence_step(gate, x, pool, slots, form)
    torch.cuda.synchronize()
    want, err = exact.linear_recurrence(s["gate"], s["x"], before[slots.long()], None, form)
    near(h, want["h"][:, 0], err["h"][:, 0], "h")
    near(pool[slots.long()], want["final"], err["final"], "state")
    rest = torch.ones(S, dtype=torch.bool, device="cuda")
    rest[slots.long()] = False
    assert torch.equal(pool[rest], before[rest])
    own = before.clone()
    out = torch.full((S, H), 3.0, device="cuda")
    h2 = ops.linear_recurrence_step(gate, x, own, form=form, state_out=out)
    torch.cuda.synchronize()
    want, err = exact.linear_recurrence(s["gate"], s["x"], before[:B], None, form)
    near(h2, want["h"][:, 0], err["h"][:, 0], "h")
    near(out[:B], want["final"], err["final"], "state_out")
    assert torch.equal(own, before) and torch.equal(out[B:], torch.full_like(out[B:], 3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 5])
def test_steps_make_the_sequence(ops, T):
    """Token by token through the step: the state of the whole-sequence call."""
    s = make(3, T, 50, torch.float32, "sigmoid", seed=T)
    state = s["state"].clone()
    hs = [ops.linear_recurrence_step(s["gate"][:, t], s["x"][:, t], state, form="sigmoid") for t in range(T)]
    torch.cuda.synchronize()
    want, err = exact.linear_recurrence(s["gate"], s["x"], s["state"], None, "sigmoid")
    near(torch.stack(hs, 1), want["h"], err["h"])
    near(state, want["final"], err["final"])


@pytest.mark.gpu
def test_step_same_slot_twice_and_slots_out_of_range(ops):
    """Rows of one slot are consecutive tokens of one sequence; rows without a slot are left alone."""
    H = 37
    slots = torch.tensor([2, 0, -1, 2, 9, 2, 0], dtype=torch.int32, device="cuda")
    s = make(7, 1, H, torch.float32, "sigmoid", seed=1)
    gate, x = s["gate"][:, 0], s["x"][:, 0]
    pool = torch.randn(4, H, device="cuda")
    before = pool.clone()
    out = torch.full((7, H), 5.0, device="cuda")
    ops.linear_recurrence_step(gate, x, pool, slots, "sigmoid", out=out)
    torch.cuda.synchronize()
    for slot, rows in ((2, [0, 3, 5]), (0, [1, 6])):
        want, err = exact.linear_recurrence(gate[rows][None], x[rows][None], before[slot:slot + 1], None, "sigmoid")
        near(out[rows], want["h"][0], err["h"][0])
        near(pool[slot:slot + 1], want["final"], err["final"])
    assert torch.equal(out[[2, 4]], torch.full((2, H), 5.0, device="cuda"))
    assert torch.equal(pool[[1, 3]], before[[1, 3]])


@pytest.mark.gpu
def test_same_bits_on_every_call_and_stream(ops):
    s = make(2, 3000, 200, torch.bfloat16, "sigmoid", seed=13, reset_p=0.001)
    first = None
    for k in range(12):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            h, final, ck = ops.linear_recurrence_train(s["gate"], s["x"], s["state"], s["reset"], "sigmoid")
            grads = ops.linear_recurrence_backward(s["gate"], s["x"], ck, s["grad_h"], s["grad_final"], s["reset"],
                                                   "sigmoid")
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        now = (h, final, *grads)
        if first is None:
            first = now
        assert all(same_bits(a, b) for a, b in zip(now, first))


@pytest.mark.gpu
def test_workspace_serves_other_sizes(ops):
    """Calls of different sizes and directions on one stream share scratch: large, small, large again."""
    for k, (B, T, H) in enumerate([(2, 3000, 96), (1, 130, 32), (4, 700, 64), (2, 3000, 96), (1, 5000, 40)]):
        check(ops, make(B, T, H, torch.float32, "decay", seed=k), "decay")


@pytest.mark.gpu
def test_captured_and_replayed(ops):
    """Two graphs of the same shapes, replayed at the same time on two streams and beside an eager call."""
    sets = [make(2, 1500, 96, torch.float32, "sigmoid", seed=k, reset_p=0.002) for k in range(3)]

    def call(s):
        h, final, ck = ops.linear_recurrence_train(s["gate"], s["x"], s["state"], s["reset"], "sigmoid")
        return (h, final, *ops.linear_recurrence_backward(s["gate"], s["x"], ck, s["grad_h"], s["grad_final"],
                                                          s["reset"], "sigmoid"))

    (ga, oa), (gb, ob) = captured(lambda: call(sets[0])), captured(lambda: call(sets[1]))
    want = [[t.clone() for t in call(s)] for s in sets]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        torch.cuda.synchronize()
        for t in (*oa, *ob):
            t.fill_(9)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            ga.replay()
        with torch.cuda.stream(b):
            gb.replay()
        eager = call(sets[2])
        torch.cuda.synchronize()
        for got, w in ((oa, want[0]), (ob, want[1]), (eager, want[2])):
            assert all(same_bits(x, y) for x, y in zip(got, w))
    sets[0]["x"].copy_(sets[2]["x"])  # a replay reads what its inputs hold then
    changed = call(sets[0])
    ga.replay()
    torch.cuda.synchronize()
    assert all(same_bits(x, y) for x, y in zip(oa, changed))


@pytest.mark.gpu
def test_autograd(ops):
    s = make(2, 150, 24, torch.float32, "sigmoid", seed=3, reset_p=0.02)
    gate, x = s["gate"].clone().requires_grad_(), s["x"].clone().requires_grad_()
    state = s["state"].clone().requires_grad_()
    h, final = ops.LinearRecurrenceFunction.apply(gate, x, state, s["reset"], "sigmoid")
    torch.autograd.backward([h, final], [s["grad_h"], s["grad_final"]])
    want, err = exact.linear_recurrence(s["gate"], s["x"], s["state"], s["reset"], "sigmoid", s["grad_h"],
                                        s["grad_final"])
    for t, k in ((gate, "grad_gate"), (x, "grad_x"), (state, "grad_state")):
        near(t.grad, want[k], err[k], k)
    # only h used, through an expanded gradient; no state
    gate.grad = x.grad = None
    ops.LinearRecurrenceFunction.apply(gate, x, None, s["reset"], "sigmoid")[0].sum().backward()
    want, err = exact.linear_recurrence(s["gate"], s["x"], None, s["reset"], "sigmoid", np.ones((2, 150, 24)))
    near(gate.grad, want["grad_gate"], err["grad_gate"])
    near(x.grad, want["grad_x"], err["grad_x"])


@pytest.mark.gpu
def test_refusals(ops):
    x = torch.zeros(2, 3, 4, device="cuda")
    for bad in (lambda: ops.linear_recurrence(x, x.half()), lambda: ops.linear_recurrence(x[:, :2], x),
                lambda: ops.linear_recurrence(x.double(), x.double()), lambda: ops.linear_recurrence(x[0], x[0]),
                lambda: ops.linear_recurrence(x.transpose(1, 2), x.transpose(1, 2)),
                lambda: ops.linear_recurrence(x, x, state=torch.zeros(2, 3, device="cuda")),
                lambda: ops.linear_recurrence(x, x, state=torch.zeros(2, 4, device="cuda").half()),
                lambda: ops.linear_recurrence(x, x, reset=torch.zeros(2, 3, device="cuda")),
                lambda: ops.linear_recurrence(x, x, reset=torch.zeros(3, 2, device="cuda", dtype=torch.bool)),
                lambda: ops.linear_recurrence(x, x, out=torch.zeros(1, 3, 4, device="cuda").expand(2, 3, 4)),
                lambda: ops.linear_recurrence(x, x.clone(), out=x),
                lambda: ops.linear_recurrence_step(x[0], x[0].clone(), torch.zeros(3, 4, device="cuda"), out=x[0]),
                lambda: ops.linear_recurrence_backward(x, x, torch.zeros(3, device="cuda"), x),
                lambda: ops.linear_recurrence_step(x[0], x[0], torch.zeros(2, 4, device="cuda")),
                lambda: ops.linear_recurrence_step(x[0], x[0], torch.zeros(3, 5, device="cuda")),
                lambda: ops.linear_recurrence_step(x[0], x[0], torch.zeros(3, 4, device="cuda"),
                                                   torch.zeros(3, device="cuda", dtype=torch.int64))):
        with pytest.raises((ValueError, TypeError)):
            bad()
    lib = pkg().load()
    st = (pkg()._native.c_i64 * 8)(12, 4, 12, 4, 12, 4, 0, 0)
    need = lib.b200_linear_recurrence_workspace_bytes(2, 300, 4)
    if need:  # too small a workspace is refused before anything is launched
        p = x.data_ptr()
        assert lib.b200_linear_recurrence_async(p, p, 0, 0, st, None, None, 2, 300, 4, p, None, None, p, need - 1,
                                                None) == 4


@pytest.mark.gpu
def test_refuses_inputs_in_the_written_state(ops):
    pool = torch.randn(8, 40, device="cuda")
    gate, x = torch.rand(2, 40, device="cuda"), torch.randn(2, 40, device="cuda")
    slots = torch.tensor([7, 6], dtype=torch.int32, device="cuda")
    before = pool.clone()
    for kw in (dict(gate=pool[:2], x=x), dict(gate=gate, x=pool[1:5:2])):
        with pytest.raises(ValueError, match="written state overlaps"):
            ops.linear_recurrence_step(state=pool, slots=slots, **kw)
        with pytest.raises(ValueError, match="written state overlaps"):
            ops.linear_recurrence_step(state=before, slots=slots, state_out=pool, **kw)
    assert torch.equal(pool, before)
    ops.linear_recurrence_step(gate, before[:2], pool, slots)          # reading another pool is fine
    state = torch.randn(2, 40, device="cuda")
    with pytest.raises(ValueError, match="out overlaps state"):
        ops.linear_recurrence(gate[:, None], x[:, None], state, out=state[:, None])
