"""Token log-probabilities and entropies from logits, and the gradient of the logits.

The oracle (oracle.exact.token_logprob) works in fp64 and bounds an fp32 evaluation; on the CPU its
gradients are checked against differences.  GPU: every type, vocabularies from 1 to some hundred
thousand, odd row lengths and alignments, views, masked rows, masked logits, extreme values.
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


def make(B, T, V, dtype, seed, masked=0.15, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, T, V, generator=g) * scale).to("cuda", dtype)
    token = torch.randint(0, V, (B, T), generator=g)
    token[torch.rand(B, T, generator=g) < masked] = -100
    return {"logits": logits, "token": token.cuda(), "gl": torch.randn(B, T, generator=g).cuda(),
            "ge": torch.randn(B, T, generator=g).cuda()}


def check(ops, s, temperature=1.0, entropy=True):
    lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"], temperature, entropy)
    lp2, ent2 = ops.token_logprob(s["logits"], s["token"], temperature, entropy)
    grad = ops.token_logprob_backward(s["logits"], s["token"], stats, s["gl"], s["ge"] if entropy else None, temperature)
    torch.cuda.synchronize()
    assert same_bits(lp, lp2) and (not entropy or same_bits(ent, ent2))
    want, err = exact.token_logprob(s["logits"], s["token"], temperature, s["gl"], s["ge"] if entropy else None)
    near(lp, want["log_prob"], err["log_prob"], "log_prob")
    if entropy:
        near(ent, want["entropy"], err["entropy"], "entropy")
    else:
        assert ent is None
    near(grad, want["grad_logits"], err["grad_logits"], "grad_logits")
    assert grad.is_contiguous() and grad.dtype == s["logits"].dtype
    return lp, ent, grad


# --------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("temperature", [0.7, 1.0])
def test_oracle_gradients_against_differences(temperature):
    rng = np.random.default_rng(2)
    x = rng.normal(size=(3, 6))
    tok = np.array([2, 5, -1])
    gl, ge = rng.normal(size=3), rng.normal(size=3)
    got = exact.token_logprob(x, tok, temperature, gl, ge)[0]["grad_logits"]

    def loss(x):
        v = exact.token_logprob(x, tok, temperature)[0]
        return (v["log_prob"] * gl).sum() + (v["entropy"] * ge).sum()

    for at in np.ndindex(x.shape):
        up, dn = x.copy(), x.copy()
        up[at] += 1e-6
        dn[at] -= 1e-6
        assert abs((loss(up) - loss(dn)) / 2e-6 - got[at]) < 1e-8


def test_refusals_on_the_cpu():
    ops = pkg().ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprob(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    lib = pkg().load()
    st = (pkg()._native.c_i64 * 4)()
    P = 4096  # never dereferenced: each call is refused before any CUDA call
    for args in ((P, 0, st, P, -1, 1, 5, 1.0, P, None, None), (P, 0, st, P, 1, 1, 0, 1.0, P, None, None),
                 (P, 5, st, P, 1, 1, 5, 1.0, P, None, None), (P, 0, st, P, 1, 1, 5, 0.0, P, None, None),
                 (P, 0, st, P, 1, 1, 5, float("nan"), P, None, None), (P, 0, None, P, 1, 1, 5, 1.0, P, None, None),
                 (None, 0, st, P, 1, 1, 5, 1.0, P, None, None), (P, 0, st, P, 1, 1, 5, 1.0, None, None, None),
                 (P, 0, st, P, 2**31 - 1, 2, 5, 1.0, P, None, None)):
        assert lib.b200_token_logprob_async(*args, None) == 1
    assert lib.b200_token_logprob_async(None, 0, st, None, 0, 1, 5, 1.0, None, None, None, None) == 0
    assert lib.b200_token_logprob_backward_async(P, 0, st, P, None, P, None, 1, 1, 5, 1.0, P, None) == 1


# --------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 2, 2), (2, 3, 7), (3, 5, 31), (1, 4, 255), (2, 9, 1000), (1, 7, 4099),
                                   (2, 2, 8192), (1, 3, 32768), (1, 2, 50001), (1, 1, 200_003), (40, 30, 64),
                                   (20, 50, 515)])
def test_against_oracle(ops, dtype, B, T, V):
    check(ops, make(B, T, V, dtype, seed=V + T))


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [True, False])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 2.5])
def test_temperature_and_without_entropy(ops, entropy, temperature):
    check(ops, make(2, 5, 3001, torch.bfloat16, seed=3), temperature, entropy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("V", [33, 1000, 9001])
def test_views(ops, dtype, V):
    """Next-token training: logits[:, :-1] against token[:, 1:]; rows of a wider buffer; an odd start."""
    s = make(3, 6, V, dtype, seed=V)
    full = torch.randint(0, V, (3, 7), device="cuda")
    wide = torch.randn(3, 7, V, device="cuda").to(dtype)
    a = dict(s, logits=wide[:, :-1], token=full[:, 1:])
    check(ops, a)
    check(ops, dict(s, logits=torch.randn(3, 6, V + 11, device="cuda").to(dtype)[..., 3:V + 3]))
    odd = torch.empty(3 * 6 * V + 1, dtype=dtype, device="cuda")[1:].view(3, 6, V)
    odd.copy_(s["logits"])
    check(ops, dict(s, logits=odd))
    flat = dict(s, logits=s["logits"][0], token=s["token"][0], gl=s["gl"][0], ge=s["ge"][0])
    check(ops, flat)
    check(ops, dict(s, logits=s["logits"][:1].expand(3, 6, V)))  # one sequence's logits against several targets


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("V", [40, 5003, 40_000])
def test_masked_logits(ops, dtype, V):
    """Logits of -inf and of the type's lowest value; tokens among them; a row of nothing but the lowest."""
    s = make(2, 4, V, dtype, seed=1, masked=0.0)
    x = s["logits"]
    x[0, 0, V // 3:] = float("-inf")
    x[0, 1, : V // 2] = torch.finfo(dtype).min
    x[0, 2] = torch.finfo(dtype).min
    x[0, 3, 1:] = float("-inf")  # one token left: probability 1
    x[1, 0, 0] = torch.finfo(dtype).max
    x[1, 1, ::2] = float("-inf")
    s["token"][:] = torch.tensor([[0, V - 1, 3, 0], [0, 1, 2, 5]], device="cuda")
    check(ops, s)
    s["token"][0, 0] = V - 1  # a token of probability 0
    lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"])
    g = ops.token_logprob_backward(s["logits"], s["token"], stats, s["gl"], s["ge"])
    torch.cuda.synchronize()
    assert lp[0, 0] == float("-inf") and torch.isfinite(ent).all() and torch.isfinite(g).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 5003, 40_000])
def test_undefined_rows_are_nan_and_stay_alone(ops, V):
    s = make(1, 6, V, torch.float32, seed=5, masked=0.0)
    x = s["logits"]
    x[0, 0] = float("-inf")
    x[0, 1, V // 2] = float("nan")
    x[0, 2, V // 2] = float("inf")
    s["token"][0, 3] = V  # not a token
    s["token"][0, 4] = -1
    lp, ent, stats = ops.token_logprob_train(x, s["token"])
    g = ops.token_logprob_backward(x, s["token"], stats, s["gl"], s["ge"])
    torch.cuda.synchronize()
    assert torch.isnan(lp[0, :4]).all() and torch.isnan(ent[0, :3]).all()
    assert torch.isnan(g[0, :4]).any(-1).all()
    assert lp[0, 4] == 0 and ent[0, 4] == 0 and (g[0, 4] == 0).all()
    want, err = exact.token_logprob(x[0, 5:], s["token"][0, 5:], 1.0, s["gl"][0, 5:], s["ge"][0, 5:])
    near(lp[0, 5:], want["log_prob"], err["log_prob"])
    near(g[0, 5:], want["grad_logits"], err["grad_logits"])


@pytest.mark.gpu
def test_masked_rows_are_not_read(ops):
    s = make(2, 3, 777, torch.bfloat16, seed=9, masked=0.0)
    s["token"][1, 1] = -100
    s["logits"][1, 1] = float("nan")
    lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"])
    g = ops.token_logprob_backward(s["logits"], s["token"], stats, s["gl"], s["ge"])
    torch.cuda.synchronize()
    assert torch.isfinite(lp).all() and torch.isfinite(ent).all() and torch.isfinite(g).all()
    assert (g[1, 1] == 0).all()


@pytest.mark.gpu
def test_large_offsets_keep_their_digits(ops):
    """A constant added to a row (exactly, in fp32) changes nothing."""
    g = torch.Generator().manual_seed(4)
    x = (torch.randint(-64, 64, (1, 8, 3000), generator=g).float() / 16).cuda()
    token = torch.randint(0, 3000, (1, 8), generator=g).cuda()
    lp, ent = ops.token_logprob(x, token)
    lp2, ent2 = ops.token_logprob(x + 2.0 ** 16, token)
    torch.cuda.synchronize()
    assert same_bits(lp, lp2) and same_bits(ent, ent2)


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets(ops):
    """More than 2^31 logits: the last rows are where they should be."""
    V, N = 131072, 16400
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 8191, 16383, N - 1])
    g = torch.Generator().manual_seed(1)
    part = (torch.randn(4, V, generator=g) * 2).to("cuda", torch.bfloat16)
    x[rows.cuda()] = part
    token = torch.full((N,), -1, device="cuda")
    token[rows.cuda()] = torch.randint(0, V, (4,), generator=g).cuda()
    lp, ent, stats = ops.token_logprob_train(x, token)
    gl = torch.ones(N, device="cuda")
    grad = ops.token_logprob_backward(x, token, stats, gl, gl)
    torch.cuda.synchronize()
    want, err = exact.token_logprob(part, token[rows.cuda()], 1.0, gl[:4], gl[:4])
    near(lp[rows.cuda()], want["log_prob"], err["log_prob"])
    near(grad[rows.cuda()], want["grad_logits"], err["grad_logits"])
    assert not grad[1:8191].any() and not grad[8192:16383].any()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1000, 1001, 60_000])
def test_gradient_over_the_logits(ops, V):
    s = make(2, 5, V, torch.bfloat16, seed=V)
    _, _, grad = check(ops, s)
    x = s["logits"].clone()
    _, _, stats = ops.token_logprob_train(x, s["token"])
    out = ops.token_logprob_backward(x, s["token"], stats, s["gl"], s["ge"], out=x)
    torch.cuda.synchronize()
    assert out is x and same_bits(x, grad)


@pytest.mark.gpu
def test_captured_streams_and_repeats(ops):
    s = make(3, 4, 30_001, torch.bfloat16, seed=17)

    def call():
        lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"])
        return lp, ent, ops.token_logprob_backward(s["logits"], s["token"], stats, s["gl"], s["ge"])

    want = call()
    graph, out = captured(call)
    other = torch.cuda.Stream()
    for _ in range(3):
        for t in out:
            t.fill_(3)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        now = call()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) and same_bits(a, c) for a, b, c in zip(want, out, now))


@pytest.mark.gpu
def test_autograd(ops):
    s = make(2, 5, 700, torch.float32, seed=2)
    x = s["logits"].clone().requires_grad_()
    lp, ent = ops.TokenLogProbFunction.apply(x, s["token"], 0.8)
    (lp * s["gl"]).sum().add((ent * s["ge"]).sum()).backward()
    want, err = exact.token_logprob(s["logits"], s["token"], 0.8, s["gl"], s["ge"])
    near(x.grad, want["grad_logits"], err["grad_logits"])
    x.grad = None
    ops.TokenLogProbFunction.apply(x, s["token"], 0.8)[1].sum().backward()  # entropy alone, expanded gradient
    want, err = exact.token_logprob(s["logits"], s["token"], 0.8, torch.zeros(2, 5), torch.ones(2, 5))
    near(x.grad, want["grad_logits"], err["grad_logits"])


@pytest.mark.gpu
def test_empty_and_refusals(ops):
    lp, ent = ops.token_logprob(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (0,) and ent.shape == (0,)
    x, k = torch.zeros(2, 3, 5, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    stats, g = torch.zeros(2, 3, 3, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in (lambda: ops.token_logprob(x.double(), k), lambda: ops.token_logprob(x, k.int()),
                lambda: ops.token_logprob(x, k[:, :2]), lambda: ops.token_logprob(x.transpose(1, 2), k),
                lambda: ops.token_logprob(x, k, 0.0), lambda: ops.token_logprob(x, k, float("inf")), lambda: ops.token_logprob(x, k, 1e-40),
                lambda: ops.token_logprob(x[..., :0], k), lambda: ops.token_logprob(x, k.cpu()),
                lambda: ops.token_logprob(x[0, 0], k[0, 0]),
                lambda: ops.token_logprob_backward(x, k, stats[..., :2], g),
                lambda: ops.token_logprob_backward(x, k, stats, g.half()),
                lambda: ops.token_logprob_backward(x, k, stats, g[:1]),
                lambda: ops.token_logprob_backward(x, k, stats, g, out=x[:1]),
                lambda: ops.token_logprob_backward(x.flatten()[:25].view(5, 5), k[:1, 0].expand(5), stats[0, 0].expand(5, 3)
                                                   .contiguous(), g[0, 0].expand(5).contiguous(),
                                                   out=x.flatten()[1:26].view(5, 5))):
        with pytest.raises((ValueError, TypeError)):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(127, 2048), (128, 2048), (511, 2048), (513, 2048), (2469, 8995), (2600, 8995)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_both_sides_of_a_warp_per_row(ops, dtype, rows, V):
    """Row numbers on either side of where a warp takes a row alone, forward and backward."""
    check(ops, make(1, rows, V, dtype, seed=rows), 0.9)


@pytest.mark.gpu
def test_backward_refuses_an_output_over_its_inputs(ops):
    s = make(1, 6, 50, torch.float32, seed=2)
    lp, ent, stats = ops.token_logprob_train(s["logits"], s["token"])
    whole = torch.zeros(300 + 18, device="cuda")
    inside = whole[300:].view(1, 6, 3).copy_(stats)
    ops.token_logprob_backward(s["logits"], s["token"], inside, s["gl"], out=whole[:300].view(1, 6, 50))
    with pytest.raises(ValueError, match="out overlaps stats"):
        ops.token_logprob_backward(s["logits"], s["token"], inside, s["gl"], out=whole[18:].view(1, 6, 50))
    with pytest.raises(ValueError, match="out overlaps grad_log_prob"):
        ops.token_logprob_backward(s["logits"], s["token"], stats, whole[:6].view(1, 6), out=whole[:300].view(1, 6, 50))
