"""Categorical actions and gradient clipping (``isaaclab_amd.rl``) against their definitions in float64 (oracle/policy_np.py).

Drawn actions are whole numbers and have to be equal; a log-probability is within its one rounding.  With u = 2^-24, half a
step of float32, the tolerances of the 32-bit results are (V entries a row, d = (x - max) / T, at most the entry's own):
  log_prob   d carries three roundings, ln s the relative error of s: each term's exp (2 u) and its own 3 u |d| (weighted by
             p: 3 u H <= 3 u ln V), and at most V / 64 + 16 additions in a chain: u (8 |d| + V / 64 + 3 ln V + 32)
  entropy    ln s - t / s, t's terms like those of s times |d|: u (V / 64 + 3 ln V + 32) (2 + 2 ln V)
  gradient   p (gl + ge (ln p + H)): p has the relative error of its exponent, so p (|gl| + |ge| (|ln p| + H + 1)) times
             4 u (8 |d| + V / 64 + 3 ln V + 32), and one rounding to its type: half a step of it
  norm       64-bit sums, one rounding: 2 u of it;  clipped: the factor's rounding, the product's: (2 u + half a step) of it"""
import math
import zlib

import numpy as np
import pytest
import torch

import isaaclab_amd._lib as L
from isaaclab_amd import rl
from oracle import policy_np as O
from test_abi import _c_sizeof

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.detach().double().cpu().numpy()


def f32v(v):
    return float(np.float32(v))


def rng_of(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


# -- without a GPU ----------------------------------------------------------------------------------------------------
def test_struct_mirrors():
    import ctypes as C

    for (name, cls), size in zip([("mdp_categorical_sample_t", L.MdpCategoricalSample),
                                  ("mdp_categorical_eval_t", L.MdpCategoricalEval), ("mdp_grad_t", L.MdpGrad)],
                                 _c_sizeof(["mdp_categorical_sample_t", "mdp_categorical_eval_t", "mdp_grad_t"])):
        assert C.sizeof(cls) == size, name


def test_oracle_against_torch():
    """The restatement against torch's own log_softmax, entropy and autograd in float64."""
    g = rng_of("oracle")
    x = torch.randn(6, 17, generator=g, dtype=torch.float64, requires_grad=True)
    a = torch.randint(0, 17, (6,), generator=g)
    gl, ge = torch.randn(6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    dist = torch.distributions.Categorical(logits=x / 0.7)
    lp, h = dist.log_prob(a), dist.entropy()
    (grad,) = torch.autograd.grad((lp, h), x, (gl, ge))
    for r in range(6):
        got = O.evaluate_row(x[r].detach().numpy(), int(a[r]), None, 0.7, float(gl[r]), float(ge[r]))
        np.testing.assert_allclose(got[0], lp[r].item(), rtol=1e-12)
        np.testing.assert_allclose(got[1], h[r].item(), rtol=1e-12)
        np.testing.assert_allclose(got[2], grad[r].numpy(), rtol=1e-10, atol=1e-14)
    # kept entries by hand: weights 4, 2, 1, 1 of 8
    x = np.log(np.array([1.0, 4.0, 1.0, 2.0]))
    assert O.kept_entries(x, top_k=3)[0].tolist() == [0, 1, 3]          # the first of equal ones
    assert O.kept_entries(x, top_p=0.6)[0].tolist() == [1, 3]
    assert O.kept_entries(x, min_p=0.3)[0].tolist() == [1, 3]
    assert O.kept_entries(x, top_p=0.0)[0].tolist() == [1]
    assert O.kept_entries(x, temperature=0.0)[0].tolist() == [1]
    assert O.sample_row(x, 0.124)[0] == 0 and O.sample_row(x, 0.126)[0] == 1
    assert O.sample_row(np.full(3, -np.inf), 0.5) == (-1, 0.0)


def test_refusals_before_any_launch():
    """Bad arguments at the C entries; the pointers are never read."""
    import ctypes as C

    a = L.MdpCategoricalSample()
    assert L.lib.mdp_categorical_sample(None, None) == L.MDP_ERR_INVALID
    a.rows, a.vocab, a.dtype = -1, 4, 0
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "negative shape" in L.last_error()
    a.rows, a.dtype = 2, 7
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "element type" in L.last_error()
    a.dtype, a.vocab = 0, 0
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "without entries" in L.last_error()
    a.vocab = 4
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "null logits" in L.last_error()
    a.logits, a.ld = 4096, 4
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "null output" in L.last_error()
    a.actions = a.log_prob = 4096
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "generator state" in L.last_error()
    a.rows = 1 << 41
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "too many" in L.last_error()
    a.rows, a.logits = 2, 4098
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_ERR_INVALID and "between two elements" in L.last_error()
    a.rows = 0
    assert L.lib.mdp_categorical_sample(C.byref(a), None) == L.MDP_OK
    e = L.MdpCategoricalEval()
    e.rows, e.vocab, e.logits, e.ld = 2, 4, 4096, 4
    assert L.lib.mdp_categorical_evaluate(C.byref(e), None) == L.MDP_ERR_INVALID
    assert L.lib.mdp_categorical_evaluate_grad(C.byref(e), None, None, None, 4, None) == L.MDP_ERR_INVALID
    e.actions = e.stats = 4096
    assert L.lib.mdp_categorical_evaluate_grad(C.byref(e), None, None, 4096, 3, None) == L.MDP_ERR_INVALID
    assert "overlap" in L.last_error()

    def clip(rows, kind=2, max_norm=1.0, ws=64, norm=64):
        table = (L.MdpGrad * max(1, len(rows)))(*[L.MdpGrad(*r) for r in rows])
        return L.lib.mdp_grad_clip(table, len(rows), kind, max_norm, ws, norm, None)

    ok = (4096, 4096, 16, 0, 0)
    for rows, kw in [([ok], dict(kind=3)), ([ok], dict(max_norm=-1.0)), ([ok], dict(max_norm=math.nan)), ([ok], dict(ws=None)),
                     ([ok], dict(norm=None)), ([(4096, 4096, -1, 0, 0)], {}), ([(None, 4096, 4, 0, 0)], {}),
                     ([(4096, None, 4, 0, 0)], {}), ([(4096, 8192, 4, 0, 1)], {}), ([(4096, 8192, 4, 9, 9)], {}),
                     ([(4096, 4096, 4, 1, 0)], {}),                              # in place into another type
                     ([ok, ok], {}),                                             # the same memory twice
                     ([ok, (8192, 4096 + 60, 4, 0, 0)], {}),                     # an output inside another gradient
                     ([(8192, 4096, 16, 0, 0), (16384, 4096 + 32, 2, 0, 0)], {}),   # two outputs overlap
                     ([(4096, 4100, 16, 0, 0)], {}),                             # an output shifted over its own gradient
                     ([(4096, 4096, 1 << 41, 0, 0)], {}), ([(4098, 4098, 4, 0, 0)], {}), ([(4096, 8193, 4, 1, 1)], {})]:
        assert clip(rows, **kw) == L.MDP_ERR_INVALID, (rows, kw)
        assert L.last_error()
    assert L.lib.mdp_grad_norm(None, 1, 2, 64, 64, None) == L.MDP_ERR_INVALID
    assert L.lib.mdp_grad_workspace(0) >= 1 and L.lib.mdp_grad_workspace(1000) > L.lib.mdp_grad_workspace(10)


def test_no_cpu_path():
    x, a = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: rl.sample_categorical(x), lambda: rl.evaluate_categorical(x, a),
                 lambda: rl.evaluate_categorical_grad(x, a, None, None), lambda: rl.grad_norm([x]), lambda: rl.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="norm_type"):
        rl.grad_norm([x], 3.0)
    with pytest.raises(ValueError, match="max_norm"):
        rl.clip_grads([x], -1.0)
    assert float(rl.grad_norm([])) == 0.0 and float(rl.clip_grad_norm_([], 1.0)) == 0.0


# -- drawing ----------------------------------------------------------------------------------------------------------
def check_draw(x, u, got, mask=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Every row of a call against the definition: equal actions, log-probabilities within their rounding."""
    V = x.shape[-1]
    xs, us = f64(x).reshape(-1, V), f64(u).reshape(-1)
    ms = None if mask is None else mask.expand(x.shape).cpu().numpy().reshape(-1, V)
    cols = [np.broadcast_to(f64(v) if isinstance(v, torch.Tensor) else f32v(v), x.shape[:-1]).reshape(-1)
            for v in (temperature, top_k, top_p, min_p)]
    a, lp = got[0].cpu().numpy().reshape(-1), f64(got[1]).reshape(-1)
    assert got[0].shape == x.shape[:-1] == got[1].shape and got[0].dtype == torch.int64 and got[1].dtype == torch.float32
    for r in range(len(xs)):
        want = O.sample_row(xs[r], us[r], None if ms is None else ms[r], *(c[r] for c in cols))
        assert a[r] == want[0], (r, a[r], want, us[r])
        np.testing.assert_allclose(lp[r], want[1], rtol=2 * U, atol=1e-12, err_msg=f"row {r}")


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=5, temperature=1.7), dict(top_k=50, top_p=0.8),
            dict(top_p=0.9), dict(top_p=0.3, min_p=0.05), dict(min_p=0.2), dict(min_p=1.0), dict(top_p=0.0), dict(temperature=0.0),
            dict(top_k=1000000, top_p=0.999, temperature=3.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 19, 63, 64, 65, 255, 256, 257, 1000, 1025, 1500, 2500, 4000, 4099])
def test_draw(device, dtype, vocab):
    g = rng_of("draw", dtype, vocab)
    for n, s in enumerate(SETTINGS):
        rows = 9 if vocab < 4000 else 4
        x = (torch.randn(rows, vocab, generator=g) * (0.3, 2.0, 6.0)[n % 3]).to(DT[dtype]).to(device)
        u = torch.rand(rows, generator=g).to(device)
        check_draw(x, u, rl.sample_categorical(x, u, **s), **s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [8191, 16411, 33000, 70001, 140003, 300007])
def test_draw_long_rows(device, dtype, vocab):
    g = rng_of("long", dtype, vocab)
    for n, s in enumerate([dict(), dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_p=0.95), dict(min_p=0.01, top_p=0.99),
                           dict(top_k=20000, top_p=0.7, temperature=2.0), dict(temperature=0.0)]):
        x = (torch.randn(3, vocab, generator=g) * (3.0, 0.5)[n % 2]).to(DT[dtype]).to(device)
        u = torch.rand(3, generator=g).to(device)
        check_draw(x, u, rl.sample_categorical(x, u, **s), **s)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 64, 300, 1800, 3900, 5000, 40000])
def test_draw_equal_logits(device, vocab):
    """Few different values: the border of every setting falls among equal entries, which go by lowest index."""
    g = rng_of("ties", vocab)
    for s in SETTINGS + [dict(top_k=vocab // 2), dict(top_k=max(1, vocab // 3), top_p=0.7), dict(top_p=0.45, temperature=2.0)]:
        for levels in (1, 2, 3):
            x = torch.randint(0, levels, (5, vocab), generator=g).float().to(device)
            x = torch.where(torch.rand(5, vocab, generator=g).to(device) < 0.5, x, -0.0 * x)     # zeros of both signs
            u = torch.rand(5, generator=g).to(device)
            check_draw(x, u, rl.sample_categorical(x, u, **s), **s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [4, 77, 700, 1500, 3500, 6000])
def test_draw_masks_and_special_values(device, dtype, vocab):
    """Rows that a mask or -inf leaves empty, single entries, lowest and largest finite values, NaN and infinities behind the
    mask and in front of it."""
    g = rng_of("mask", dtype, vocab)
    rows = 16
    x = (torch.randn(rows, vocab, generator=g) * 2).to(DT[dtype])
    mask = torch.rand(rows, vocab, generator=g) < 0.6
    low, high = torch.finfo(DT[dtype]).min, torch.finfo(DT[dtype]).max
    mask[0] = False                                     # nothing allowed
    x[1] = -math.inf                                    # nothing possible
    mask[2] = False
    mask[2, vocab - 1] = True                           # one entry
    x[3] = low                                          # all at the type's lowest value: uniform
    mask[3] = True
    x[4, ::2] = low
    x[5, mask[5].logical_not()] = math.nan              # behind the mask: no effect
    x[6, mask[6].logical_not()] = math.inf
    x[7, 1], mask[7, 1] = math.nan, True                # in front of it
    x[8, 2], mask[8, 2] = math.inf, True
    x[9, 1:] = -math.inf
    mask[9, 0] = True                                   # one finite entry
    x[10, 3], mask[10, 3] = high, True
    x[11, 0], mask[11, 0] = low, True
    x[11, 1:] = -math.inf
    x, mask = x.to(device), mask.to(device)
    u = torch.rand(rows, generator=g).to(device)
    for s in SETTINGS:
        got = rl.sample_categorical(x, u, mask=mask, **s)
        check_draw(x, u, got, mask=mask, **s)
        assert got[0][:2].tolist() == [-1, -1] and got[1][:2].tolist() == [0.0, 0.0] and got[0][2] == vocab - 1
        assert got[0][7:9].tolist() == [-1, -1] and bool(got[1][7:9].isnan().all())
    row = torch.rand(vocab, generator=g).to(device) < 0.5          # one mask for every row
    row[0] = True
    check_draw(x[4:7], u[4:7], rl.sample_categorical(x[4:7], u[4:7], mask=row), mask=row)


@pytest.mark.gpu
def test_draw_uniform_edges(device):
    """u = 0, the largest below 1, and values outside [0, 1), which count as the nearest inside."""
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0, -40.0]], device=device).repeat(6, 1)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -3.0, math.inf, math.nan], device=device)
    a, lp = rl.sample_categorical(x, u)
    assert a.tolist() == [0, 3, 3, 0, 3, 0]
    check_draw(x, u, (a, lp))
    far = torch.full((1, 300), -2000.0, device=device)              # weights below every 64-bit number are never drawn
    far[0, 250] = 0.0
    assert rl.sample_categorical(far, torch.zeros(1, device=device))[0].item() == 250


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [33, 900, 1700, 3600, 9000])
def test_draw_per_row_settings(device, vocab):
    g = rng_of("rows", vocab)
    lead = (3, 4)
    x = (torch.randn(*lead, vocab, generator=g) * 2).to(device)
    u = torch.rand(lead, generator=g).to(device)
    t = torch.rand(lead, generator=g) * 2
    t[0, 0], t[0, 1], t[0, 2], t[1, 0] = 0.0, -1.0, math.nan, math.inf
    k = torch.randint(-1, 40, lead, generator=g)
    p = torch.rand(lead, generator=g) * 1.2
    q = torch.rand(lead, generator=g) * 0.3 - 0.05
    s = dict(temperature=t.to(device), top_k=k.to(device), top_p=p.to(device), min_p=q.to(device))
    check_draw(x, u, rl.sample_categorical(x, u, **s), **s)
    one = dict(temperature=torch.tensor([[0.5], [1.0], [2.0]], device=device), top_k=torch.tensor(1 << 40, device=device))
    check_draw(x, u, rl.sample_categorical(x, u, **one), **one)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [700, 3000, 9001, 70001, 300007])
def test_draw_rising_and_falling_rows(device, vocab):
    """Rows in order of their values: the largest entry so far changes with every entry, or never; the border is a place."""
    line = torch.linspace(-7.0, 7.0, vocab)
    step = torch.arange(vocab) * 1e-7
    x = torch.stack([line, line.flip(0), step, step.flip(0), (line * 1e-3), line ** 3 / 10]).to(device)
    for s in (dict(top_p=0.5), dict(top_p=0.93, temperature=0.3), dict(top_k=vocab // 3, top_p=0.8), dict(min_p=0.3), dict()):
        for shift in (0.0, 0.61):
            u = torch.tensor([0.1, 0.25, 0.4, 0.5, 0.7, 0.9], device=device).add(shift).remainder(1.0)
            check_draw(x, u, rl.sample_categorical(x, u, **s), **s)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, vocab, scale", [(3000, 40, 0.1), (700, 1000, 0.3), (300, 3000, 2.0), (100, 9000, 0.2), (40, 70001, 1.0)])
def test_draw_repeats_itself(device, rows, vocab, scale):
    """The same call gives the same bits, whatever order its lanes list entries in."""
    g = rng_of("again", vocab)
    x = (torch.randn(rows, vocab, generator=g) * scale).to(torch.bfloat16).to(device)
    u = torch.rand(rows, generator=g).to(device)
    first = rl.sample_categorical(x, u, top_p=0.7, top_k=vocab // 2)
    check_draw(x[:4], u[:4], (first[0][:4], first[1][:4]), top_p=0.7, top_k=vocab // 2)
    for _ in range(4):
        again = rl.sample_categorical(x, u, top_p=0.7, top_k=vocab // 2)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_draw_layouts(device):
    """Any strides and offsets, one row, no rows, an expanded row, a non-default stream."""
    g = rng_of("layout")
    base = (torch.randn(12, 41, 7, generator=g) * 2).to(device)
    u = torch.rand(12, generator=g).to(device)
    wide = torch.randn(12, 1003, generator=g).to(torch.bfloat16).to(device)
    for x in (base[:, :, 3], base[:, :, 0].t()[:12, :].contiguous().t()[:, :12], wide[:, 3:990], wide[:, 1:65], base[:, 5, :],
              wide[::2][:, ::3].repeat(2, 1), wide[:1, 5:].expand(12, -1)):
        check_draw(x, u[:x.shape[0]], rl.sample_categorical(x, u[:x.shape[0]], top_p=0.9), top_p=0.9)
    m = (torch.rand(12, 2100, generator=g) < 0.5).to(device)[:, 1:1976:2]
    x = wide[:, 3:991]
    check_draw(x, u, rl.sample_categorical(x, u, mask=m), mask=m)
    check_draw(wide[0], u[0], rl.sample_categorical(wide[0], u[0]))
    a, lp = rl.sample_categorical(wide[:0], u[:0])
    assert a.shape == (0,) and lp.shape == (0,)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rl.sample_categorical(x, u, top_k=7)
    side.synchronize()
    check_draw(x, u, got, top_k=7)


@pytest.mark.gpu
def test_draw_generator(device):
    """Without u: the device generator, by seed, moving with every call and every replay; frequencies within five standard
    errors of their shares."""
    from isaaclab_amd.utils import math as M

    x = torch.log(torch.tensor([0.1, 0.2, 0.3, 0.4], device=device)).expand(200_000, 4)
    M.seed_samplers(11, device)
    a = rl.sample_categorical(x)[0]
    b = rl.sample_categorical(x)[0]
    assert not torch.equal(a, b)
    M.seed_samplers(11, device)
    assert torch.equal(rl.sample_categorical(x)[0], a)
    share = torch.bincount(a, minlength=4).double().cpu().numpy() / len(a)
    want = np.array([0.1, 0.2, 0.3, 0.4])
    assert (np.abs(share - want) < 5 * np.sqrt(want * (1 - want) / len(a))).all()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = rl.sample_categorical(x)[0]
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    M.seed_samplers(1, device)


@pytest.mark.gpu
def test_draw_refusals(device):
    x, u = torch.zeros(2, 3, device=device), torch.zeros(2, device=device)
    for match, call in [("float32, bfloat16", lambda: rl.sample_categorical(x.double(), u)),
                        ("at least one entry", lambda: rl.sample_categorical(x[:, :0], u)),
                        ("u must be", lambda: rl.sample_categorical(x, u[:1])),
                        ("u must be", lambda: rl.sample_categorical(x, u.double())),
                        ("temperature", lambda: rl.sample_categorical(x, u, temperature=-0.5)),
                        ("temperature", lambda: rl.sample_categorical(x, u, temperature=math.nan)),
                        ("top_k", lambda: rl.sample_categorical(x, u, top_k=-1)),
                        ("whole number", lambda: rl.sample_categorical(x, u, top_k=2.5)),
                        ("top_p", lambda: rl.sample_categorical(x, u, top_p=1.5)),
                        ("min_p", lambda: rl.sample_categorical(x, u, min_p=-0.1)),
                        ("top_p of shape", lambda: rl.sample_categorical(x, u, top_p=torch.ones(3, device=device))),
                        ("top_p lives on", lambda: rl.sample_categorical(x, u, top_p=torch.ones(2))),
                        ("bool", lambda: rl.sample_categorical(x, u, mask=torch.ones(2, 3, device=device))),
                        ("broadcast", lambda: rl.sample_categorical(x, u, mask=torch.ones(4, 3, dtype=torch.bool, device=device)))]:
        with pytest.raises(ValueError, match=match):
            call()


# -- evaluating -------------------------------------------------------------------------------------------------------
def check_evaluation(x, a, lp, h, grad, gl, ge, mask=None, temperature=1.0):
    V = x.shape[-1]
    xs, as_ = f64(x).reshape(-1, V), a.cpu().numpy().reshape(-1)
    ms = None if mask is None else mask.expand(x.shape).cpu().numpy().reshape(-1, V)
    t = np.broadcast_to(f64(temperature) if isinstance(temperature, torch.Tensor) else f32v(temperature), x.shape[:-1]).reshape(-1)
    lps, hs, gs = f64(lp).reshape(-1), f64(h).reshape(-1), f64(grad).reshape(-1, V)
    gls, ges = f64(gl).reshape(-1), f64(ge).reshape(-1)
    assert lp.dtype == h.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
    chain = V / 64 + 3 * math.log(V + 1) + 32
    step = torch.finfo(x.dtype).eps / 2
    floor = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps          # one step of the denormals
    for r in range(len(xs)):
        want = O.evaluate_row(xs[r], as_[r], None if ms is None else ms[r], t[r], gls[r], ges[r])
        ok = O.allowed_entries(xs[r], None if ms is None else ms[r])
        d = np.zeros(V)
        if ok.any() and np.isfinite(xs[r][ok]).all():
            d[ok] = np.minimum((xs[r][ok].max() - xs[r][ok]) / t[r], 200.0)
            d_full = (xs[r][ok].max() - xs[r][as_[r]]) / t[r] if 0 <= as_[r] < V and ok[as_[r]] else 0.0
            # ln w is held at -200 in what is summed, not in the log-probability of an action
            np.testing.assert_allclose(lps[r], want[0], rtol=0, atol=U * (8 * abs(d_full) + chain), err_msg=f"log_prob {r}")
        else:
            np.testing.assert_allclose(lps[r], want[0], rtol=0, atol=U * chain, equal_nan=True, err_msg=f"log_prob {r}")
        np.testing.assert_allclose(hs[r], want[1], rtol=0, atol=U * chain * (2 + 2 * math.log(V + 1)), equal_nan=True, err_msg=f"entropy {r}")
        if not np.isfinite(want[1]) or not np.isfinite(want[2]).all():
            assert np.array_equal(np.isnan(gs[r]), np.isnan(want[2])), f"gradient {r}"
            continue
        log_p = O.evaluate_row(xs[r], -1, None if ms is None else ms[r], t[r])[2]      # zeros; shape only
        z = np.where(ok, -d, 0.0)
        p = np.where(ok, np.exp(z), 0.0)
        if ok.any():
            log_p = np.where(ok, z - np.log(p.sum()), 0.0)
            p = p / p.sum()
        tol = p * (abs(gls[r]) + abs(ges[r]) * (np.abs(log_p) + want[1] + 1)) * 4 * U * (8 * d + chain) / t[r]
        tol += (step + 4 * U) * np.abs(want[2]) + floor
        assert (np.abs(gs[r] - want[2]) <= tol).all(), (r, np.abs(gs[r] - want[2]).max(), tol[np.abs(gs[r] - want[2]).argmax()])
        assert (gs[r][~ok] == 0).all()


def run_evaluation(x, a, gl, ge, **kw):
    leaf = x.detach().requires_grad_()
    lp, h = rl.evaluate_categorical(leaf, a, **kw)
    (grad,) = torch.autograd.grad((lp, h), leaf, (gl, ge))
    raw = rl.evaluate_categorical_grad(x, a, gl, ge, **kw)
    assert all(torch.equal(p.view(torch.uint8), q.contiguous().view(torch.uint8)) for p, q in zip(raw[:2], (lp.detach(), h.detach())))
    assert torch.equal(raw[2].isnan(), grad.isnan()) and torch.equal(raw[2].nan_to_num(), grad.nan_to_num())
    return lp, h, grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 19, 33, 64, 65, 128, 255, 513, 1024, 1500, 2050, 3001, 5003, 33001, 131075])
def test_evaluation(device, dtype, vocab):
    g = rng_of("evaluate", dtype, vocab)
    for n, t in enumerate((1.0, 0.6, 2.5)):
        rows = 37 if vocab < 3000 else 3
        x = (torch.randn(rows, vocab, generator=g) * (0.5, 3.0, 20.0)[n]).to(DT[dtype]).to(device)
        a = torch.randint(0, vocab, (rows,), generator=g).to(device)
        gl, ge = (torch.randn(rows, generator=g).to(device) for _ in range(2))
        check_evaluation(x, a, *run_evaluation(x, a, gl, ge, temperature=t), gl, ge, temperature=t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [5, 60, 700, 1600, 9001])
def test_evaluation_masks_and_special_values(device, dtype, vocab):
    g = rng_of("evaluate mask", dtype, vocab)
    rows = 16
    x = (torch.randn(rows, vocab, generator=g) * 2).to(DT[dtype])
    mask = torch.rand(rows, vocab, generator=g) < 0.6
    mask[:, 1] = True
    a = torch.ones(rows, dtype=torch.int64)
    low = torch.finfo(DT[dtype]).min
    mask[0], a[0] = False, -1                           # nothing allowed, and told so
    x[1], a[1] = -math.inf, -1                          # nothing possible
    mask[2] = False                                     # nothing allowed, but an action all the same
    mask[3, 1] = False                                  # an action that is not allowed
    mask[3, 0] = True
    x[4], mask[4] = low, True                           # uniform at the type's lowest value
    x[5, 2:] = low
    x[6, ~mask[6]] = math.nan                           # behind the mask: no effect
    x[7, ~mask[7]] = math.inf
    x[8, 1] = math.nan                                  # in front of it
    x[9, 1] = math.inf
    a[10], a[11] = vocab, -2                            # no such entries
    x[12, 0], mask[12, 0] = -math.inf, True
    a[12] = 0                                           # an impossible action
    mask[13] = False
    mask[13, 1] = True                                  # one entry
    a[14] = -1                                          # no action where there are entries
    x, mask, a = x.to(device), mask.to(device), a.to(device)
    gl, ge = (torch.randn(rows, generator=g).to(device) for _ in range(2))
    lp, h, grad = run_evaluation(x, a, gl, ge, mask=mask)
    check_evaluation(x, a, lp, h, grad, gl, ge, mask=mask)
    assert lp[:2].tolist() == [0.0, 0.0] and h[:3].tolist() == [0.0] * 3 and not bool(grad[:3].any())
    assert lp[3].item() == lp[2].item() == lp[12].item() == -math.inf and lp[13].item() == 0.0 == h[13].item()
    assert bool(lp[8:12].isnan().all()) and lp[14].item() == 0.0


@pytest.mark.gpu
def test_evaluation_gradient_against_differences(device):
    """Central differences of the float64 definition along random directions."""
    g = rng_of("differences")
    rows, vocab, t = 8, 23, 0.8
    x = torch.randn(rows, vocab, generator=g).to(device)
    a = torch.randint(0, vocab, (rows,), generator=g).to(device)
    gl, ge = (torch.randn(rows, generator=g).to(device) for _ in range(2))
    grad = f64(rl.evaluate_categorical_grad(x, a, gl, ge, temperature=t)[2])
    xs = f64(x)
    for r in range(rows):
        v = torch.randn(vocab, generator=g).double().numpy()

        def value(s):
            lp, h, _ = O.evaluate_row(xs[r] + s * v, int(a[r]), None, f32v(t))
            return float(gl[r]) * lp + float(ge[r]) * h

        # the difference quotient's own error: h^2 / 6 of a third derivative of order 10, and 1e-16 / h
        np.testing.assert_allclose(grad[r] @ v, (value(1e-5) - value(-1e-5)) / 2e-5, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_evaluation_layouts_and_autograd(device):
    """Strided and expanded logits (the gradient of a shared row is the sum), one loss through one of the two results, per-row
    temperatures, a leading shape, gradients that arrive expanded."""
    g = rng_of("evaluate layout")
    base = torch.randn(6, 4, 50, generator=g).to(device)
    a = torch.randint(0, 46, (6, 4), generator=g).to(device)
    t = (torch.rand(6, 1, generator=g) + 0.5).to(device)
    leaf = base.clone().requires_grad_()
    x = leaf[:, :, 3:49]
    lp, h = rl.evaluate_categorical(x, a, temperature=t)
    (lp.sum() + 0.0 * h.sum()).backward()
    one = torch.ones(6, 4, device=device)
    check_evaluation(x, a, lp, h, leaf.grad[:, :, 3:49], one, 0 * one, temperature=t)
    assert not bool(leaf.grad[:, :, :3].any()) and not bool(leaf.grad[:, :, 49:].any())
    lp, h = rl.evaluate_categorical(x, a, temperature=t)
    (only_h,) = torch.autograd.grad(h.sum(), x)
    check_evaluation(x, a, lp, h, only_h, 0 * one, one, temperature=t)
    row = torch.randn(46, generator=g).to(device).requires_grad_()
    lp, _ = rl.evaluate_categorical(row.expand(24, 46), a.view(-1))
    (shared,) = torch.autograd.grad(lp.sum(), row)
    want = sum(O.evaluate_row(f64(row), int(i), None, 1.0, 1.0, 0.0)[2] for i in a.view(-1).tolist())
    np.testing.assert_allclose(f64(shared), want, rtol=0, atol=24 * U * 200)
    turned = torch.randn(46, 24, generator=g).to(device).requires_grad_()
    lp, h = rl.evaluate_categorical(turned.t(), a.view(-1))
    (grad,) = torch.autograd.grad(lp.sum() + h.sum(), turned)
    check_evaluation(turned.t(), a.view(-1), lp, h, grad.t(), one.view(-1), one.view(-1))
    empty = torch.zeros(0, 5, device=device, requires_grad=True)
    lp, h = rl.evaluate_categorical(empty, a.view(-1)[:0])
    assert torch.autograd.grad(lp.sum(), empty)[0].shape == (0, 5)
    bad = torch.tensor([1.0, 0.0, -1.0, math.nan], device=device)
    lp, h = rl.evaluate_categorical(base[0, :, :46], a[0], temperature=bad)
    assert bool(lp[1:].isnan().all()) and bool(h[1:].isnan().all()) and bool(lp[0].isfinite())
    x = base.clone().requires_grad_()
    y = x * 1.0
    lp, _ = rl.evaluate_categorical(y, a)
    y.add_(1.0)                                          # the saved logits changed: autograd says so
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        lp.sum().backward()
    for match, call in [("actions must be", lambda: rl.evaluate_categorical(base, a.int())),
                        ("actions must be", lambda: rl.evaluate_categorical(base, a[:2])),
                        ("temperature", lambda: rl.evaluate_categorical(base, a, temperature=0.0)),
                        ("no gradient", lambda: rl.evaluate_categorical(base, a, temperature=t.clone().requires_grad_())),
                        ("grad_entropy", lambda: rl.evaluate_categorical_grad(base, a, None, one.double()))]:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(device):
    """A row whose first entry lies more than 2^32 entries into its tensor, read and written."""
    vocab, rows = 1000, 4_400_000
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=device)
    last = torch.randn(1, vocab, generator=rng_of("far")).to(torch.bfloat16).to(device)
    x[:] = 0
    x[-1:] = last
    x[0] = 1
    u = torch.full((rows,), 0.37, device=device)
    a, lp = rl.sample_categorical(x, u, top_p=0.9)
    check_draw(last, u[-1:], (a[-1:], lp[-1:]), top_p=0.9)
    assert a[1].item() == a[rows - 2].item() == O.sample_row(np.zeros(vocab), f32v(0.37), top_p=f32v(0.9))[0]
    one = torch.ones(rows, device=device)
    lp, h, grad = rl.evaluate_categorical_grad(x, a, one, one)
    check_evaluation(last, a[-1:], lp[-1:], h[-1:], grad[-1:], one[:1], one[:1])


@pytest.mark.gpu
def test_more_rows_than_a_launch_holds(device):
    """Rows beyond 2^21 are drawn, evaluated and differentiated by further launches; the generator goes by the row of the call."""
    from isaaclab_amd.utils import math as M

    rows, n = (1 << 21) + 1003, 5
    g = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(rows, 3, generator=g, device=device)
    u = torch.rand(rows, generator=g, device=device)
    temperature = torch.rand(rows, generator=g, device=device) + 0.5
    mask = torch.rand(rows, 3, generator=g, device=device) < 0.8
    got = rl.sample_categorical(x, u, mask=mask, top_p=0.8, temperature=temperature)
    gl = torch.randn(rows, generator=g, device=device)
    lp, h, grad = rl.evaluate_categorical_grad(x, got[0], gl, gl, mask=mask, temperature=temperature)
    for at in (0, (1 << 21) - n, 1 << 21, rows - n):
        part = slice(at, at + n)
        check_draw(x[part], u[part], (got[0][part], got[1][part]), mask=mask[part], top_p=0.8, temperature=temperature[part])
        check_evaluation(x[part], got[0][part], lp[part], h[part], grad[part], gl[part], gl[part], mask=mask[part],
                         temperature=temperature[part])
    M.seed_samplers(4, device)
    a = rl.sample_categorical(x[:1].expand(rows, 3))[0]
    assert not torch.equal(a[:1003], a[1 << 21:])
    M.seed_samplers(1, device)


@pytest.mark.gpu
def test_a_very_long_row(device):
    """Sums of many more terms than 24 bits count: a flat row of 3.3e7 entries."""
    vocab = (1 << 25) + 77
    x = torch.zeros(1, vocab, dtype=torch.float16, device=device)
    u = torch.tensor([0.75], device=device)
    a, lp = rl.sample_categorical(x, u)
    assert a.item() == int(0.75 * vocab)                            # the first i with i + 1 > 0.75 vocab
    np.testing.assert_allclose(lp.item(), -math.log(vocab), rtol=2 * U)
    a, lp = rl.sample_categorical(x, u, top_p=0.5)
    kept = math.ceil(0.5 * vocab)
    assert a.item() == int(0.75 * kept)
    np.testing.assert_allclose(lp.item(), -math.log(kept), rtol=2 * U)
    one = torch.ones(1, device=device)
    lp, h, grad = rl.evaluate_categorical_grad(x, a, one, one)
    # exact sums: what is left is the rounding of ln s and of one product
    np.testing.assert_allclose([lp.item(), h.item()], [-math.log(vocab), math.log(vocab)], rtol=4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 3000])
def test_smallest_temperatures(device, vocab):
    """Down to the smallest normal number the definition holds -- logits that lie 1e-37 apart are then far apart --, below it the
    largest logit is taken."""
    g = rng_of("cold", vocab)
    x = (torch.rand(6, vocab, generator=g) * 4e-36).to(device)
    u = torch.rand(6, generator=g).to(device)
    t = torch.tensor([2e-36, 1.2e-38, 1e-39, 1e-45, 1e-30, 3e38], device=device)
    a, lp = rl.sample_categorical(x, u, temperature=t, top_p=0.9)
    exact = torch.where(t < 1.1754944e-38, 0.0, t)
    check_draw(x, u, (a, lp), temperature=exact, top_p=0.9)


# -- gradients --------------------------------------------------------------------------------------------------------
def grads_of(g, sizes, types, device, scale=0.1):
    return [(torch.randn(n, generator=g) * scale).to(DT[t]).to(device) for n, t in zip(sizes, types)]


def check_clip(before, after, norm, max_norm, norm_type=2.0):
    arrays = [f64(t) for t in before]
    want = O.grad_norm(arrays, norm_type)
    assert norm.dtype == torch.float32 and norm.shape == ()
    np.testing.assert_allclose(float(norm), want, rtol=2 * U)
    f = O.clip_factor(want, max_norm)
    for b, x, y in zip(before, arrays, after):
        got = f64(y)
        assert y.shape == b.shape
        if f == 1.0:
            assert np.array_equal(got, x)
        else:
            floor = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
            np.testing.assert_allclose(got, x * f, rtol=2 * U + torch.finfo(y.dtype).eps / 2, atol=floor)


@pytest.mark.gpu
@pytest.mark.parametrize("norm_type", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4095, 4096, 4097], [1_000_003], [7] * 97, [13, 900, 70_001] * 70])
def test_clip_in_place_and_out_of_place(device, sizes, norm_type):
    g = rng_of("clip", sizes[:3], len(sizes), norm_type)
    for types in (["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16"]):
        types = (types * len(sizes))[:len(sizes)]
        grads = grads_of(g, sizes, types, device)
        want = O.grad_norm([f64(t) for t in grads], norm_type)
        np.testing.assert_allclose(float(rl.grad_norm(grads, norm_type)), want, rtol=2 * U)
        for max_norm in (0.3 * want, 3.0 * want, 0.0):
            out, norm = rl.clip_grads(grads, max_norm, norm_type)
            check_clip(grads, out, norm, max_norm, norm_type)
            wide = [torch.full(t.shape, math.nan, device=device) for t in grads]
            got, norm = rl.clip_grads(grads, max_norm, norm_type, out=wide)
            assert all(p is q for p, q in zip(got, wide))
            check_clip(grads, wide, norm, max_norm, norm_type)
            params = [torch.nn.Parameter(torch.empty_like(t)) for t in grads]
            for p, t in zip(params, grads):
                p.grad = t.clone()
            norm = rl.clip_grad_norm_(params + params[:1], max_norm, norm_type)        # one given twice counts once
            check_clip(grads, [p.grad for p in params], norm, max_norm, norm_type)


@pytest.mark.gpu
def test_clip_layouts(device):
    """Odd offsets inside one buffer, turned and channels-last gradients, a parameter without a gradient, a single tensor."""
    g = rng_of("clip layout")
    for t in ("f32", "bf16", "f16"):
        for shift in (1, 2, 3, 5):
            flat = torch.randn(40_000, generator=g).to(DT[t]).to(device)
            keep = flat.clone()
            cuts = [shift, 1003 + shift, 9000, 9001, 30_007]
            views = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
            before = [v.clone() for v in views]
            out, norm = rl.clip_grads(views, 1.0, out=views)
            check_clip(before, views, norm, 1.0)
            assert torch.equal(flat[:shift], keep[:shift]) and torch.equal(flat[30_007:], keep[30_007:])
    turned = torch.randn(30, 70, generator=g).to(device).t()
    last = torch.randn(2, 5, 6, 7, generator=g).to(device).to(memory_format=torch.channels_last)
    before = [turned.clone(), last.clone()]
    out, norm = rl.clip_grads([turned, last], 2.0)
    check_clip(before, out, norm, 2.0)
    p, q = torch.nn.Parameter(turned.clone()), torch.nn.Parameter(last.clone())
    p.grad, unused = turned, torch.nn.Parameter(torch.zeros(3, device=device))
    check_clip(before[:1], [p.grad], rl.clip_grad_norm_([p, unused], 2.0), 2.0)
    q.grad = last
    check_clip(before[1:], [q.grad], rl.clip_grad_norm_(q, 2.0), 2.0)


@pytest.mark.gpu
def test_clip_range_and_special_values(device):
    big = torch.full((5000,), 1e30, device=device)                   # squares beyond 32 bits
    small = torch.full((5000,), 1e-30, device=device)
    for t in (big, small):
        np.testing.assert_allclose(float(rl.grad_norm(t)), f64(t)[0] * math.sqrt(5000), rtol=2 * U)
    x = torch.randn(9000, generator=rng_of("special")).to(device)
    for where in (0, 4500, 8999):
        y = x.clone()
        y[where] = math.inf
        out, norm = rl.clip_grads([y], 1.0)
        assert float(norm) == math.inf and bool(out[0][where].isnan()) and int(out[0].count_nonzero()) == 1
        y[where] = math.nan
        for kind in (2.0, 1.0, math.inf):
            out, norm = rl.clip_grads([y, x], 1.0, kind)
            assert math.isnan(float(norm)) and all(bool(o.isnan().all()) for o in out)
    zero = torch.zeros(10, device=device)
    out, norm = rl.clip_grads([zero], 1.0)
    assert float(norm) == 0.0 and not bool(out[0].any())
    first = [float(rl.grad_norm([x, big * 1e-30])) for _ in range(3)]
    assert first[0] == first[1] == first[2]


@pytest.mark.gpu
def test_clip_refusals(device):
    x, half = torch.zeros(64, device=device), torch.zeros(64, dtype=torch.float16, device=device)
    for match, call in [("float32, bfloat16", lambda: rl.grad_norm([x.double()])),
                        ("gaps or overlap", lambda: rl.grad_norm([x[::2]])),
                        ("gaps or overlap", lambda: rl.grad_norm([x[:1].expand(5)])),
                        ("1 outputs for 2", lambda: rl.clip_grads([x, half], 1.0, out=[x])),
                        ("gradient's type or float32", lambda: rl.clip_grads([x], 1.0, out=[half])),
                        ("shape and strides", lambda: rl.clip_grads([x], 1.0, out=[torch.zeros(63, device=device)])),
                        ("shape and strides", lambda: rl.clip_grads([x.view(8, 8)], 1.0, out=[torch.zeros(8, 8, device=device).t()])),
                        ("overlaps another", lambda: rl.clip_grads([x, x], 1.0, out=[x, x])),
                        ("overlaps another", lambda: rl.clip_grads([x[:32], x[32:]], 1.0, out=[x[32:], x[:32]])),
                        ("overlaps another", lambda: rl.clip_grads([x[:32]], 1.0, out=[x[1:33]])),
                        ("strided", lambda: rl.grad_norm([x.to_sparse()])),
                        ("norm_type", lambda: rl.clip_grads([x], 1.0, 3)),
                        ("max_norm", lambda: rl.clip_grads([x], math.nan))]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(TypeError):
        rl.clip_grads([3.0], 1.0)


# -- together ---------------------------------------------------------------------------------------------------------
class Policy(torch.nn.Module):
    def __init__(self, obs, joints, bins):
        super().__init__()
        self.joints, self.bins = joints, bins
        self.net = torch.nn.Sequential(torch.nn.Linear(obs, 64), torch.nn.ELU(), torch.nn.Linear(64, joints * bins))

    def forward(self, x):
        return self.net(x).view(*x.shape[:-1], self.joints, self.bins)


def surrogate(ratio, advantage, entropy):
    return -torch.min(ratio * advantage, ratio.clamp(0.8, 1.2) * advantage).mean() - 0.01 * entropy.mean()


@pytest.mark.gpu
def test_one_update(device):
    """Draw while rolling out, evaluate the stored actions with gradients, clip: the parameters' gradients against the same
    loss on torch's float64 distribution, and the ratio of an unchanged policy is one."""
    torch.manual_seed(5)
    net = Policy(20, 12, 33).to(device)
    g = rng_of("update")
    obs, u = torch.randn(64, 20, generator=g).to(device), torch.rand(64, 12, generator=g).to(device)
    advantage = torch.randn(64, 12, generator=g).to(device)
    forbidden = (torch.rand(64, 12, 33, generator=g) < 0.2).to(device)
    with torch.no_grad():
        actions, old = rl.sample_categorical(net(obs), u, mask=~forbidden)
    log_prob, entropy = rl.evaluate_categorical(net(obs), actions, mask=~forbidden)
    # two roundings of numbers up to ln(33) + the spread of the logits
    np.testing.assert_allclose(f64(log_prob), f64(old), rtol=0, atol=U * 200)
    surrogate(torch.exp(log_prob - old), advantage, entropy).backward()
    got = [p.grad.clone() for p in net.parameters()]
    norm = rl.clip_grad_norm_(net.parameters(), 0.05)
    twin = Policy(20, 12, 33).to(device).double()
    twin.load_state_dict(net.state_dict())
    dist = torch.distributions.Categorical(logits=twin(obs.double()).masked_fill(forbidden, -1e300))
    p = dist.probs
    entropy = -(p * torch.where(p > 0, p, 1.0).log()).sum(-1)
    surrogate(torch.exp(dist.log_prob(actions) - old.double()), advantage.double(), entropy).backward()
    want = [f64(p.grad) for p in twin.parameters()]
    for a, b in zip(got, want):          # float32 products of 64 x 64 numbers around it: 1e-5 of the largest entry
        np.testing.assert_allclose(f64(a), b, rtol=0, atol=1e-5 * np.abs(b).max())
    total = O.grad_norm(want)
    assert total > 0.05
    np.testing.assert_allclose(float(norm), total, rtol=1e-5)
    np.testing.assert_allclose(O.grad_norm([f64(q.grad) for q in net.parameters()]), 0.05, rtol=1e-4)


@pytest.mark.gpu
def test_update_captured_and_replayed(device):
    """Draw, evaluation with its gradient and clipping in one captured graph, while an eager autograd graph of the same logits
    lives: every replay, on new contents of the same buffers, equals the eager calls bit for bit."""
    g = rng_of("capture")
    rows, vocab = 257, 301
    logits = torch.randn(rows, vocab, generator=g).to(device).requires_grad_()
    u = torch.rand(rows, generator=g).to(device)
    gl, ge = (torch.randn(rows, generator=g).to(device) for _ in range(2))
    grads = grads_of(g, [3000, 17, 90_001], ["f32", "bf16", "f16"], device)
    eager_lp, _ = rl.evaluate_categorical(logits, torch.zeros(rows, dtype=torch.int64, device=device))   # stays alive

    def step():
        a, old = rl.sample_categorical(logits, u, top_p=0.9, temperature=0.9)
        lp, h, grad = rl.evaluate_categorical_grad(logits, a, gl, ge)
        out, norm = rl.clip_grads(grads + [grad], 0.7)
        return [a, old, lp, h, grad, norm] + out

    step()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        captured = step()
    for n in range(4):
        with torch.no_grad():
            logits.copy_(torch.randn(rows, vocab, generator=g))
            u.copy_(torch.rand(rows, generator=g))
            for t in grads:
                t.copy_(torch.randn(t.shape, generator=g) * (0.001, 0.1)[n % 2])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in captured]
        for i, (p, q) in enumerate(zip(seen, step())):
            assert torch.equal(p, q), (n, i)
        torch.cuda.synchronize()
    with torch.no_grad():
        logits.mul_(1.0)
    del eager_lp


@pytest.mark.gpu
def test_two_streams_at_once(device):
    """Calls of their own on two streams share nothing: each equals its result alone."""
    g = rng_of("streams")
    xs = [(torch.randn(300, 5000, generator=g) * 3).to(torch.bfloat16).to(device) for _ in range(2)]
    us = [torch.rand(300, generator=g).to(device) for _ in range(2)]
    grads = [grads_of(g, [100_003, 5], ["f32", "bf16"], device) for _ in range(2)]
    alone = [rl.sample_categorical(x, u, top_p=0.9) + (rl.clip_grads(q, 0.5)[1],) for x, u, q in zip(xs, us, grads)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(rl.sample_categorical(xs[i], us[i], top_p=0.9) + (rl.clip_grads(grads[i], 0.5)[1],))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(r, alone[i]))
