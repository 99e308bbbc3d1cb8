"""The policy-side operators at the ends of their ranges: rows of -inf, the smallest temperatures and weights, peaks over long tails,
the longest rows with masks and in large batches, tolerances derived from the kernels' own roundings.

U = 2^-24 is half a step of float32; helpers and the float64 definitions are those of test_policy_ops.py."""
import math

import numpy as np
import pytest
import torch

import isaaclab_amd._lib as L
from isaaclab_amd import rl
from oracle import policy_np as O
from test_policy_ops import DT, U, check_draw, check_evaluation, f64, f32v, rng_of, run_evaluation


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [60, 700, 3000, 9001, 131072])
def test_draw_peaks_over_long_tails(device, vocab):
    """The border lies in a tail whose entries weigh less than 2^-32 of the row: found by a few cuts (the host program of
    test_border_search.py counts them)."""
    g = rng_of("peak", vocab)
    x = torch.randn(6, vocab, generator=g) * 0.1
    for r, peak in enumerate((10.0, 15.0, 20.0, 22.8, 23.0, 30.0)):
        x[r, vocab // 3 + r] = peak
    x = x.to(device)
    for p in (0.9999, 0.99995, 0.99999, 1 - 2.0 ** -23):
        u = (1 - torch.rand(6, generator=g) * 1e-5).to(device)        # draws from the tail
        check_draw(x, u, rl.sample_categorical(x, u, top_p=p), top_p=p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 5, 700, 9001])
def test_evaluation_of_rows_of_minus_infinity(device, dtype, vocab):
    """A row that holds nothing but -inf where it is allowed: an action in range is one that is not allowed, log_prob -inf, as in
    a row that a mask empties; entropy and gradient 0."""
    x = torch.full((5, vocab), -math.inf, dtype=DT[dtype], device=device)
    a = torch.tensor([0, vocab - 1, vocab // 2, -1, vocab], device=device)
    one = torch.ones(5, device=device)
    some = torch.rand(5, vocab, generator=rng_of("allowed", vocab)).to(device) < 0.5
    behind = torch.where(some, x, torch.zeros_like(x))                 # what is not allowed is finite
    for y, mask in ((x, None), (x, torch.ones_like(some)), (x, some), (behind, some)):
        lp, h, grad = run_evaluation(y, a, one, one, mask=mask)
        check_evaluation(y, a, lp, h, grad, one, one, mask=mask)
        assert lp[:4].tolist() == [-math.inf] * 3 + [0.0] and bool(lp[4].isnan())
        assert h.tolist() == [0.0] * 5 and not bool(grad[:4].any())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 700, 9001])
def test_evaluation_below_the_smallest_normal_temperature(device, vocab):
    x = torch.randn(5, vocab, generator=rng_of("none", vocab)).to(device)
    t = torch.tensor([2.0 ** -127, 1e-39, 1e-45, 0.0, -0.0], device=device)
    a, one = x.argmax(1), torch.ones(5, device=device)
    for v in run_evaluation(x, a, one, one, temperature=t):
        assert bool(v.isnan().all())
    with pytest.raises(ValueError, match="temperature"):
        rl.evaluate_categorical(x, a, temperature=2.0 ** -127)


def roundings(x, a, lp, h, grad, gl, ge, mask, t, moves):
    """One row (float64) against its definition, within what the kernels' own roundings allow.  Per entry and unit of U:
      exponent   (x - max), 1 / T, log2(e) / T (constant and product), their product: 5 |d|, d = (x - max) / T
      weight     2^x to one step: 2;  sums of a chunk of at most 8: 7;  beyond it in 64 bits;  each change of a thread's largest
                 entry multiplies what it has by another 2^x: 2 each, at most `moves`
      s          5 E|d| + 10 + 2 moves (p-weighted mean; the last 1 is its rounding to 32 bits);  ln s: that and 4 of itself (logf)
      t / s      5 E d^2 + (17 + 2 moves) E|d| + E|d| (what s is off)
      H          ln s - t / s: both, and 1 of itself
      log_prob   3 |d_a|, ln s, 1 of itself
      gradient   p: its exponent 4 |d|, log2 s as ln s and 2 more of itself, 1 of ln p, 2 for 2^x;  gl + ge (ln p + H): ge times what
                 ln p and H are off, 4 of each term;  1 / T: 1;  gl / T at the action: 2;  the result's own rounding
    and a tenth more for products of these.  Above T = 8.5e37, 1 / T is a denormal: T 2^-126 more wherever it enters (half a step,
    2^-150, of 1 / T, in units of U), and half a step of what is made of it: gl + ge H and ge |log2 p| over T, their sum, gl / T, the
    sum of that and the action's own.  A p below 2^-126 is 0 in 32 bits: what it would give, its terms over T, is lost."""
    ok = np.ones(len(x), bool) if mask is None else mask
    want = O.evaluate_row(x, a, mask, t, gl, ge)
    d = np.where(ok, (x[ok].max() - np.where(ok, x, 0.0)) / t, 0.0)
    w = np.where(ok, np.exp(-d), 0.0)
    s = w.sum()
    p, ln_s = w / s, math.log(s)
    ln_p = np.where(ok, -d - ln_s, 0.0)
    mean, square = (p * d).sum(), (p * d * d).sum()
    more = t * 2.0 ** -126
    off_s = (5 + more) * mean + 10 + 2 * moves
    off_ln = off_s + 4 * ln_s
    off_h = off_ln + (5 + more) * square + (17 + more + 2 * moves) * mean + mean * off_s + abs(want[1])
    u = 1.1 * U
    assert abs(lp - want[0]) <= u * ((3 + more) * d[a] + off_ln + abs(want[0])) + 1e-30, (lp, want[0])
    assert abs(h - want[1]) <= u * off_h + 1e-30, (h, want[1])
    off_lnp = (4 + more) * d + off_ln + 2 * ln_s + np.abs(ln_p)
    terms = abs(gl) + abs(ge) * (np.abs(ln_p) + abs(want[1]))
    tol = p * ((off_lnp + 2) * np.abs(gl + ge * (ln_p + want[1])) + abs(ge) * (off_lnp + off_h) + (5 + more) * terms) * u / t
    tol[a] += (2 + more) * u * abs(gl) / t
    tol += 2.0 ** -150 * p * (2 + np.abs(ln_p) / math.log(2))
    tol[a] += 2.0 ** -149
    tol += 2.0 ** -126 * terms / t
    return want, tol


def check_roundings(x, a, lp, h, grad, gl, ge, mask=None, temperature=1.0, moves=0):
    step = torch.finfo(grad.dtype).eps / 2
    floor = torch.finfo(grad.dtype).smallest_normal * torch.finfo(grad.dtype).eps / 2
    xs, gs, lps, hs, gls, ges = f64(x), f64(grad), f64(lp), f64(h), f64(gl), f64(ge)
    for r in range(len(xs)):
        want, tol = roundings(xs[r], int(a[r]), lps[r], hs[r], gs[r], gls[r], ges[r],
                              None if mask is None else mask[r].cpu().numpy(),
                              f64(temperature)[r] if isinstance(temperature, torch.Tensor) else f32v(temperature), moves)
        tol = tol + step * np.abs(want[2]) * 1.01 + floor
        err = np.abs(gs[r] - want[2])
        assert (err <= tol).all(), (r, err.max(), tol[(err - tol).argmax()])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [9, 700, 9001])
def test_evaluation_at_the_smallest_temperatures(device, dtype, vocab):
    """Down to the smallest normal number the definition holds, with logits that lie as near to each other: gradients are of the
    order of 1 / T, and 0 where the probability is.  Below it, as for a single number, a temperature is none: NaN."""
    g = rng_of("cold evaluation", dtype, vocab)
    t = torch.tensor([2.0 ** -126, 1.2e-38, 2e-38, 1e-37, 1e-36, 1e-30])
    x = (-torch.rand(6, vocab, generator=g) * 2000 * t[:, None]).to(DT[dtype])
    a = torch.randint(0, vocab, (6,), generator=g)
    a[::2] = x.float().argmax(1)[::2]
    gl, ge = (torch.rand(6, generator=g) * 2 - 1 for _ in range(2))
    x, a, gl, ge, t = (v.to(device) for v in (x, a, gl, ge, t))
    moves = 0 if vocab < 1000 else 6
    check_roundings(x, a, *run_evaluation(x, a, gl, ge, temperature=t), gl, ge, temperature=t, moves=moves)
    mask = torch.rand(6, vocab, generator=g).to(device) < 0.7
    mask.scatter_(1, a[:, None], True)
    check_roundings(x, a, *run_evaluation(x, a, gl, ge, temperature=t, mask=mask), gl, ge, mask=mask, temperature=t, moves=moves)
    # an action that is certain: nothing is left of a gradient whose terms are beyond float32
    sure = torch.full((2, vocab), -1.0, dtype=DT[dtype], device=device)
    sure[:, 3] = 1.0
    three, five = torch.full((2,), 3, device=device), torch.tensor([5.0, -40.0], device=device)
    lp, h, grad = run_evaluation(sure, three, five, five, temperature=t[:2])
    assert not bool(lp.any()) and not bool(h.any()) and not bool(grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32, torch.bool])
def test_draw_top_k_of_any_integer_type(device, kind):
    g = rng_of("kinds")
    x, u = torch.randn(5, 300, generator=g).to(device), torch.rand(5, generator=g).to(device)
    k = torch.tensor([0, 1, 3, 7, 120]).to(kind)
    check_draw(x, u, rl.sample_categorical(x, u, top_k=k.to(device)), top_k=k.to(torch.int64))


@pytest.mark.gpu
def test_draw_refuses_fractions_of_entries(device):
    """A top_k for each row is of whole numbers, as the one for all rows: their type says so."""
    x, u = torch.zeros(2, 3, device=device), torch.zeros(2, device=device)
    for k in (torch.tensor([2.5, 1.0], device=device), torch.ones(2, dtype=torch.bfloat16, device=device)):
        with pytest.raises(ValueError, match="whole number"):
            rl.sample_categorical(x, u, top_k=k)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 200, 700, 3000, 9000, 40000])
def test_draw_of_the_smallest_weights(device, vocab):
    """u = 0 draws the first kept entry, however light: its log-probability keeps 32 bits where its weight, below 2^-1022, does not."""
    d = torch.tensor([-700.0, -708.0, -712.3, -725.1, -735.0, -743.0])
    x = torch.full((6, vocab), -2000.0)
    x[:, 1] = d
    x[:, vocab - 1] = 0.0
    x, u = x.to(device), torch.zeros(6, device=device)
    for s in (dict(), dict(top_k=2), dict(temperature=0.5)):
        t = s.get("temperature", 1.0)
        a, lp = rl.sample_categorical(x * t, u, **s)
        assert a.tolist() == [1] * 6
        np.testing.assert_allclose(f64(lp), f64(x[:, 1]), rtol=2 * U)              # ln(1 + e^-700) is 0
    x[:, 0] = math.nan
    a, lp = rl.sample_categorical(x, u)
    assert a.tolist() == [-1] * 6 and bool(lp.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_grad_sums_do_not_depend_on_the_address(device, dtype, kind):
    """The same values behind an odd offset give the same partial sums, bit for bit."""
    n = 5 * 4096 + 77
    x = (torch.randn(n, generator=rng_of("address", dtype)) * 0.1).to(DT[dtype]).to(device)
    sums = []
    for shift in range(9):
        base = torch.zeros(n + 16, dtype=DT[dtype], device=device)
        y = base[shift:shift + n].copy_(x)
        work = torch.zeros(L.lib.mdp_grad_workspace(1), dtype=torch.float64, device=device)
        norm = torch.zeros((), device=device)
        table = (L.MdpGrad * 1)(L.MdpGrad(y.data_ptr(), None, n, L.DTYPES[y.dtype], 0))
        L.launch(L.lib.mdp_grad_norm, 0, table, 1, kind, work.data_ptr(), norm.data_ptr())
        sums.append(work[:7].clone())                   # six partial sums and what they join to
    want = f64(x)
    want = np.abs(want).max() if kind == 0 else np.abs(want).sum() if kind == 1 else (want ** 2).sum()
    np.testing.assert_allclose(sums[0][6].item(), want, rtol=n * 2.0 ** -53)
    assert all(torch.equal(s, sums[0]) for s in sums[1:])


@pytest.mark.gpu
def test_results_outside_autograd(device):
    """evaluate_categorical_grad and clip_grads work on values: what they are given may require a gradient, what they give has none."""
    g = rng_of("outside")
    x = torch.randn(4, 30, generator=g).to(device).requires_grad_()
    a = torch.randint(0, 30, (4,), generator=g).to(device)
    gl, ge = (torch.randn(4, generator=g).to(device).requires_grad_() for _ in range(2))
    got = rl.evaluate_categorical_grad(x, a, gl, ge)
    out, norm = rl.clip_grads([x], 0.5)
    for p, q in zip(got, rl.evaluate_categorical_grad(x.detach(), a, gl.detach(), ge.detach())):
        assert not p.requires_grad and torch.equal(p, q)
    assert not norm.requires_grad and not out[0].requires_grad
    assert torch.equal(out[0], rl.clip_grads([x.detach()], 0.5)[0][0])


@pytest.mark.gpu
def test_clip_with_an_infinite_bound(device):
    """An infinite bound measures the norm and leaves finite gradients as they are; over an infinite norm it is no number."""
    x = torch.randn(5000, generator=rng_of("unbounded")).to(device)
    out, norm = rl.clip_grads([x], math.inf)
    assert torch.equal(out[0], x) and bool(norm.isfinite())
    y = x.clone()
    y[77] = math.inf
    out, norm = rl.clip_grads([y], math.inf)
    assert float(norm) == math.inf and bool(out[0].isnan().all())


@pytest.mark.gpu
def test_ratio_of_an_unchanged_policy(device):
    """What is drawn uncut, with the temperature and the mask that it is evaluated with, has the ratio 1: the documented update.  A
    draw that top_p cuts has the log-probability of what is left, so the ratio is the kept mass."""
    g = rng_of("ratio")
    logits = (torch.randn(64, 12, 33, generator=g) * 2).to(device)
    allowed = torch.rand(64, 12, 33, generator=g).to(device) < 0.8
    u = torch.rand(64, 12, generator=g).to(device)
    actions, old = rl.sample_categorical(logits, u, temperature=0.9, mask=allowed)
    log_prob, _ = rl.evaluate_categorical(logits, actions, temperature=0.9, mask=allowed)
    # three roundings of d = (x - max) / T below 2 * 9 / 0.9, and the sum's: see test_evaluation_within_its_roundings
    np.testing.assert_allclose(f64(log_prob - old), 0.0, atol=U * 250)
    actions, old = rl.sample_categorical(logits, u, temperature=0.9, top_p=0.7, mask=allowed)
    log_prob, _ = rl.evaluate_categorical(logits, actions, temperature=0.9, mask=allowed)
    ratio = f64(torch.exp(log_prob - old))
    assert ratio.min() >= f32v(0.7) - 1e-5 and (ratio < 1.0).mean() > 0.9


LARGE = [dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.8, temperature=0.7), dict(min_p=0.05), dict(top_k=200),
         dict(top_p=0.99, temperature=3.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype, vocab", [("f32", 4101), ("f32", 16380), ("bf16", 8203), ("bf16", 32001), ("f16", 9000), ("f16", 32750)])
def test_draw_large_batches_of_long_rows(device, dtype, vocab, masked):
    """512 rows and more of 1025 to 4096 chunks are drawn by blocks of 256 threads."""
    g = rng_of("many long", dtype, vocab)
    rows = 515
    x = (torch.randn(rows, vocab, generator=g) * torch.rand(rows, 1, generator=g) * 4).to(DT[dtype]).to(device)
    u = torch.rand(rows, generator=g).to(device)
    mask = (torch.rand(rows, vocab, generator=g) < torch.rand(rows, 1, generator=g)).to(device) if masked else None
    pick = torch.cat([torch.arange(0, rows, 41), torch.tensor([1, rows - 1])]).to(device)
    per_row = dict(temperature=(torch.rand(rows, generator=g) * 2).to(device), top_k=torch.randint(0, 300, (rows,), generator=g).to(device),
                   top_p=(torch.rand(rows, generator=g) * 1.2).to(device))
    for s in LARGE + [per_row]:
        a, lp = rl.sample_categorical(x, u, mask=mask, **s)
        part = {k: v[pick] if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        check_draw(x[pick], u[pick], (a[pick], lp[pick]), mask=None if mask is None else mask[pick], **part)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, vocab", [("f32", 16390), ("f32", 70001), ("bf16", 32771), ("bf16", 140003), ("f16", 50001)])
def test_draw_longest_rows_with_masks(device, dtype, vocab):
    """Rows of more than 4096 chunks, masked: at random, all but a few, everything, at the chunks' edges."""
    g = rng_of("long masked", dtype, vocab)
    x = (torch.randn(7, vocab, generator=g) * 2).to(DT[dtype])
    mask = torch.rand(7, vocab, generator=g) < torch.tensor([0.7, 0.01, 0.5, 0.5, 1.0, 0.0, 0.9])[:, None]
    mask[3, :vocab // 2] = False
    mask[4, ::8] = False
    x[2, ~mask[2]] = math.nan
    x, mask = x.to(device), mask.to(device)
    u = torch.rand(7, generator=g).to(device)
    wide = torch.zeros(7, vocab + 3, dtype=torch.bool, device=device)
    wide[:, 3:] = mask                                   # the same at an odd offset
    for s in LARGE:
        for m in (mask, wide[:, 3:]):
            check_draw(x, u, rl.sample_categorical(x, u, mask=m, **s), mask=m, **s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [2, 19, 64, 255, 1024, 2050, 5003, 33001, 131075, 1000003])
def test_evaluation_within_its_roundings(device, dtype, vocab):
    """A thread's largest entry changes at most once in 1024 chunks, once at the row's edges and once when the waves join."""
    g = rng_of("roundings", dtype, vocab)
    chunk = 128 // torch.finfo(DT[dtype]).bits
    moves = 0 if vocab <= 512 * chunk - chunk else vocab // (1024 * chunk) + 3
    for n, t in enumerate((1.0, 0.6, 2.5)):
        rows = 16 if vocab < 3000 else 2
        x = (torch.randn(rows, vocab, generator=g) * (0.5, 3.0, 8.0)[n]).to(DT[dtype]).to(device)
        a = torch.randint(0, vocab, (rows,), generator=g).to(device)
        gl, ge = (torch.randn(rows, generator=g).to(device) for _ in range(2))
        check_roundings(x, a, *run_evaluation(x, a, gl, ge, temperature=t), gl, ge, temperature=t, moves=moves)
        mask = torch.rand(rows, vocab, generator=g).to(device) < 0.6
        mask.scatter_(1, a[:, None], True)
        check_roundings(x, a, *run_evaluation(x, a, gl, ge, temperature=t, mask=mask), gl, ge, mask=mask, temperature=t, moves=moves)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_evaluation_sums_what_32_bits_would_lose(device, dtype):
    """8192 large entries, then four million that weigh 7e-8 to 1.5e-8 of one each: 584 to 130 U of the sum, which a thread that added
    them up one by one in 32 bits, 32 large ones first, would lose; the tolerance is about 60 U.  No thread's largest entry changes
    behind its first."""
    vocab, first = (1 << 22) + 5, 8192
    x = torch.zeros(3, vocab, dtype=DT[dtype])
    for r, low in enumerate((-16.5, -17.25, -18.0)):
        x[r, first:] = low
    x = x.to(device)
    a = torch.tensor([0, first, vocab - 1], device=device)
    gl, ge = torch.tensor([1.0, -2.0, 0.5], device=device), torch.tensor([0.5, 1.0, -1.0], device=device)
    check_roundings(x, a, *run_evaluation(x, a, gl, ge), gl, ge)


@pytest.mark.gpu
def test_gradient_of_a_very_long_flat_row(device):
    """3.3e7 equal entries: gl (delta - 1 / V); the entropy of a flat row is at its maximum, its gradient 0.  Its two terms, ln p and
    H = ln V, cancel within their roundings: 4 ln V of ln s, 2 and 1 more of it, 12 of the sum, in either, and 4 of each product."""
    vocab = (1 << 25) + 77
    x = torch.zeros(1, vocab, device=device)
    gl, ge = torch.tensor([3.0], device=device), torch.tensor([-2.0], device=device)
    for at in (0, 12345, vocab - 1):
        a = torch.tensor([at], device=device)
        lp, h, grad = rl.evaluate_categorical_grad(x, a, gl, ge)
        ln = math.log(vocab)
        tol = U / vocab * (3.0 * (7 * ln + 20) + 2.0 * (2 * (7 * ln + 20) + 8 * ln))
        rest = f64(grad)[0]
        assert abs(rest[at] - 3.0 * (1 - 1 / vocab)) <= tol + 3 * 2 * U
        rest = np.delete(rest, at)
        assert np.abs(rest + 3.0 / vocab).max() <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("seed", ["seed_samplers", "manual_seed"])
def test_seeding_behind_a_capture(device, seed):
    """A captured draw goes on with the device's generator, whatever it is seeded with later, and writes to nothing else."""
    from isaaclab_amd.utils import math as M

    x = torch.zeros(5000, 50, device=device)
    M.seed_samplers(5, device)

    def reseed(n):
        if seed == "seed_samplers":
            return M.seed_samplers(n, device)
        M._sampler_seed[0] = -1                         # a state that follows torch's seed, as it does until seed_samplers
        torch.manual_seed(n)

    reseed(6)
    rl.sample_categorical(x)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = rl.sample_categorical(x)[0]
    reseed(7)
    eager = [rl.sample_categorical(x)[0] for _ in range(3)]
    reseed(7)
    first = rl.sample_categorical(x)[0]
    others = [torch.zeros(2, dtype=torch.int64, device=device) for _ in range(64)]       # where a state might have been
    assert torch.equal(first, eager[0])
    for n in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[n])
    assert not any(bool(t.any()) for t in others)
    with torch.inference_mode():
        reseed(8)
        inside = rl.sample_categorical(x)[0]
    reseed(8)
    assert torch.equal(rl.sample_categorical(x)[0], inside)
    M.seed_samplers(1, device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [9, 700, 3000, 9001, 40000])
def test_logits_further_apart_than_the_largest_number(device, dtype, vocab):
    """Logits of both signs near the ends of the range, at temperatures that bring them together again: their differences are beyond
    32 bits, what is drawn and evaluated is not."""
    g = rng_of("ends", dtype, vocab)
    top = torch.finfo(DT[dtype]).max
    x = ((torch.rand(6, vocab, generator=g) * 2 - 1) * top).to(DT[dtype])
    x[:, 0], x[:, 1] = -top, top
    a = torch.randint(0, vocab, (6,), generator=g)
    a[0], a[1] = 0, 1
    u = torch.rand(6, generator=g)
    gl, ge = (torch.randn(6, generator=g) for _ in range(2))
    x, a, u, gl, ge = (v.to(device) for v in (x, a, u, gl, ge))
    moves = 0 if vocab < 2000 else vocab // 4096 + 3
    for t in (3e38, 1e38, 1e37):
        for s in (dict(), dict(top_p=0.9), dict(top_k=vocab // 2), dict(min_p=0.1)):
            check_draw(x, u, rl.sample_categorical(x, u, temperature=t, **s), temperature=t, **s)
        check_roundings(x, a, *run_evaluation(x, a, gl, ge, temperature=t), gl, ge, temperature=t, moves=moves)
    assert rl.evaluate_categorical(x, a, temperature=1.0)[0][0].item() == -math.inf
