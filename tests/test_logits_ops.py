"""Log probabilities, entropy, top alternatives and distillation over rows of logits, against the
definitions in float64.

Tolerances.  With d = x - max and p the probabilities: a float32 difference is off by 2^-24 |d|, its
product with log2(e)/T by as much again, ex2 by 2^-22 relative, and a sum of n terms in sequence by
(n - 1) 2^-24; a thread adds at most n/32 + 64 terms of a row (n/256 in the long ones), so the sum
S is off by
    rel(S) = (n/32 + 64) 2^-24 + 2^-22 + 2^-22 sum p |d|.
What follows adds the rounding of each later operation; every factor is rounded up to a power of two.
"""
import ctypes

import numpy as np
import pytest

EPS = 2.0 ** -24


# ---------------------------------------------------------------------- float64 definitions
def shifted(x):
    x = x.astype(np.float64)
    m = x.max(axis=1, keepdims=True)
    m = np.where(np.isneginf(m), 0.0, m)
    return x - m


def softmax64(x, t=1.0):
    e = np.exp(shifted(x) / t)
    s = e.sum(axis=1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        return e / s, np.where(s > 0, shifted(x) / t - np.log(s), -np.inf)


def weighted(p, v):
    """sum p v over a row, with 0 * inf = 0."""
    return np.where(p > 0, p * np.where(p > 0, v, 0.0), 0.0).sum(axis=1, keepdims=True)


def rel_sum(x, t=1.0):
    p, _ = softmax64(x, t)
    return (x.shape[1] / 32 + 64) * EPS + 4 * EPS + 4 * EPS * weighted(p, np.abs(shifted(x)) / t)


def logprobs64(x):
    return softmax64(x)[1]


def tol_logprob(x, at):
    """For log p of the tokens `at` [rows, n]."""
    d = np.take_along_axis(np.where(np.isinf(shifted(x)), 0.0, shifted(x)), at, axis=1)
    log_s = np.log(np.maximum(np.exp(shifted(x)).sum(axis=1, keepdims=True), 1.0))
    return 2 * rel_sum(x) + 4 * EPS * (np.abs(d) + log_s)


def entropy64(x):
    p, lp = softmax64(x)
    return -weighted(p, lp)[:, 0]


def tol_entropy(x):
    p, _ = softmax64(x)
    far = weighted(p, np.abs(shifted(x)))
    log_s = np.log(np.maximum(np.exp(shifted(x)).sum(axis=1, keepdims=True), 1.0))
    square = weighted(p, shifted(x) ** 2)
    return (4 * rel_sum(x) * (1 + far) + 8 * EPS * (log_s + far + square))[:, 0]


def distill64(x, tokens, z, labels, t, w, g):
    """Loss, gradient and the tolerance of each."""
    rows, vocab = x.shape
    pt, lpt = softmax64(x, t)
    p, lp = softmax64(x)
    loss, grad = np.zeros(rows), np.zeros((rows, vocab))
    tol_l, tol_g = np.zeros(rows), np.zeros((rows, vocab))
    rs_t, rs = rel_sum(x, t)[:, 0], rel_sum(x)[:, 0]
    d = np.abs(np.where(np.isinf(shifted(x)), 0.0, shifted(x)))
    for r in range(rows):
        if np.all(np.isneginf(x[r])):
            continue
        if w > 0 and tokens is not None:
            here = [k for k in range(tokens.shape[1]) if 0 <= tokens[r, k] < vocab and z[r, k] != -np.inf]
            if here:
                zt = z[r, here].astype(np.float64) / t
                zt = zt - zt.max()
                lq = zt - np.log(np.exp(zt).sum())
                q = np.exp(lq)
                own = 8 * EPS * (np.abs(zt) + np.abs(z[r, here] / t))
                rel_q = (len(here) + 16) * EPS + own + weighted(q[None], own[None])[0, 0]
                for k, token in enumerate(tokens[r, here]):
                    if q[k] > 1e-37:
                        loss[r] += w * t * t * q[k] * (lq[k] - lpt[r, token])
                        tol_l[r] += w * t * t * q[k] * (
                            2 * rel_q[k] * (1 + abs(lq[k] - lpt[r, token])) + 2 * rs_t[r]
                            + 8 * EPS * (abs(lq[k]) + abs(z[r, here][k] / t) + d[r, token] / t
                                         + abs(lpt[r, token]))) if np.isfinite(lpt[r, token]) else 0.0
                    grad[r, token] -= g[r] * w * t * q[k]
                    tol_g[r, token] += abs(g[r]) * w * t * q[k] * (2 * rel_q[k] + 8 * EPS)
                grad[r] += g[r] * w * t * pt[r]
                tol_g[r] += abs(g[r]) * w * t * pt[r] * (2 * rs_t[r] + 8 * EPS * (d[r] / t + 2))
        if w < 1 and labels is not None and 0 <= labels[r] < vocab:
            loss[r] -= (1 - w) * lp[r, labels[r]]
            tol_l[r] += (1 - w) * (2 * rs[r] + 8 * EPS * (d[r, labels[r]] + abs(lp[r, labels[r]]))
                                   if np.isfinite(lp[r, labels[r]]) else 0.0)
            grad[r] += g[r] * (1 - w) * p[r]
            grad[r, labels[r]] -= g[r] * (1 - w)
            tol_g[r] += abs(g[r]) * (1 - w) * p[r] * (2 * rs[r] + 8 * EPS * (d[r] + 2))
            tol_g[r, labels[r]] += abs(g[r]) * (1 - w) * 8 * EPS
        # the last additions round the sum of the parts
        tol_g[r] += 4 * EPS * np.abs(grad[r]) + 1e-38
        tol_l[r] += 8 * EPS * abs(loss[r])
    return loss, grad, tol_l, tol_g


def close(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= tol
    return bool(np.all(same | near))


# ---------------------------------------------------------------------- calls
def run_logprobs(g, x, tokens=None, top=0, entropy=True, ld=None):
    rows, vocab = x.shape
    ld = vocab if ld is None else ld
    stored = np.full((rows, ld), np.float32(777.0))
    stored[:, :vocab] = x
    bx = g.Buffer.from_host(stored)
    n = 0 if tokens is None else tokens.shape[1]
    bt = g.Buffer.from_host_int32(tokens) if n else None
    lp = g.Buffer.empty(rows * n * 4) if n else None
    h = g.Buffer.empty(rows * 4) if entropy else None
    tt = g.Buffer.empty(rows * top * 4) if top else None
    tl = g.Buffer.empty(rows * top * 4) if top else None
    g.token_logprobs(bx, rows, vocab, tokens=bt, n_tokens=n, logprobs=lp, entropy=h, top_n=top, top_tokens=tt,
                     top_logprobs=tl, ld=ld)
    return (lp.retrieve((rows, n)) if n else None, h.retrieve((rows,)) if entropy else None,
            tt.retrieve_int32((rows, top)) if top else None, tl.retrieve((rows, top)) if top else None)


def run_distill(g, kind, x, tokens, z, labels, t, w, grad_loss=None, scale=1.0, ld=None, in_place=False):
    """Returns loss (None for the backward alone), stats and the whole stored gradient."""
    rows, vocab = x.shape
    ld = vocab if ld is None else ld
    stored = np.full((rows, ld), np.float32(777.0))
    stored[:, :vocab] = x
    bx = g.Buffer.from_host(stored)
    top = 0 if tokens is None else tokens.shape[1]
    bt = g.Buffer.from_host_int32(tokens) if top else None
    bz = g.Buffer.from_host(z) if top else None
    bl = g.Buffer.from_host_int32(labels) if labels is not None else None
    bg = g.Buffer.from_host(np.asarray(grad_loss, np.float32)) if grad_loss is not None else None
    loss, stats = g.Buffer.empty(rows * 4), g.Buffer.empty(rows * 12)
    grad = bx if in_place else g.Buffer.from_host(np.full((rows, ld), np.float32(555.0)))
    args = (bx, rows, vocab, bt, bz, top, bl, t, w)
    if kind == "step":
        g.distill_step(*args, loss=loss, grad=grad, grad_loss=bg, grad_scale=scale, ld=ld, ld_grad=ld)
        return loss.retrieve((rows,)), None, grad.retrieve((rows, ld))
    g.distill_forward(*args, loss=loss, stats=stats, ld=ld)
    if kind == "forward":
        return loss.retrieve((rows,)), stats.retrieve((rows, 3)), None
    g.distill_backward(*args, stats=stats, grad=grad, grad_loss=bg, grad_scale=scale, ld=ld, ld_grad=ld)
    return loss.retrieve((rows,)), stats.retrieve((rows, 3)), grad.retrieve((rows, ld))


def some_logits(rng, rows, vocab, masked=False):
    x = (2.0 * rng.standard_normal((rows, vocab))).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += np.float32(9.0)
    if masked:
        x[rng.random((rows, vocab)) < 0.2] = -np.inf
    return x


def some_teacher(rng, x, top):
    rows, vocab = x.shape
    tokens = np.stack([rng.permutation(vocab)[:top] for _ in range(rows)]).astype(np.int32)
    z = (3.0 * rng.standard_normal((rows, top))).astype(np.float32)
    return tokens, z, rng.integers(0, vocab, rows).astype(np.int32)


# ---------------------------------------------------------------------- CPU: refusals, bookkeeping
def refused(g, call, code):
    with pytest.raises(g.GonnError) as e:
        call()
    assert e.value.code == code and e.value.message, e.value


class Handle:
    """A handle that the library never issued: what it refuses before it looks at buffers."""
    handle = ctypes.c_void_p(0x1234)


def test_dimensions_are_refused_before_anything_else(built_lib):
    g, h = built_lib, Handle()
    for rows, vocab, ld, top in ((0, 8, 8, 1), (-1, 8, 8, 1), (4, 0, 8, 0), (4, 8, 7, 1), (4, 8, 8, 9), (4, 500, 500, 129),
                                 (4, 8, 8, -1), (4, 2 ** 31, 2 ** 31, 1), (2 ** 31, 8, 8, 1)):
        refused(g, lambda: g.token_logprobs(h, rows, vocab, entropy=h, top_n=top, top_tokens=h, top_logprobs=h,
                                            ld=ld), -3)
    refused(g, lambda: g.token_logprobs(h, 4, 8, tokens=h, n_tokens=-1, logprobs=h), -3)
    refused(g, lambda: g.token_logprobs(h, 4, 8, entropy=h), -2)


def test_distillation_parameters_are_refused_before_anything_else(built_lib):
    g, h = built_lib, Handle()
    nan, inf = float("nan"), float("inf")
    for t, w in ((0.0, 0.5), (-1.0, 0.5), (nan, 0.5), (inf, 0.5), (1e-7, 0.5), (1.0, -0.1), (1.0, 1.1), (1.0, nan)):
        refused(g, lambda: g.distill_forward(h, 4, 8, h, h, 2, h, t, w, loss=h), -3)
        refused(g, lambda: g.distill_step(h, 4, 8, h, h, 2, h, t, w, loss=h, grad=h), -3)
        refused(g, lambda: g.distill_backward(h, 4, 8, h, h, 2, h, t, w, stats=h, grad=h), -3)
    for scale in (nan, inf):
        refused(g, lambda: g.distill_step(h, 4, 8, h, h, 2, h, 1.0, 0.5, loss=h, grad=h, grad_scale=scale), -3)
    for rows, vocab, ld, top in ((0, 8, 8, 2), (4, 0, 0, 2), (4, 8, 7, 2), (4, 8, 8, 129), (4, 8, 8, -1)):
        refused(g, lambda: g.distill_forward(h, rows, vocab, h, h, top, h, 1.0, 0.5, loss=h, ld=ld), -3)
    refused(g, lambda: g.distill_step(h, 4, 8, h, h, 2, h, 1.0, 0.5, loss=h, grad=h, ld_grad=7), -3)
    refused(g, lambda: g.distill_forward(h, 4, 8, h, h, 2, h, 1.0, 0.5, loss=h), -2)


def test_float64_gradient_is_the_derivative_of_the_loss():
    """The gradient's formula against differences of the loss's, and q sums what a token named twice gets."""
    rng = np.random.default_rng(5)
    x = some_logits(rng, 3, 11).astype(np.float64)
    tokens = np.array([[1, 4, 4, 9], [0, 2, -1, 5], [7, 7, 7, 3]], np.int32)
    z = rng.standard_normal((3, 4)).astype(np.float32)
    labels = np.array([4, -1, 0], np.int32)
    g = np.array([0.5, 2.0, 1.0])
    for t, w in ((1.0, 0.3), (2.5, 1.0), (0.7, 0.0)):
        _, grad, _, _ = distill64(x, tokens, z, labels, t, w, g)
        for j in range(11):
            up, down = x.copy(), x.copy()
            up[:, j] += 1e-6
            down[:, j] -= 1e-6
            slope = (distill64(up, tokens, z, labels, t, w, g)[0] - distill64(down, tokens, z, labels, t, w, g)[0]) / 2e-6
            assert np.allclose(g * slope, grad[:, j], atol=1e-7)


# ---------------------------------------------------------------------- GPU: log probabilities
SIZES = [(1, 1), (1, 2), (3, 10), (5, 31), (4, 33), (7, 100), (2, 255), (2, 257), (300, 10), (3, 1000), (2, 1023),
         (3, 4097), (2, 12345), (1, 50001), (5, 32768), (1, 150001), (160, 2049), (700, 515),
         (40, 33000), (1, 600001)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("masked", [False, True])
def test_logprobs_entropy_and_alternatives(gpu, rows, vocab, masked):
    rng = np.random.default_rng(rows * 1000 + vocab)
    x = some_logits(rng, rows, vocab, masked and vocab > 1)
    x[:, 0] = np.float32(0.5)  # no row is masked as a whole
    tokens = rng.integers(0, vocab, (rows, 2)).astype(np.int32)
    top = min(vocab, 20)
    lp, h, tt, tl = run_logprobs(gpu, x, tokens, top)
    want = logprobs64(x)
    assert close(lp, np.take_along_axis(want, tokens, 1), tol_logprob(x, tokens))
    assert close(h, entropy64(x), tol_entropy(x))
    order = np.argsort(-x, axis=1, kind="stable")[:, :top].astype(np.int32)
    assert np.array_equal(tt, order)
    assert close(tl, np.take_along_axis(want, order, 1), tol_logprob(x, order))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [7, 128, 129, 1000, 8192, 70000])
@pytest.mark.parametrize("top", [1, 7, 64, 128])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "few values", "zeros of both signs", "all but few masked"])
def test_alternatives_of_hard_orders(gpu, vocab, top, kind):
    top = min(top, vocab)
    rng = np.random.default_rng(vocab + top)
    x = np.zeros((2, vocab), np.float32)
    if kind == "rising":
        x[:] = np.linspace(-20, 5, vocab)
    elif kind == "falling":
        x[:] = np.linspace(5, -20, vocab)
    elif kind == "few values":
        x[:] = rng.integers(0, 3, (2, vocab))
    elif kind == "zeros of both signs":
        x[:] = np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0)
    elif kind == "all but few masked":
        x[:] = -np.inf
        x[0, vocab // 2] = 3.0
        x[1, [0, vocab - 1]] = 1.0
    _, h, tt, tl = run_logprobs(gpu, x, None, top)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top].astype(np.int32)
    assert np.array_equal(tt, order)
    assert close(tl, np.take_along_axis(logprobs64(x), order, 1), tol_logprob(x, order))
    assert close(h, entropy64(x), tol_entropy(x))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 40, 3001, 40000])
def test_rows_that_are_masked_or_spoiled(gpu, vocab):
    """All masked, masked by the lowest float, the whole range of float, NaN, +inf, no token."""
    rng = np.random.default_rng(vocab)
    x = some_logits(rng, 8, vocab)
    low = np.finfo(np.float32).min
    x[0] = -np.inf
    x[1, 1:] = low
    x[2, :] = low
    x[3, 0], x[3, 1] = -low, low
    x[4, vocab // 2] = np.nan
    x[5, vocab - 1] = np.inf
    x[6, 1:] = -np.inf
    tokens = np.array([[1, -1]] * 8, np.int32)
    lp, h, tt, tl = run_logprobs(gpu, x, tokens, 3)
    assert lp[0, 0] == -np.inf and h[0] == 0 and list(tt[0]) == [0, 1, 2] and np.all(np.isneginf(tl[0]))
    assert np.all(lp[[0, 1, 2, 3, 6, 7], 1] == 0)
    for r in (4, 5):
        assert np.isnan(lp[r, 0]) and np.isnan(h[r]) and list(tt[r]) == [-1] * 3 and np.all(np.isnan(tl[r]))
    ok = [1, 2, 3, 6, 7]
    with np.errstate(over="ignore"):                      # row 3's difference is beyond float32
        want = logprobs64(x[ok]).astype(np.float32)
    assert close(lp[ok, :1], want[:, 1:2], tol_logprob(x[ok], tokens[ok, :1]))
    assert close(h[ok], entropy64(x[ok]), tol_entropy(x[ok]))
    assert np.array_equal(tt[ok], np.argsort(-x[ok], axis=1, kind="stable")[:, :3])


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary_are_reported(gpu):
    x = np.zeros((3, 9), np.float32)
    bx, bt = gpu.Buffer.from_host(x), gpu.Buffer.from_host_int32(np.array([[1], [9], [-7]], np.int32))
    lp = gpu.Buffer.empty(12)
    refused(gpu, lambda: gpu.token_logprobs(bx, 3, 9, tokens=bt, n_tokens=1, logprobs=lp), -3)
    got = lp.retrieve((3,))
    assert np.isnan(got[1]) and got[2] == 0 and abs(got[0] + np.log(9.0)) < 1e-6
    # the report was taken: the next call is clean; without blocking it waits for the synchronise
    gpu.token_logprobs(bx, 3, 9, entropy=lp)
    gpu.lib().gonngpu_set_blocking(0)
    try:
        gpu.token_logprobs(bx, 3, 9, tokens=bt, n_tokens=1, logprobs=lp)
        refused(gpu, gpu.synchronize, -3)
        gpu.synchronize()
    finally:
        gpu.lib().gonngpu_set_blocking(1)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,ld", [(10, 17), (1000, 1001), (4096, 4100), (33001, 33003)])
def test_row_pitch_and_offsets(gpu, vocab, ld):
    """Rows that start anywhere; the padding (777) must not be read."""
    rng = np.random.default_rng(ld)
    x = some_logits(rng, 5, vocab)
    tokens = rng.integers(0, vocab, (5, 3)).astype(np.int32)
    a = run_logprobs(gpu, x, tokens, 8)
    b = run_logprobs(gpu, x, tokens, 8, ld=ld)
    assert np.array_equal(a[2], b[2])
    assert close(b[0], np.take_along_axis(logprobs64(x), tokens, 1), tol_logprob(x, tokens))
    assert close(b[1], entropy64(x), tol_entropy(x))


@pytest.mark.gpu
def test_sizes_and_overlaps_are_refused(gpu):
    x, small = gpu.Buffer.empty(4 * 100 * 4), gpu.Buffer.empty(8)
    r4 = gpu.Buffer.empty(4 * 16)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 101, entropy=r4), -3)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 100, entropy=small), -3)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 100, entropy=x), -3)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 100, tokens=r4, n_tokens=1, logprobs=r4), -3)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 100, top_n=2, top_tokens=r4, top_logprobs=r4), -3)
    refused(gpu, lambda: gpu.token_logprobs(x, 4, 100, n_tokens=1, logprobs=r4), -2)
    st = gpu.Buffer.empty(48)
    refused(gpu, lambda: gpu.distill_forward(x, 4, 100, None, None, 0, None, 1.0, 1.0, loss=r4), -2)
    refused(gpu, lambda: gpu.distill_forward(x, 4, 100, None, None, 0, None, 1.0, 0.0, loss=r4), -2)
    refused(gpu, lambda: gpu.distill_forward(x, 4, 100, None, None, 0, r4, 1.0, 0.0, loss=small), -3)
    refused(gpu, lambda: gpu.distill_forward(x, 4, 100, None, None, 0, r4, 1.0, 0.0, loss=r4), -3)
    refused(gpu, lambda: gpu.distill_backward(x, 4, 100, None, None, 0, r4, 1.0, 0.0, stats=st, grad=st), -3)
    refused(gpu, lambda: gpu.distill_step(x, 4, 50, None, None, 0, r4, 1.0, 0.0, loss=st, grad=x, ld=100, ld_grad=50), -3)


# ---------------------------------------------------------------------- GPU: distillation
@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 10, 4), (5, 31, 31), (4, 100, 7), (300, 10, 3), (3, 1000, 64),
                                            (2, 4097, 128), (2, 12345, 20), (1, 50001, 64), (3, 32768, 33),
                                            (1, 150001, 16), (170, 515, 5),
                                            (40, 33000, 9), (1, 500003, 128)])
@pytest.mark.parametrize("t,w", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.25), (4.0, 0.0)])
@pytest.mark.parametrize("kind", ["forward", "backward", "step"])
def test_distillation(gpu, rows, vocab, top, t, w, kind):
    rng = np.random.default_rng(rows + vocab + top)
    x = some_logits(rng, rows, vocab)
    tokens, z, labels = some_teacher(rng, x, top)
    if rows > 2:
        labels[1] = -1
        tokens[2, (top + 1) // 2:] = -1
    g = rng.uniform(-2, 2, rows).astype(np.float32)
    loss, stats, grad = run_distill(gpu, kind, x, tokens, z, labels, t, w, grad_loss=g, scale=0.5)
    want, want_grad, tol, tol_g = distill64(x, tokens, z, labels, t, w, 0.5 * g.astype(np.float64))
    assert close(loss, want, tol)
    if stats is not None:
        d = shifted(x)
        assert np.array_equal(stats[:, 0], x.max(axis=1))
        assert close(stats[:, 1], np.exp(d / t).sum(axis=1), np.exp(d / t).sum(axis=1) * rel_sum(x, t)[:, 0])
        assert close(stats[:, 2], np.exp(d).sum(axis=1), np.exp(d).sum(axis=1) * rel_sum(x)[:, 0])
    if grad is not None:
        assert close(grad, want_grad, tol_g)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [6, 300, 5000, 70001])
@pytest.mark.parametrize("kind", ["backward", "step"])
def test_distillation_of_empty_and_spoiled_rows(gpu, vocab, kind):
    rng = np.random.default_rng(vocab)
    rows, top = 9, 4
    x = some_logits(rng, rows, vocab)
    tokens, z, labels = some_teacher(rng, x, top)
    x[0] = -np.inf                                        # nothing left of the student
    tokens[1], labels[1] = -1, -1                         # neither teacher nor label
    z[2] = -np.inf                                        # a teacher without mass, but a label
    tokens[3] = tokens[3, 0]                              # the same token four times
    labels[3] = tokens[3, 0]                              # and the label too
    x[4, tokens[4, 1]] = -np.inf                          # the teacher wants a masked token: loss inf
    x[5, (int(tokens[5].max()) + 1) % vocab] = np.nan
    z[6, 2] = np.nan
    x[7] = np.where(np.arange(vocab) < vocab // 2, np.finfo(np.float32).min, x[7])
    z[8, 1:] = -1e30                                      # a teacher that is certain
    loss, _, grad = run_distill(gpu, kind, x, tokens, z, labels, 2.0, 0.5)
    assert loss[0] == 0 and np.all(grad[0] == 0)
    assert loss[1] == 0 and np.all(grad[1] == 0)
    assert loss[4] == np.inf and np.all(np.isfinite(grad[4]))
    assert np.isnan(loss[5]) and np.all(np.isnan(grad[5]))
    assert np.isnan(loss[6]) and np.all(np.isnan(grad[6]))
    ok = [1, 2, 3, 7, 8]
    want, want_grad, tol, tol_g = distill64(x[ok], tokens[ok], z[ok], labels[ok], 2.0, 0.5, np.ones(len(ok)))
    # row 7's differences reach 3.4e38; only its gradient and a finite loss are compared
    fine = np.abs(want) < 1e30
    assert close(loss[ok][fine], want[fine], tol[fine])
    assert close(grad[ok], want_grad, np.nan_to_num(tol_g, nan=1e-6, posinf=1e-6))
    want4 = distill64(x[4:5], tokens[4:5], z[4:5], labels[4:5], 2.0, 0.5, np.ones(1))
    assert close(grad[4:5], want4[1], want4[3])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,ld", [(10, 13), (1000, 1024), (4097, 4099), (33000, 33004)])
@pytest.mark.parametrize("kind", ["backward", "step"])
def test_gradient_in_place_and_between_pitches(gpu, vocab, ld, kind):
    """In the logits' own place the gradient is the same, and what lies past the vocabulary stays."""
    rng = np.random.default_rng(vocab)
    x = some_logits(rng, 6, vocab)
    tokens, z, labels = some_teacher(rng, x, 5)
    _, _, apart = run_distill(gpu, kind, x, tokens, z, labels, 1.5, 0.7, scale=0.25)
    _, _, pitched = run_distill(gpu, kind, x, tokens, z, labels, 1.5, 0.7, scale=0.25, ld=ld)
    assert np.all(pitched[:, vocab:] == 555.0)
    _, want, _, tol = distill64(x, tokens, z, labels, 1.5, 0.7, np.full(6, 0.25))
    assert close(pitched[:, :vocab], want, tol)
    _, _, here = run_distill(gpu, kind, x, tokens, z, labels, 1.5, 0.7, scale=0.25, in_place=True)
    assert np.array_equal(here, apart)
    _, _, here = run_distill(gpu, kind, x, tokens, z, labels, 1.5, 0.7, scale=0.25, ld=ld, in_place=True)
    assert np.array_equal(here[:, :vocab], pitched[:, :vocab]) and np.all(here[:, vocab:] == 777.0)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["teacher", "label"])
def test_indices_outside_the_vocabulary_are_reported_and_left_out(gpu, what):
    rng = np.random.default_rng(3)
    x = some_logits(rng, 2, 50)
    tokens, z, labels = some_teacher(rng, x, 4)
    bad_tokens, bad_labels = tokens.copy(), labels.copy()
    if what == "teacher":
        bad_tokens[1, 2] = 50
        tokens[1, 2] = -1
    else:
        bad_labels[0] = 2 ** 31 - 1
        labels[0] = -1
    bx, bt, bz = gpu.Buffer.from_host(x), gpu.Buffer.from_host_int32(bad_tokens), gpu.Buffer.from_host(z)
    bl, loss, grad = gpu.Buffer.from_host_int32(bad_labels), gpu.Buffer.empty(8), gpu.Buffer.empty(400)
    refused(gpu, lambda: gpu.distill_step(bx, 2, 50, bt, bz, 4, bl, 1.0, 0.5, loss=loss, grad=grad), -3)
    want, want_grad, tol, tol_g = distill64(x, tokens, z, labels, 1.0, 0.5, np.ones(2))
    assert close(loss.retrieve((2,)), want, tol) and close(grad.retrieve((2, 50)), want_grad, tol_g)


@pytest.mark.gpu
def test_results_repeat_bit_for_bit(gpu):
    rng = np.random.default_rng(11)
    for rows, vocab in ((3, 60000), (400, 1000)):
        x = some_logits(rng, rows, vocab)
        tokens, z, labels = some_teacher(rng, x, 16)
        first = run_distill(gpu, "step", x, tokens, z, labels, 2.0, 0.5)
        lp = run_logprobs(gpu, x, tokens, 16)
        for _ in range(3):
            again = run_distill(gpu, "step", x, tokens, z, labels, 2.0, 0.5)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[2], again[2])
            for a, b in zip(lp, run_logprobs(gpu, x, tokens, 16)):
                assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["backward", "step", "forward", "logprobs"])
def test_long_runs_repeat_bit_for_bit(gpu, kind):
    """Rings under load, pass after pass: a stage that is given back before it has been read shows here."""
    rows, vocab, top, g = 2048, 32000, 16, gpu
    rng = np.random.default_rng(5)
    x = some_logits(rng, rows, vocab, masked=True)
    tokens, z, labels = some_teacher(rng, x, top)
    bx, bz = g.Buffer.from_host(x), g.Buffer.from_host(z)
    bt, bl = g.Buffer.from_host_int32(tokens), g.Buffer.from_host_int32(labels)
    loss, stats, grad = g.Buffer.empty(rows * 4), g.Buffer.empty(rows * 12), g.Buffer.empty(rows * vocab * 4)
    tt, tl = g.Buffer.empty(rows * top * 4), g.Buffer.empty(rows * top * 4)
    args = (bx, rows, vocab, bt, bz, top, bl, 2.0, 0.5)
    g.distill_forward(*args, loss=loss, stats=stats)

    def run():
        if kind == "backward":
            g.distill_backward(*args, stats=stats, grad=grad)
            return grad.retrieve((rows, vocab))
        if kind == "step":
            g.distill_step(*args, loss=loss, grad=grad)
            return grad.retrieve((rows, vocab))
        if kind == "forward":
            g.distill_forward(*args, loss=loss, stats=stats)
            return stats.retrieve((rows, 3))
        g.token_logprobs(bx, rows, vocab, tokens=bl, n_tokens=1, logprobs=loss, top_n=top, top_tokens=tt,
                         top_logprobs=tl)
        return np.concatenate([loss.retrieve((rows, 1)), tl.retrieve((rows, top))], axis=1)

    first = run()
    for _ in range(40):
        assert np.array_equal(run(), first, equal_nan=True)
    if kind in ("backward", "step"):
        for r in range(0, rows, 256):
            want = distill64(x[r:r + 8], tokens[r:r + 8], z[r:r + 8], labels[r:r + 8], 2.0, 0.5, np.ones(8))
            assert close(first[r:r + 8], want[1], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,t", [(200, 130001, 1.0), (400, 40000, 2.0), (320, 70003, 1.5), (700, 9000, 4.0)])
def test_steps_that_read_rows_twice(gpu, rows, vocab, t):
    """In place, beside the logits, and with rows at another distance from 16 bytes: the same gradient."""
    rng = np.random.default_rng(vocab)
    x = some_logits(rng, rows, vocab)
    tokens, z, labels = some_teacher(rng, x, 20)
    tokens[:, 7] = tokens[:, 3]
    labels[::3] = tokens[::3, 5]
    loss, _, grad = run_distill(gpu, "step", x, tokens, z, labels, t, 0.5)
    again, _, inside = run_distill(gpu, "step", x, tokens, z, labels, t, 0.5, in_place=True)
    assert np.array_equal(loss, again) and np.array_equal(grad, inside)
    bx, bt, bz, bl = (gpu.Buffer.from_host(x), gpu.Buffer.from_host_int32(tokens), gpu.Buffer.from_host(z),
                      gpu.Buffer.from_host_int32(labels))
    out, apart = gpu.Buffer.empty(rows * 4), gpu.Buffer.empty(rows * (vocab + 1) * 4)
    gpu.distill_step(bx, rows, vocab, bt, bz, 20, bl, t, 0.5, loss=out, grad=apart, ld_grad=vocab + 1)
    assert np.array_equal(out.retrieve((rows,)), loss)
    assert np.array_equal(apart.retrieve((rows, vocab + 1))[:, :vocab], grad)
    some = np.array([0, 1, rows // 2, rows - 1])
    want = distill64(x[some], tokens[some], z[some], labels[some], t, 0.5, np.ones(4))
    assert close(loss[some], want[0], want[2]) and close(grad[some], want[1], want[3])
