"""Token scoring and distillation on the GPU against oracle/objectives.py (float64, from the formulas).

Bars, with u = 2^-24 (half a step of float32), lp in nats, n_add = the longest chain of float32 additions behind a sum:
  * S = sum 2^y carries n_add u from adding, and per term 2 |y| u ln 2 (y = c (z - m) is rounded, c too) + 2 u (exp2); what a term
    with a large |y| adds is weighted by 2^y, so the mean of |y| over the terms is at most log2 V < 22:  |dS / S| <= (n_add + 48) u.
  * lp = (y - log2 S) ln 2:  |d| <= (n_add + 48 + 22 + 4 |lp|) u   (the rounding of log2 S <= log2 V is 22 u)
  * H = (log2 S - W / S) ln 2, |W / S| <= log2 V:  |d| <= (n_add + 70) (1 + log2 V) u
  * gradient: each term carries the relative error of its p, (n_add + 70 + 4 |lp|) u, and the sum is rounded to the type once:
    |d| <= (n_add + 80 + 4 |lp|) u * (sum of the terms' sizes) + eps_type / 2 |grad| + half the type's smallest step.
    4 |lp| p u is largest at p = 1/e and below 2 u.
  * loss: alpha tau^2 sum q (log q - lp): q has relative error (64 + 70 + ...) u, so each factor's error is bounded by
    (n_add + 160 + 4 (|lp| + |log q|)) u times alpha tau^2 q, plus the label's (1 - alpha) lp.
n_add: no kernel adds more than V / 256 terms in a row before it joins 256 or more partial sums in a tree (<= 16 + 64 deep).
"""
import numpy as np
import pytest
import torch

from oracle import objectives as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def n_add(V):
    return V / 256 + 80


def randn(shape, dtype, seed, scale=3.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g) + offset).to(dtype)


def np64(t):
    return t.detach().cpu().double().numpy()


def check_scores(got, z, labels, k, temperature=1.0):
    V = z.shape[-1]
    z2, y2 = np64(z).reshape(-1, V), None if labels is None else np64(labels).reshape(-1).astype(np.int64)
    lp, h, ids, top = O.token_logprobs(z2, y2, k, temperature)
    if labels is not None:
        d = np64(got.logprobs).reshape(-1)
        same(d, lp, (n_add(V) + 70 + 4 * np.abs(lp)) * U, "logprobs")
    if got.entropy is not None:
        same(np64(got.entropy).reshape(-1), h, np.full(len(h), (n_add(V) + 70) * (1 + np.log2(V + 1)) * U), "entropy")
    if k:
        assert np.array_equal(got.top_ids.cpu().numpy().reshape(-1, k), ids)
        same(np64(got.top_logprobs).reshape(-1, k), top, (n_add(V) + 70 + 4 * np.abs(top)) * U, "top_logprobs")


def same(got, want, tol, name):
    """NaN and infinities where the oracle has them, everything else within tol."""
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), name
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), name
    off = np.abs(got[fin] - want[fin]) - tol[fin]
    assert off.size == 0 or off.max() <= 0, (name, float(off.max()), float(np.abs(got[fin] - want[fin]).max()))


def check_grad(got, want, size, dtype, V, extra=1.0):
    info = torch.finfo(dtype)
    g = np64(got).reshape(-1, V)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126       # below it the type has no steps / the kernel flushes
    tol = (n_add(V) + 82) * U * size * extra + info.eps / 2 * np.abs(want) * (1 + 2 ** -10) + tiny
    same(g, want, tol, "grad")


SHAPES = [(1, 1), (3, 2), (5, 3), (4, 7), (2, 8), (3, 9), (2, 63), (2, 64), (3, 65), (2, 127), (2, 255), (2, 1000), (3, 1025),
          (2, 4099), (2, 8192), (3, 10000), (2, 16385), (3, 32000), (5, 50021), (2, 65537), (1, 131073), (1, 200019)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, V", SHAPES)
def test_scores(rows, V, dtype):
    from speech_to_text_amd import token_logprobs
    z = randn((rows, V), TYPES[dtype], 10 * V + rows)
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(V))
    if rows > 2:
        y[1] = -100
    for k in sorted({0, 1, min(V, 5), min(V, 16), min(V, 64)}):
        got = token_logprobs(z.to(DEV), y.to(DEV), top_k=k, entropy=True)
        check_scores(got, z, y, k)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [1, 2, 7, 64, 255, 300, 1100])
def test_many_rows(rows, dtype):
    """From a single decoding step to batches, with padding positions; int32 labels."""
    from speech_to_text_amd import token_logprobs
    V = 1009
    z = randn((rows, V), TYPES[dtype], rows, scale=2.0, offset=30.0)
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(rows), dtype=torch.int32)
    y[torch.arange(rows) % 5 == 3] = -100
    got = token_logprobs(z.to(DEV), y.to(DEV), top_k=12, entropy=True, temperature=0.7)
    check_scores(got, z, y, 12, 0.7)


@pytest.mark.parametrize("T", [0.25, 1.0, 2.0, 3.0, 10.0])
def test_temperature_and_no_labels(T):
    from speech_to_text_amd import token_logprobs
    z = randn((3, 5003), torch.bfloat16, 3, scale=4.0, offset=-50.0)
    got = token_logprobs(z.to(DEV), top_k=9, entropy=True, temperature=T)
    assert got.logprobs is None
    check_scores(got, z, None, 9, T)
    only = token_logprobs(z.to(DEV), entropy=True, temperature=T)
    assert only.top_ids is None and torch.equal(only.entropy, got.entropy)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_row_strides_and_alignment(dtype):
    """Slices of positions, batches of a larger vocabulary (rows at every alignment), an expanded batch, more dimensions."""
    from speech_to_text_amd import token_logprobs
    t = TYPES[dtype]
    base = randn((4, 7, 1037), t, 8).to(DEV)
    y = torch.randint(0, 900, (4, 7), generator=torch.Generator().manual_seed(2)).to(DEV)
    for z, lab in ((base[:, :-1], y[:, :-1]), (base[:, 1:], y[:, 1:]), (base[..., 3:1003], y), (base[..., 5:6], y * 0),
                   (base[1:, 2:, 1:1000], y[1:, 2:]), (base[:1].expand(4, 7, 1037), y), (base[:, :1].expand(4, 7, 1037), y),
                   (base.transpose(0, 1), y.T), (base[0, 0], y[0, 0]), (base.view(2, 2, 7, 1037), y.view(2, 2, 7)),
                   (base[::2, ::3], y[::2, ::3])):
        k = min(6, z.shape[-1])
        got = token_logprobs(z, lab, top_k=k, entropy=True)
        assert got.logprobs.shape == lab.shape and got.top_ids.shape == lab.shape + (k,)
        check_scores(got, z.reshape(-1, z.shape[-1]), lab.reshape(-1), k)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [37, 4099, 50021, 131073])
def test_masked_and_special_rows(V, dtype):
    """-inf among others, alone, everywhere; the type's lowest value; NaN; +inf; equal values; sorted rows."""
    from speech_to_text_amd import token_logprobs
    t = TYPES[dtype]
    low = torch.finfo(t).min
    z = randn((16, V), t, V)
    z[0, ::2] = -np.inf
    z[1] = -np.inf
    z[1, V // 3] = 2.0                           # one token left: probability 1, entropy 0
    z[2] = -np.inf                               # none left
    z[3] = low                                   # all masked by the lowest value: uniform
    z[4] = low
    z[4, V - 1] = 1.0
    z[5, 7] = np.nan
    z[6, 5] = np.inf
    z[7] = 1.5                                   # all equal: the first indices
    z[8] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(t)      # +0 and -0 are equal
    z[9] = torch.linspace(-8, 8, V).to(t)        # rising: the largest are neighbours
    z[10] = torch.linspace(8, -8, V).to(t)
    z[11] = -np.inf
    z[11, :3] = torch.tensor([0.0, 1.0, 1.0]).to(t)      # fewer finite tokens than alternatives
    z[12] = np.nan
    z[13, :] = 0.0
    z[13, min(V - 1, 20):min(V, 30)] = 4.0       # more equal values than fit between distinct ones
    z[14] = torch.finfo(t).max
    z[15] = torch.where(torch.arange(V) % 3 == 0, low, float(z[15, 0])).to(t)
    y = torch.randint(0, V, (16,), generator=torch.Generator().manual_seed(1))
    y[0], y[1], y[4], y[5] = 2, V // 3, 0, 7     # a -inf label among them
    for k in (0, 1, 8, min(V, 64)):
        check_scores(token_logprobs(z.to(DEV), y.to(DEV), top_k=k, entropy=True), z, y, k)


def test_labels_out_of_range_and_custom_ignore():
    from speech_to_text_amd import distillation_loss, token_logprobs
    z = randn((5, 300), torch.float32, 4).to(DEV).requires_grad_()
    y = torch.tensor([300, -1, 7, -100, 2 ** 40]).to(DEV)
    got = token_logprobs(z, y, entropy=True)
    assert got.logprobs.isnan().tolist() == [True, True, False, False, True] and not got.entropy.isnan().any()
    g, = torch.autograd.grad(got.logprobs.sum(), z)
    assert g.isnan().all(1).tolist() == [True, True, False, False, True] and (g[3] == 0).all()
    other = token_logprobs(z.detach(), torch.tensor([3, 3, 7, -1, 9]).to(DEV), ignore_index=7)
    assert other.logprobs.isnan().tolist() == [False, False, False, True, False] and float(other.logprobs[2]) == 0.0
    ids = torch.tensor([[1, 2], [3, 4], [5, 300], [9, 9], [1, -1]]).to(DEV)
    y = torch.tensor([300, 5, 7, -100, 2]).to(DEV)
    loss = distillation_loss(z, y, ids, torch.zeros(5, 2, device=DEV), reduction="none")
    assert loss.isnan().tolist() == [True, False, True, False, False]
    g, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    assert g.isnan().all(1).tolist() == [True, False, True, False, False] and not g[[1, 3, 4]].isnan().any()


GRAD_SHAPES = [(3, 1), (3, 2), (4, 9), (3, 64), (3, 127), (4, 1000), (3, 4099), (3, 10000), (3, 32000), (4, 50021), (2, 131073)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, V", GRAD_SHAPES)
def test_score_gradients(rows, V, dtype):
    from speech_to_text_amd import token_logprobs
    t, T, k = TYPES[dtype], 1.3, min(V, 7)
    z = randn((rows, V), t, V + 1)
    if V > 8:
        z[0, 3] = -np.inf
    g = torch.Generator().manual_seed(V)
    y = torch.randint(0, V, (rows,), generator=g)
    y[-1] = -100
    gl, gh, gt = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g)
    x = z.to(DEV).requires_grad_()
    out = token_logprobs(x, y.to(DEV), top_k=k, entropy=True, temperature=T)
    ids = out.top_ids.cpu().numpy()
    for a, b, c in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        outs = [o for o, on in zip((out.logprobs, out.entropy, out.top_logprobs), (a, b, c)) if on]
        ups = [u.to(DEV) for u, on in zip((gl, gh, gt), (a, b, c)) if on]
        d, = torch.autograd.grad(outs, x, ups, retain_graph=True)
        assert d.dtype == t and d.shape == x.shape
        want, size = O.token_logprobs_grad(np64(z), y.numpy(), gl.numpy() if a else None, gh.numpy() if b else None, ids,
                                           gt.numpy() if c else None, T)
        # the entropy term p (lp + H) is a difference: its error is that of lp and H, (1 + log2 V) (n_add + 70) u, times p
        check_grad(d, want, size + (np.abs(gh.numpy())[:, None] * (1 + np.log2(V + 1)) * np.exp(np.nan_to_num(
            O.log_softmax(np64(z), T), neginf=-1e4)) if b else 0), t, V)


def teacher_rows(rows, V, K, seed):
    """Ids with padding in the middle and the end, a row without any, a row with one id twice, the label among some."""
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(V)[:K] if V >= K else rng.integers(0, V, K) for _ in range(rows)])
    t = (2 * rng.standard_normal((rows, K))).astype(np.float32)
    if K > 2:
        ids[0, 1] = -1
        ids[-1, K // 2:] = -7
    if rows > 2:
        ids[1] = -1
        ids[2, -1] = ids[2, 0]
        t[2, 0] = -np.inf if K > 3 else t[2, 0]
    return torch.from_numpy(ids), torch.from_numpy(t)


def check_losses(got, want, z, y, ids, t, tau, alpha):
    V = z.shape[1]
    lp1, lpt = O.log_softmax(z), O.log_softmax(z, tau)
    tol = np.zeros(len(want))
    for r in range(len(want)):
        if y[r] < 0 or y[r] >= V or (ids[r] >= V).any():
            continue
        q = O.teacher(ids[r], t[r].astype(np.float64), tau)
        on = q > 0
        e = np.minimum(n_add(V) + 160 + 4 * (np.abs(lpt[r, ids[r][on]]) + np.abs(np.log(q[on]))), 1e30) * (
            1 + np.abs(np.log(q[on]) - lpt[r, ids[r][on]])) * q[on]
        tol[r] = U * (alpha * tau ** 2 * e.sum() + (1 - alpha) * (n_add(V) + 70 + 4 * abs(lp1[r, y[r]])) + 2 * abs(want[r]))
    same(got, want, tol, "loss")
    return tol


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, V, K, tau, alpha", [
    (3, 1, 1, 1.0, 0.5), (4, 2, 2, 2.0, 0.5), (5, 9, 4, 1.0, 1.0), (4, 64, 64, 2.0, 0.3), (4, 127, 5, 4.0, 0.7), (5, 1000, 16, 2.0, 0.0),
    (4, 4099, 1, 3.0, 0.5), (4, 10000, 8, 1.0, 0.5), (4, 16385, 20, 1.5, 0.9), (4, 32000, 32, 0.7, 0.5), (5, 50021, 16, 2.0, 0.5),
    (4, 50021, 64, 4.0, 1.0), (3, 65537, 9, 2.0, 0.8), (3, 131073, 24, 3.0, 0.5), (3, 200019, 64, 2.0, 0.5)])
def test_distillation(rows, V, K, tau, alpha, dtype):
    """Loss and gradient, fused ("sum") and per position ("none" with upstream weights), and the loss without a gradient."""
    from speech_to_text_amd import distillation_loss, distillation_loss_and_grad
    t = TYPES[dtype]
    z = randn((rows, V), t, 7 * V + K)
    g = torch.Generator().manual_seed(K)
    y = torch.randint(0, V, (rows,), generator=g)
    ids, teacher = teacher_rows(rows, V, K, V + K)
    y[0] = max(0, int(ids[0, 0]))
    if rows > 3:
        y[3] = -100
    want, grad, size = O.distillation(np64(z), y.numpy(), ids.numpy(), teacher.numpy(), tau, alpha)
    x = z.to(DEV).requires_grad_()
    args = (y.to(DEV), ids.to(DEV), teacher.to(DEV))
    kw = dict(temperature=tau, alpha=alpha)
    each = distillation_loss(x, *args, reduction="none", **kw)
    tol = check_losses(np64(each), want, np64(z), y.numpy(), ids.numpy(), teacher.numpy(), tau, alpha)
    with torch.no_grad():
        assert torch.equal(distillation_loss(x, *args, reduction="none", **kw), each)
    w = torch.randn(rows, generator=g)
    d, = torch.autograd.grad(each, x, w.to(DEV))
    check_grad(d, grad * w.numpy()[:, None], size * np.abs(w.numpy())[:, None], t, V)
    n = int((y != -100).sum())
    for red, f in (("sum", 1.0), ("mean", 1.0 / n)):
        total = distillation_loss(x, *args, reduction=red, **kw)
        d, = torch.autograd.grad(total, x)
        total = total.detach()
        assert abs(float(total) - want.sum() * f) <= (tol.sum() + 4 * U * np.abs(want).sum()) * f
        check_grad(d, grad * f, size * f, t, V)
        loss2, d2 = distillation_loss_and_grad(x, *args, reduction=red, **kw)
        assert abs(float(loss2) - float(total)) <= 2 * (tol.sum() + 4 * U * np.abs(want).sum()) * f
        check_grad(d2, grad * f, size * f, t, V)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_distillation_specials(dtype):
    """Student logits of -inf (at a teacher's id: loss +inf), rows of the lowest value, of only -inf, NaN, +inf."""
    from speech_to_text_amd import distillation_loss
    t = TYPES[dtype]
    V, K = 4099, 3
    z = randn((8, V), t, 5)
    ids = torch.tensor([[1, 2, 3]] * 8)
    z[0, 2] = -np.inf                             # a kept entry the student rules out
    z[1, 100:] = -np.inf
    z[2] = torch.finfo(t).min
    z[3] = -np.inf
    z[4, 9] = np.nan
    z[5, 9] = np.inf
    teacher = torch.tensor([[0.0, -1.0, -2.0]] * 8)
    teacher[6] = -np.inf                          # entries without weight: no teacher term
    ids[7] = -1
    y = torch.tensor([1, 5, 7, 1, 2, 2, 3, 4])
    want, grad, size = O.distillation(np64(z), y.numpy(), ids.numpy(), teacher.numpy(), 2.0, 0.5)
    assert np.isposinf(want[0]) and np.isfinite(want[[1, 2, 6, 7]]).all() and np.isnan(want[[3, 4, 5]]).all()
    x = z.to(DEV).requires_grad_()
    each = distillation_loss(x, y.to(DEV), ids.to(DEV), teacher.to(DEV), temperature=2.0, reduction="none")
    check_losses(np64(each), want, np.nan_to_num(np64(z), nan=0, neginf=-1e4), y.numpy(), ids.numpy(), teacher.numpy(), 2.0, 0.5)
    d, = torch.autograd.grad(each, x, torch.ones(8, device=DEV))
    check_grad(d, grad, size, t, V)
    d, = torch.autograd.grad(distillation_loss(x, y.to(DEV), ids.to(DEV), teacher.to(DEV), temperature=2.0, reduction="sum"), x)
    check_grad(d, grad, size, t, V)


def test_strided_student_and_types_of_the_teacher():
    from speech_to_text_amd import distillation_loss
    base = randn((3, 6, 2049), torch.bfloat16, 6).to(DEV)
    x = base[:, :-1, 1:].detach().requires_grad_()
    y = torch.randint(0, 2048, (3, 5), generator=torch.Generator().manual_seed(3))
    y[0, 3:] = -100
    ids, t = teacher_rows(15, 2048, 6, 1)
    t = t.to(torch.bfloat16)
    want, grad, size = O.distillation(np64(x).reshape(15, -1), y.numpy().reshape(-1), ids.numpy(), t.float().numpy(), 2.0, 0.4)
    loss = distillation_loss(x, y.int().to(DEV), ids.int().view(3, 5, 6).to(DEV), t.view(3, 5, 6).to(DEV), temperature=2.0, alpha=0.4)
    d, = torch.autograd.grad(loss, x)
    assert d.shape == x.shape and d.is_contiguous()
    check_grad(d, grad / 13, size / 13, torch.bfloat16, 2048)
    # one student row for every position: autograd sums the positions' gradients
    row = base[0, 0, 1:].detach().float().requires_grad_()
    loss = distillation_loss(row.expand(3, 5, 2048), y.to(DEV), ids.view(3, 5, 6).to(DEV), t.float().view(3, 5, 6).to(DEV), reduction="sum")
    d, = torch.autograd.grad(loss, row)
    _, grad, size = O.distillation(np.broadcast_to(np64(row), (15, 2048)), y.numpy().reshape(-1), ids.numpy(), t.float().numpy())
    check_grad(d, grad.sum(0, keepdims=True), size.sum(0, keepdims=True), torch.float32, 2048)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_backward_twice_and_upstream_factors(dtype):
    """A graph that is kept gives the same gradient again, whatever the first upstream gradient was; the loss stays usable."""
    from speech_to_text_amd import distillation_loss
    z = randn((6, 3001), TYPES[dtype], 9)
    y = torch.randint(0, 3001, (6,), generator=torch.Generator().manual_seed(9))
    ids, t = teacher_rows(6, 3001, 5, 2)
    want, grad, size = O.distillation(np64(z), y.numpy(), ids.numpy(), t.numpy())
    x = z.to(DEV).requires_grad_()
    loss = distillation_loss(x, y.to(DEV), ids.to(DEV), t.to(DEV), weight=0.25)
    first, = torch.autograd.grad(loss, x, torch.tensor(3.0, device=DEV), retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, x, torch.tensor(-1.0, device=DEV), retain_graph=True)
    loss.mul_(2.0)                                 # the caller's tensor, not the graph's
    f = 0.25 / 6
    assert torch.equal(first, kept)
    # an upstream factor rounds the made gradient a second time (bf16 / fp32): one more half step
    tol_twice = 2.0 if dtype != "fp16" else 1.0
    for d, g in ((first, 3.0), (second, -1.0)):
        info = torch.finfo(TYPES[dtype])
        w = grad * f * g
        tol = (n_add(3001) + 82) * U * size * f * abs(g) + tol_twice * info.eps / 2 * np.abs(w) * (1 + 2 ** -6) + 2 ** -24
        same(np64(d), w, tol, "grad")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(distillation_loss(x, y.to(DEV), ids.to(DEV), t.to(DEV)), x, create_graph=True)[0].sum(), x)


def test_no_rows_that_count():
    from speech_to_text_amd import distillation_loss, token_logprobs
    x = randn((4, 99), torch.float32, 1).to(DEV).requires_grad_()
    y = torch.full((4,), -100, device=DEV)
    ids, t = torch.full((4, 3), -1, device=DEV), torch.zeros(4, 3, device=DEV)
    loss = distillation_loss(x, y, ids, t)
    d, = torch.autograd.grad(loss, x)
    assert float(loss.detach()) == 0.0 and (d == 0).all()
    e = x[:0]
    loss = distillation_loss(e, y[:0], ids[:0], t[:0])
    d, = torch.autograd.grad(loss, x)
    assert float(loss.detach()) == 0.0 and (d == 0).all()
    assert distillation_loss(e.detach(), y[:0], ids[:0], t[:0], reduction="none").shape == (0,)
    s = token_logprobs(e.detach(), y[:0], top_k=2, entropy=True)
    assert s.logprobs.shape == (0,) and s.top_ids.shape == (0, 2)
    s = token_logprobs(x.detach(), y, top_k=2, entropy=True)
    assert (s.logprobs == 0).all() and (s.entropy == 0).all() and (s.top_ids == -1).all() and (s.top_logprobs == -np.inf).all()


def test_gradients_against_differences():
    """Central differences of the kernels' own losses along random directions: with h = 2^-5 and third derivatives along a unit
    direction below 1, |difference - slope| <= h^2 / 6 + (error of a loss, n_add + 250 u times its size) / h."""
    from speech_to_text_amd import distillation_loss, token_logprobs
    rows, V, h = 4, 37, 2.0 ** -5
    z = randn((rows, V), torch.float32, 11, scale=1.0)
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(8)).to(DEV)
    ids, t = (a.to(DEV) for a in teacher_rows(rows, V, 4, 3))

    def score(x):
        s = token_logprobs(x, y, top_k=3, entropy=True, temperature=1.5)
        return (s.logprobs + 0.5 * s.entropy + 0.1 * s.top_logprobs.sum(-1)).sum()

    def distil(x):
        return distillation_loss(x, y, ids, t, temperature=1.5, alpha=0.6, reduction="sum")

    for f in (score, distil):
        x = z.to(DEV).requires_grad_()
        slope, = torch.autograd.grad(f(x), x)
        for seed in range(4):
            v = randn((rows, V), torch.float32, 100 + seed)
            v = (v / v.norm()).to(DEV)
            with torch.no_grad():
                up, down = f(x + h * v), f(x - h * v)
            diff = (float(up) - float(down)) / (2 * h)
            assert abs(diff - float((slope * v).sum())) <= h * h / 6 + 350 * U * max(abs(float(up)), 10.0) / h


def test_far_rows():
    """Rows behind 2^31 elements and 2^32 bytes."""
    from speech_to_text_amd import distillation_loss_and_grad, token_logprobs
    B, P, V = 35, 2000, 32003                      # 2.24e9 elements, 4.48e9 bytes
    z = torch.zeros((B, P, V), dtype=torch.bfloat16, device=DEV)
    z[-1, -3:] = randn((3, V), torch.bfloat16, 1).to(DEV)
    y = torch.full((B, P), -100, device=DEV)
    y[-1, -3:] = torch.tensor([5, 31000, 32002], device=DEV)
    y[0, 0] = 1
    ids = torch.full((B, P, 4), -1, device=DEV)
    ids[-1, -3:] = torch.tensor([5, 9, 32002, 20000], device=DEV)
    t = torch.zeros((B, P, 4), device=DEV)
    s = token_logprobs(z, y, top_k=4, entropy=True)
    check_scores(type(s)(*(a[-1, -3:] for a in s)), z[-1, -3:], y[-1, -3:], 4)
    check_scores(type(s)(*(a[0, :2] for a in s)), z[0, :2], y[0, :2], 4)
    _, g = distillation_loss_and_grad(z, y, ids, t, temperature=2.0, reduction="sum")
    _, grad, size = O.distillation(np64(z[-1, -3:]), y[-1, -3:].cpu().numpy(), ids[-1, -3:].cpu().numpy(), t[-1, -3:].cpu().numpy(), 2.0)
    check_grad(g[-1, -3:], grad, size, torch.bfloat16, V)
    assert (g[-1, :-3] == 0).all() and (g[1:3] == 0).all()


def test_results_repeat_and_neighbours_stay():
    """Twice the same bits, with and without the other outputs asked for; a view's surroundings are not written."""
    from speech_to_text_amd import _lib, distillation_loss_and_grad, token_logprobs
    z = randn((300, 5003), torch.bfloat16, 2).to(DEV)
    y = torch.randint(0, 5003, (300,), generator=torch.Generator().manual_seed(4)).to(DEV)
    a, b = token_logprobs(z, y, top_k=20, entropy=True), token_logprobs(z, y, top_k=20, entropy=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c = token_logprobs(z, y)
    assert torch.equal(c.logprobs, a.logprobs)
    ids, t = (v.to(DEV) for v in teacher_rows(300, 5003, 8, 5))
    p, q = distillation_loss_and_grad(z, y, ids, t), distillation_loss_and_grad(z, y, ids, t)
    assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1])
    # through the C ABI: a gradient that starts and ends inside a larger buffer, at an odd element
    for dtype, code in ((torch.bfloat16, 2), (torch.float16, 1), (torch.float32, 0)):
        zz = z.to(dtype)
        buf = torch.full((300 * 5003 + 34,), 7.0, dtype=dtype, device=DEV)
        out = buf[17:-17]
        losses, stats = torch.empty(300, device=DEV), torch.empty(300, 4, device=DEV)
        st = torch.cuda.current_stream().cuda_stream
        n = __import__("ctypes").c_size_t()
        _lib.check(_lib.lib().sttfe_distill_workspace_bytes(300, 5003, code, __import__("ctypes").byref(n)))
        ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device=DEV)
        P = _lib.ptr
        _lib.check(_lib.lib().sttfe_distill_loss(P(zz), code, 1, 300, 0, 5003, 5003, P(y), -100, P(ids), P(t), 8, 1.0, 0.5, 1.0, 0,
                                                 P(losses), None, None, P(stats), P(out), P(ws), n.value, st))
        _, want = distillation_loss_and_grad(zz, y, ids, t, reduction="sum")
        assert torch.equal(out.view(300, 5003), want) and (buf[:17] == 7).all() and (buf[-17:] == 7).all()


def test_another_stream():
    from speech_to_text_amd import distillation_loss_and_grad, token_logprobs
    z = randn((64, 50021), torch.bfloat16, 3).to(DEV)
    y = torch.randint(0, 50021, (64,), generator=torch.Generator().manual_seed(4)).to(DEV)
    ids, t = (v.to(DEV) for v in teacher_rows(64, 50021, 8, 5))
    want, grad = token_logprobs(z, y, top_k=5, entropy=True), distillation_loss_and_grad(z, y, ids, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, g2 = token_logprobs(z, y, top_k=5, entropy=True), distillation_loss_and_grad(z, y, ids, t)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(grad[1], g2[1])


@pytest.mark.parametrize("rows, V", [(1, 50021), (40, 10000), (300, 5003), (3, 200019)])
def test_captured_graphs(rows, V):
    """Two captured graphs (a decoding step's scores, a training step's loss and gradient) replayed in turn on new inputs."""
    from speech_to_text_amd import distillation_loss_and_grad, token_logprobs
    z = randn((rows, V), torch.bfloat16, 0).to(DEV)
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(4)).to(DEV)
    ids, t = (v.to(DEV) for v in teacher_rows(rows, V, 8, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(z, y, top_k=5, entropy=True), distillation_loss_and_grad(z, y, ids, t)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = token_logprobs(z, y, top_k=5, entropy=True)
    with torch.cuda.graph(g2):
        b = distillation_loss_and_grad(z, y, ids, t)
    for k in range(4):
        z.copy_(randn((rows, V), torch.bfloat16, 20 + k).to(DEV))
        y.copy_(torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(50 + k)).to(DEV))
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        want, (loss, grad) = token_logprobs(z, y, top_k=5, entropy=True), distillation_loss_and_grad(z, y, ids, t)
        assert all(torch.equal(p, q) for p, q in zip(a, want))
        assert torch.equal(b[0], loss) and torch.equal(b[1], grad)


def test_teacher_to_student(tmp_path):
    """The run as it is used: a teacher's logits over a batch go to the cache (token_logprobs on the GPU), come back through
    dataset and collator, and the student's gradient is the oracle's for those alternatives; the alternatives are a softmax's."""
    from speech_to_text_amd import AudioCollator, DataConfig, FeatureCacheDataset, FeatureCacheWriter, distillation_loss, token_logprobs
    B, V, K = 5, 10007, 12
    rng = np.random.default_rng(0)
    labels = [rng.integers(0, V, n).tolist() for n in (7, 1, 12, 0, 5)]
    teacher = randn((B, 14, V), torch.bfloat16, 1).to(DEV)
    w = FeatureCacheWriter(str(tmp_path), "speech2text", 80, shard_clips=2, teacher_top=K)
    w.add_batch(list(range(B)), torch.zeros(B, 80, 30), [0] * B, labels=labels, teacher_logits=teacher)
    w.close()
    ds = FeatureCacheDataset(str(tmp_path))
    batch = AudioCollator(DataConfig(), "speech2text", True)([ds[i] for i in range(B)])
    y, ids, t = batch["labels"], batch["teacher_ids"], batch["teacher_logits"]
    assert y.shape == (B, 12) and ids.shape == (B, 12, K)
    for b in range(B):
        n = len(labels[b])
        _, _, want, top = O.token_logprobs(np64(teacher[b, :n]), None, K)
        assert np.array_equal(ids[b, :n].numpy(), want)
        same(np64(t[b, :n]), top, (n_add(V) + 70 + 4 * np.abs(top)) * U, "kept")
    z = randn((B, 12, V), torch.bfloat16, 2)
    x = z.to(DEV).requires_grad_()
    loss = distillation_loss(x, y.to(DEV), ids.to(DEV), t.to(DEV), temperature=2.0, alpha=0.8)
    loss.backward()
    want, grad, size = O.distillation(np64(z).reshape(-1, V), y.numpy().reshape(-1), ids.numpy().reshape(-1, K),
                                      t.numpy().reshape(-1, K), 2.0, 0.8)
    n = sum(map(len, labels))
    tol = check_losses(want, want, np64(z).reshape(-1, V), y.numpy().reshape(-1), ids.numpy().reshape(-1, K), t.numpy().reshape(-1, K), 2.0, 0.8)
    assert abs(float(loss.detach()) - want.sum() / n) <= (tol.sum() + 4 * U * np.abs(want).sum()) / n
    check_grad(x.grad, grad / n, size / n, torch.bfloat16, V)
    # the same labels scored by the student: the loss without a teacher is the mean of the label's -logprob
    s = token_logprobs(x.detach(), y.to(DEV))
    ce = distillation_loss(x.detach(), y.to(DEV), ids.to(DEV), t.to(DEV), alpha=0.0)
    assert abs(float(ce) + float(s.logprobs.double().sum()) / n) <= 4 * U * abs(float(ce)) + 2 * (n_add(V) + 70) * U


@pytest.mark.parametrize("rows", [1, 700, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("V", [129, 17001])
def test_means_over_few_and_many_rows(rows, V):
    """The rows that count are counted in two ways, and dealt among teams from some number on: the mean, its gradient and the
    rows that hold nothing, with labels that count in runs, at random, hardly any, and all."""
    from speech_to_text_amd import distillation_loss_and_grad, token_logprobs
    rng = np.random.default_rng(rows + V)
    z = randn((1, V), torch.bfloat16, V, scale=2.0).to(DEV).repeat(rows, 1)
    for kind in ("all", "runs", "random", "few"):
        y = rng.integers(0, V, rows)
        keep = {"all": np.ones(rows, bool), "runs": np.arange(rows) % 97 < 40, "random": rng.random(rows) < 0.6,
                "few": np.arange(rows) == rows // 2}[kind]
        y[~keep] = -100
        yt = torch.from_numpy(y).to(DEV)
        ids = torch.full((rows, 2), 5, device=DEV)
        t = torch.zeros(rows, 2, device=DEV)
        want, grad, size = O.distillation(np64(z[:1]), np.array([7]), np.array([[5, 5]]), np.zeros((1, 2)), 2.0, 0.5)
        lp = O.log_softmax(np64(z[:1]))[0]
        n = keep.sum()
        each = np.where(keep, want[0] + 0.5 * lp[7] - 0.5 * lp[np.maximum(y, 0)], 0.0)
        loss, g = distillation_loss_and_grad(z, yt, ids, t, temperature=2.0)
        tol = (n_add(V) + 400) * 20 * U * np.abs(each).max()
        assert abs(float(loss) - each.sum() / max(n, 1)) <= tol
        off = g.float()
        assert (off[torch.from_numpy(~keep).to(DEV)] == 0).all()
        if n == 0:
            continue
        r = int(np.flatnonzero(keep)[-1])
        w = grad[0].copy()
        w[7] += 0.5
        w[y[r]] -= 0.5
        sz = size[0].copy()
        sz[y[r]] += 1.0
        check_grad(g[r], (w / n)[None], (sz / n)[None], torch.bfloat16, V)
        s = token_logprobs(z, yt, top_k=3, entropy=True)
        assert np.abs(np64(s.logprobs) - np.where(keep, lp[np.maximum(y, 0)], 0.0)).max() <= (n_add(V) + 70 + 80) * U
        assert ((s.entropy == 0).cpu().numpy() == ~keep).all()
        assert ((s.top_ids[:, 0] == -1).cpu().numpy() == ~keep).all() and len(s.top_ids[torch.from_numpy(keep).to(DEV)].unique(dim=0)) == 1


@pytest.mark.parametrize("dtype", list(TYPES))
def test_wide_vocabulary_many_rows(dtype):
    """Rows of several segments, more than the chip's teams: ragged labels, scores and gradients."""
    from speech_to_text_amd import distillation_loss, token_logprobs
    rows, V, K = 700, 70001, 6
    z = randn((5, V), TYPES[dtype], 3).to(DEV)
    pick = torch.arange(rows, device=DEV) % 5
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(1)).to(DEV)
    y[torch.arange(rows, device=DEV) % 7 > 3] = -100
    x = z[pick]
    rng = np.random.default_rng(1)
    ids5, t5 = rng.integers(0, V, (5, K)), rng.standard_normal((5, K)).astype(np.float32)
    ids, t = torch.from_numpy(ids5).to(DEV)[pick], torch.from_numpy(t5).to(DEV)[pick]
    s = token_logprobs(x, y, top_k=K, entropy=True)
    _, h, top, _ = O.token_logprobs(np64(z), None, K)
    lp = O.log_softmax(np64(z))
    live, p5, yn = (y >= 0).cpu().numpy(), pick.cpu().numpy(), y.cpu().numpy()
    same(np64(s.logprobs), np.where(live, lp[p5, np.maximum(yn, 0)], 0.0), np.full(rows, (n_add(V) + 70 + 80) * U), "logprobs")
    same(np64(s.entropy), np.where(live, h[p5], 0.0), np.full(rows, (n_add(V) + 70) * (1 + np.log2(V + 1)) * U), "entropy")
    assert np.array_equal(s.top_ids.cpu().numpy(), np.where(live[:, None], top[p5], -1))
    x.requires_grad_()
    for red, f in (("sum", 1.0), ("mean", 1.0 / live.sum())):
        loss = distillation_loss(x, y, ids, t, temperature=3.0, alpha=0.7, weight=0.5, reduction=red)
        g, = torch.autograd.grad(loss, x)
        assert (g[~torch.from_numpy(live).to(DEV)] == 0).all()
        rs = [int(r) for r in np.flatnonzero(live)[[0, 1, 7, -1]]]
        want, grad, size = O.distillation(np64(x[rs]), yn[rs], ids5[p5[rs]], t5[p5[rs]], 3.0, 0.7)
        check_grad(g[rs], grad * f * 0.5, size * f * 0.5, TYPES[dtype], V)
        every, _, _ = O.distillation(np64(z), np.zeros(5, np.int64), ids5, t5, 3.0, 0.7)
        total = sum(every[p5[r]] + 0.3 * lp[p5[r], 0] - 0.3 * lp[p5[r], yn[r]] for r in np.flatnonzero(live)) * f * 0.5
        assert abs(float(loss.detach()) - total) <= (n_add(V) + 400) * 20 * U * abs(total)


def hard_rows(V, dtype, seed):
    """Rows whose alternatives are not few elements above a bound: sorted, equal, masked, NaN in places, few distinct values."""
    g = torch.Generator().manual_seed(seed)
    rows = {}
    rows["rising"] = torch.linspace(-8, 12, V)
    rows["falling"] = torch.linspace(12, -8, V)
    rows["equal"] = torch.full((V,), 1.5)
    rows["equal below 0"] = torch.full((V,), -1.5)
    zeros = torch.zeros(V)
    zeros[torch.arange(V) % 3 == 1] = -0.0
    rows["zeros of both signs"] = zeros
    few = torch.full((V,), -float("inf"))
    few[torch.randperm(V, generator=g)[: 8]] = torch.randn(min(8, V), generator=g)
    rows["masked to 8"] = few
    run = torch.full((V,), -float("inf"))
    run[V // 3 : V // 3 + 500] = torch.randn(len(run[V // 3 : V // 3 + 500]), generator=g)
    rows["masked to a run"] = run
    rows["two values"] = (torch.rand(V, generator=g) < 0.5).float()
    rows["quarters"] = (torch.randn(V, generator=g) * 4).round() / 4 - 3
    block = torch.randn(V, generator=g)
    block[V // 2 : V // 2 + 90] += 20
    rows["a high block"] = block
    lowest = torch.full((V,), torch.finfo(dtype).min)
    lowest[torch.randperm(V, generator=g)[: 3]] = 2.0
    rows["lowest value but 3"] = lowest
    for name, n in (("a few NaN", 3), ("many NaN", 200)):
        nan = torch.randn(V, generator=g)
        nan[torch.randperm(V, generator=g)[:n]] = float("nan")
        rows[name] = nan
    nan = torch.full((V,), -float("inf"))
    nan[-1] = float("nan")
    rows["NaN behind -inf"] = nan
    inf = torch.randn(V, generator=g)
    inf[torch.randperm(V, generator=g)[: 100]] = float("inf")
    rows["many inf"] = inf
    rows["nothing but -inf"] = torch.full((V,), -float("inf"))
    return rows


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [70, 401, 2000, 4099, 10007, 32001, 50021, 200019])
def test_alternatives_of_hard_rows(V, dtype):
    """The ids are exact whatever the row: value falling, NaN first, equal values by index.  Every row at two alignments."""
    from speech_to_text_amd import token_logprobs

    rows = hard_rows(V, TYPES[dtype], V)
    z = torch.stack(list(rows.values())).to(TYPES[dtype])
    store = torch.zeros((len(rows), V + 3), dtype=TYPES[dtype], device=DEV)
    store[:, 2 : V + 2] = z.to(DEV)
    for k in (1, 7, 16, 64):
        want = [O.alternatives(np64(row), k) for row in z]
        for x in (z.to(DEV), store[:, 2 : V + 2]):
            got = token_logprobs(x, top_k=k).top_ids.cpu().numpy()
            for r, name in enumerate(rows):
                assert np.array_equal(got[r], want[r]), (name, k)


@pytest.mark.parametrize("T", [1e-3, 1e3])
@pytest.mark.parametrize("V", [401, 32001])
def test_extreme_temperatures(V, T):
    from speech_to_text_amd import distillation_loss, token_logprobs
    z = randn((5, V), torch.float32, V, offset=40.0)
    y = torch.randint(0, V, (5,), generator=torch.Generator().manual_seed(V))
    check_scores(token_logprobs(z.to(DEV), y.to(DEV), top_k=9, entropy=True, temperature=T), z, y, 9, T)
    ids, teacher = teacher_rows(5, V, 6, V)
    want, grad, size = O.distillation(np64(z), y.numpy(), ids.numpy(), teacher.numpy(), T, 0.5)
    x = z.to(DEV).requires_grad_()
    each = distillation_loss(x, y.to(DEV), ids.to(DEV), teacher.to(DEV), temperature=T, reduction="none")
    check_losses(np64(each), want, np64(z), y.numpy(), ids.numpy(), teacher.numpy(), T, 0.5)
    d, = torch.autograd.grad(each.sum(), x)
    check_grad(d, grad, size, torch.float32, V)


@pytest.mark.parametrize("V", [2000, 9001, 66001])
def test_more_rows_than_are_dealt_at_once(V):
    """Rows far apart in a call of 20000 (several rounds of dealing them out, many of them ignored) have the bits that they have
    alone, read from the same place: the alignment of a row decides the order of its sums."""
    from speech_to_text_amd import distillation_loss, distillation_loss_and_grad, token_logprobs
    n = 20000
    g = torch.Generator(device=DEV).manual_seed(V)
    z = torch.empty((n, V), dtype=torch.bfloat16, device=DEV).normal_(0, 2.5, generator=g)
    y = torch.randint(0, V, (n,), generator=g, device=DEV)
    y[torch.rand(n, generator=g, device=DEV) < 0.3] = -100
    y[5000:9000] = -100
    ids = torch.randint(0, V, (n, 4), generator=g, device=DEV)
    t = torch.randn((n, 4), generator=g, device=DEV)
    some = (0, 1, 255, 256, 1023, 4999, 5000, 8191, 8192, 9000, 12345, 16383, 16384, 16385, 19998, 19999)
    for k in (0, 5):
        got = token_logprobs(z, y, top_k=k, entropy=True)
        for r in some:
            alone = token_logprobs(z[r : r + 1], y[r : r + 1], top_k=k, entropy=True)
            assert all(torch.equal(a[r : r + 1], b) for a, b in zip(got, alone) if a is not None), r
        assert bool((got.logprobs[y == -100] == 0).all()) and bool((got.entropy[y == -100] == 0).all())
        assert bool((got.logprobs[y != -100] < 0).all())
    each = distillation_loss(z, y, ids, t, temperature=2.0, reduction="none")
    loss, grad = distillation_loss_and_grad(z, y, ids, t, temperature=2.0, reduction="sum")
    for r in some:
        one = tuple(v[r : r + 1] for v in (z, y, ids, t))
        assert torch.equal(each[r : r + 1], distillation_loss(*one, temperature=2.0, reduction="none")), r
        assert torch.equal(grad[r : r + 1], distillation_loss_and_grad(*one, temperature=2.0, reduction="sum")[1]), r
    assert bool((grad[y == -100] == 0).all()) and bool((grad.abs().amax(1)[y != -100] > 0).all())
    total = float(each.double().sum())
    assert abs(float(loss) - total) <= 2 * U * abs(total)


@pytest.mark.parametrize("V", [5003, 70001])
def test_two_streams_at_once(V):
    """Calls on two streams that run side by side share nothing."""
    from speech_to_text_amd import distillation_loss_and_grad, token_logprobs
    sets, want = [], []
    for s in range(2):
        z = randn((300, V), torch.bfloat16, s).to(DEV)
        y = torch.randint(0, V, (300,), generator=torch.Generator().manual_seed(s)).to(DEV)
        sets.append((z, y, *(v.to(DEV) for v in teacher_rows(300, V, 8, s))))
        want.append((token_logprobs(z, y, top_k=7, entropy=True), distillation_loss_and_grad(*sets[s], temperature=2.0)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                z, y = sets[s][:2]
                got[s].append((token_logprobs(z, y, top_k=7, entropy=True), distillation_loss_and_grad(*sets[s], temperature=2.0)))
    torch.cuda.synchronize()
    for s in range(2):
        for scores, (loss, grad) in got[s]:
            assert all(torch.equal(a, b) for a, b in zip(scores, want[s][0]))
            assert torch.equal(loss, want[s][1][0]) and torch.equal(grad, want[s][1][1])


def confident_rows(V, dtype, seed):
    """Rows in which one token (or two, or a stair of them) stands `gap` nats above all others, anywhere in the row, as a model
    that is sure of its transcript gives them; and rows of one large negative value.  -> rows, index of each row's largest."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows = []
    for n, gap in enumerate((0.5, 1.5, 2.5, 3.5, 5.0, 8.0, 12.0, 16.0, 20.0, 25.0, 30.0, 40.0)):
        for at in {0, V - 1, V // 2 + n, *(int(v) for v in rng.integers(0, V, 2))}:
            z = torch.randn(V, generator=g) + (3.0 if n % 2 else -60.0)
            z[at] = z.max() + gap
            rows.append(z)
    for gap in (10.0, 25.0):
        z = torch.randn(V, generator=g)
        z[[V // 3, 2 * V // 3]] = float(z.max()) + gap
        rows.append(z)
    z = torch.randn(V, generator=g)
    stair = torch.arange(7, V, max(1, V // 23))
    z[stair] = 5.0 + 2.0 * torch.arange(len(stair)).float()                # rises by less than is climbed at once, and goes on
    rows.append(z)
    z = torch.full((V,), -float("inf"))
    z[V // 5], z[V - V // 5 - 1] = 1.0, 28.0
    rows.append(z)
    for low in (-1e4, -3e4, -1e9 if dtype != torch.float16 else -6e4):
        rows.append(torch.full((V,), low))
        z = torch.full((V,), low)
        z[rng.integers(0, V, 3)] = torch.tensor([0.0, -1.0, 24.0])
        rows.append(z)
    z = torch.stack(rows).to(dtype)
    return z, z.float().argmax(1)


def sums_of(z, T):
    """What the bars of confident rows need of a row, in float64: log probabilities, ln S, relative error of S, A, A2, eps."""
    lp = O.log_softmax(z, T)
    p, top = np.exp(lp), lp.max(-1)
    a = (top[:, None] - np.where(np.isfinite(lp), lp, top[:, None])) / np.log(2)      # distance from the largest, in bits
    A, A2 = (p * a).sum(-1), (p * a * a).sum(-1)
    first = lp.argmax(-1)
    rest = p * (np.arange(z.shape[1]) != first[:, None])
    eps, eps_w = rest.sum(-1), (rest * (a + 4.1)).sum(-1)
    rel = (4.3 * A + 22) * U + np.minimum(n_add(z.shape[1]) * U, eps)
    return lp, -top, rel, A, A2, eps_w, a


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V, T", [(401, 1.0), (2000, 1.0), (10007, 1.0), (10007, 0.6), (32001, 1.0), (50021, 1.0), (50021, 2.5),
                                  (51865, 1.0), (200019, 1.0)])
def test_confident_rows(V, T, dtype):
    """Sure tokens keep the precision of a softmax taken against the row's maximum: no log probability above 0, no entropy below 0,
    and bars without the slack of a flat row.

    With a_j the distance of element j from the row's largest in bits, all powers of two are taken within 4.1 bits of the
    maximum, so a term of S is off by (4.3 a_j + 14) u (rounded exponents 2.8 a_j + 5.7, three exponentials 6, products 2, steps
    from one reference to a higher one 1.5 a_j; the square of a power, for a second softmax, 8 more), and adding errs by n_add u at
    most, and by no more than what is added: eps = the mass outside the largest element.
      |dS / S| <= rel = (4.3 A + 22) u + min(n_add u, eps),  A = sum p a
      |d lp| <= rel + (2 + 4 ln S + 3 |lp|) u
      |d W| <= (4.3 A2 + 19 A + 17) u + min(n_add (A + 4.1) u, eps_w), A2 = sum p a^2, eps_w = sum over the others p (a + 4.1)
      |d H| <= ln 2 (|d W| + A rel + 3 A u) + rel + (4 ln S + 2 H) u
      |d p_j| <= p_j (rel + (10 + 4 ln S + 2.8 a_j) u), or 2^-126 where p_j is below that: v_exp_f32 flushes its result, and the
    flushed p_j is then multiplied by 1 / T (by alpha tau and 1 - alpha), so that 2^-126 is, too."""
    from speech_to_text_amd import distillation_loss, token_logprobs
    t = TYPES[dtype]
    z, at = confident_rows(V, t, V)
    n = len(z)
    other = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(V))
    store = torch.zeros((n, V + 3), dtype=t, device=DEV)
    store[:, 1 : V + 1] = z.to(DEV)
    lp, ln_s, rel, A, A2, eps_w, a = sums_of(np64(z), T)
    p = np.exp(lp)
    h = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum(-1)
    dw = (4.3 * A2 + 19 * A + 17) * U + np.minimum(n_add(V) * (A + 4.1) * U, eps_w)
    bar_h = np.log(2) * (dw + A * rel + 3 * A * U) + rel + (4 * ln_s + 2 * h) * U
    rows = np.arange(n)
    for y in (at, other):
        want = lp[rows, y.numpy()]
        bar = rel + (2 + 4 * ln_s + 3 * np.abs(want)) * U
        for x in (z.to(DEV), store[:, 1 : V + 1]):
            for k in (0, 4):
                got = token_logprobs(x, y.to(DEV), top_k=k, entropy=True, temperature=T)
                same(np64(got.logprobs), want, bar, "logprobs")
                same(np64(got.entropy), h, bar_h, "entropy")
                assert not (got.logprobs > 0).any() and not (got.entropy < 0).any()
                if k:
                    assert np.array_equal(got.top_ids[:, 0].cpu().numpy(), at.numpy()) and not (got.top_logprobs > 0).any()
                    top = np.take_along_axis(lp, got.top_ids.cpu().numpy(), 1)
                    same(np64(got.top_logprobs), top, rel[:, None] + (2 + 4 * ln_s[:, None] + 3 * np.abs(top)) * U, "top_logprobs")
    # gradient of the sure token's log probability: p_j, and 1 - p of its own
    info, tiny = torch.finfo(t), 2.0 ** -25 if dtype == "fp16" else 2.0 ** -126
    x = z.to(DEV).requires_grad_()
    d, = torch.autograd.grad(token_logprobs(x, at.to(DEV), temperature=T).logprobs.sum(), x)
    dp = p * (rel[:, None] + (10 + 4 * ln_s[:, None] + 2.8 * a) * U)
    one = np.arange(V) == at.numpy()[:, None]
    want = (one - p) / T
    same(np64(d), want, dp / T + (info.eps / 2 + 2 * U) * np.abs(want) * (1 + 2 ** -10) + tiny + 2.0 ** -126 / T, "grad")
    # distillation with the sure token as the teacher's only entry and as the label
    ids, teacher, alpha = at[:, None].to(DEV), torch.zeros(n, 1, device=DEV), 0.5
    for tau in (1.0, 2.0, 3.0):
        lpt, ln_t, rel_t, _, _, _, a_t = sums_of(np64(z), tau)
        lp1, ln_1, rel_1, _, _, _, a_1 = sums_of(np64(z), 1.0)
        want = alpha * tau ** 2 * -lpt[rows, at] - (1 - alpha) * lp1[rows, at]
        bar = (alpha * tau ** 2 * (rel_t + (2 + 4 * ln_t) * U) + (1 - alpha) * (rel_1 + (2 + 4 * ln_1) * U) + 6 * U * np.abs(want))
        each = distillation_loss(x, at.to(DEV), ids, teacher, temperature=tau, alpha=alpha, reduction="none")
        same(np64(each), want, bar, "loss")
        assert not (each < 0).any()
        pt, p1 = np.exp(lpt), np.exp(lp1)
        grad = alpha * tau * (pt - one) + (1 - alpha) * (p1 - one)
        dg = (alpha * tau * pt * (rel_t[:, None] + (12 + 4 * ln_t[:, None] + 2.8 * a_t) * U)
              + (1 - alpha) * p1 * (rel_1[:, None] + (12 + 4 * ln_1[:, None] + 2.8 * a_1) * U) + 3 * U * (alpha * tau + 1 - alpha) * one)
        tol = dg + (info.eps / 2 + 2 * U) * np.abs(grad) * (1 + 2 ** -10) + tiny + 2.0 ** -126 * (alpha * tau + 1 - alpha)
        d, = torch.autograd.grad(each, x, torch.ones(n, device=DEV))
        same(np64(d), grad, tol, "grad")
        d, = torch.autograd.grad(distillation_loss(x, at.to(DEV), ids, teacher, temperature=tau, alpha=alpha, reduction="sum"), x)
        same(np64(d), grad, tol, "grad of the sum")


@pytest.mark.parametrize("alpha", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("V", [300, 10007, 140001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_outside_the_vocabulary_is_nan_whatever_the_terms(dtype, V, alpha):
    """A label or an id outside the vocabulary makes loss and gradient of its row NaN: with and without the teacher's term or the
    label's, with entries that are all outside (none is kept), and beside a row that keeps none and is sound."""
    from speech_to_text_amd import distillation_loss, distillation_loss_and_grad
    z = randn((8, V), TYPES[dtype], V)
    y = torch.tensor([V, 5, 7, -100, -1, 2, 2 ** 40, 3])
    ids = torch.tensor([[1, 2], [V, V + 3], [V, -1], [V, V], [-1, -1], [-1, -1], [4, 4], [5, V]])
    bad = torch.tensor([True, True, True, False, True, False, True, True])
    teacher = torch.zeros(8, 2)
    x = z.to(DEV).requires_grad_()
    args = (y.to(DEV), ids.to(DEV), teacher.to(DEV))
    for tau in (1.0, 2.0, 3.0):
        each = distillation_loss(x, *args, temperature=tau, alpha=alpha, reduction="none")
        d, = torch.autograd.grad(each, x, torch.ones(8, device=DEV))
        s, = torch.autograd.grad(distillation_loss(x, *args, temperature=tau, alpha=alpha, reduction="sum"), x)
        total, m = distillation_loss_and_grad(x, *args, temperature=tau, alpha=alpha)
        assert torch.equal(each.detach().isnan().cpu(), bad) and bool(total.isnan())
        for g in (d, s, m):
            assert torch.equal(g.isnan().all(1).cpu(), bad) and not g[~bad.to(DEV)].isnan().any() and bool((g[3] == 0).all())


@pytest.mark.parametrize("V", [300, 50021, 140001])
def test_entropy_and_alternatives_do_not_depend_on_the_label(V):
    """A label outside the vocabulary is NaN where it is asked for and nowhere else; a gradient without its log probability is that
    of the same row with any other label."""
    from speech_to_text_amd import token_logprobs
    z = randn((4, V), torch.bfloat16, V).to(DEV)
    bad, good = torch.tensor([V, -1, 2 ** 40, 3], device=DEV), torch.tensor([0, V - 1, 7, 3], device=DEV)
    grads = []
    for y in (bad, good):
        x = z.clone().requires_grad_()
        s = token_logprobs(x, y, top_k=5, entropy=True)
        d, = torch.autograd.grad((s.entropy.sum(), s.top_logprobs.sum()), x, retain_graph=True)
        full, = torch.autograd.grad(s.logprobs.sum(), x)
        grads.append((s.entropy, s.top_ids, s.top_logprobs, d))
        want = [y is bad] * 3 + [False]
        assert s.logprobs.isnan().tolist() == want and full.isnan().all(1).tolist() == want and full.isnan().any(1).tolist() == want
    assert all(torch.equal(a, b) and not a.isnan().any() for a, b in zip(*grads))


def test_as_many_rows_as_a_call_takes():
    """2^24 rows, the most a call takes: 2^32 threads for the gradients are one too many for a launch.  Rows repeat, so a row's
    result is known; the first, the last and those around the launches' border are looked at, and all by equality."""
    from speech_to_text_amd import distillation_loss, token_logprobs
    n, V, period = 2 ** 24, 5, 64
    z = randn((period, V), torch.bfloat16, 1)
    y = torch.randint(0, V, (period,), generator=torch.Generator().manual_seed(2))
    y[5] = -100
    ids, t = teacher_rows(period, V, 2, 3)
    lp, _, _, _ = O.token_logprobs(np64(z), y.numpy())
    want_s, size_s = O.token_logprobs_grad(np64(z), y.numpy(), np.ones(period))
    loss, want_d, size_d = O.distillation(np64(z), y.numpy(), ids.numpy(), t.numpy(), 3.0, 0.5)
    x = z.to(DEV).repeat(n // period, 1).requires_grad_()
    yy, ii, tt = (v.to(DEV).repeat(n // period, *([1] * (v.dim() - 1))) for v in (y, ids, t))
    s = token_logprobs(x, yy)
    same(np64(s.logprobs[-period:]), lp, (n_add(V) + 70 + 4 * np.abs(lp)) * U, "logprobs")
    d, = torch.autograd.grad(s.logprobs.sum(), x)
    check_grad(d[:period], want_s, size_s, torch.bfloat16, V)
    assert bool((d.view(-1, period, V) == d[:period]).all())
    each = distillation_loss(x, yy, ii, tt, temperature=3.0, reduction="none")
    d, = torch.autograd.grad(each, x, torch.ones_like(each))
    check_grad(d[:period], want_d, size_d, torch.bfloat16, V)
    assert bool((d.view(-1, period, V) == d[:period]).all()) and bool((each.view(-1, period) == each[:period]).all())
    with pytest.raises(Exception, match="unsupported|not supported|failed"):
        token_logprobs(x.detach()[:1].expand(n + 1, V), top_k=1)


def test_forward_mode_tangent_of_an_upstream_gradient_is_refused():
    from torch.autograd import forward_ad
    from speech_to_text_amd import distillation_loss, token_logprobs
    y, ids, t = torch.tensor([1, 2], device=DEV), torch.ones(2, 3, dtype=torch.long, device=DEV), torch.zeros(2, 3, device=DEV)
    for f in (lambda x: token_logprobs(x, y).logprobs.sum(), lambda x: distillation_loss(x, y, ids, t)):
        x = randn((2, 50), torch.float32, 1).to(DEV).requires_grad_()
        loss = f(x)
        with forward_ad.dual_level():
            up = forward_ad.make_dual(torch.ones((), device=DEV), torch.ones((), device=DEV))
            with pytest.raises(ValueError, match="forward-mode tangent"):
                torch.autograd.grad(loss, x, up)


@pytest.mark.parametrize("V", [2003, 10007, 140001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scaled_gradients(dtype, V):
    """A loss scale is applied before the gradient is rounded: a float16 gradient of a mean keeps what it would lose (2^-25 is the
    largest value that rounds to 0), every type has the oracle's gradient times the scale, the loss has no scale in it; numbers,
    tensors, and a captured call whose scale changes between replays."""
    from speech_to_text_amd import distillation_loss_and_grad
    rows = 300 if V < 100000 else 40
    z = randn((rows, V), TYPES[dtype], V, scale=2.0)
    y = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(V))
    y[3] = -100
    ids, teacher = teacher_rows(rows, V, 4, V)
    some = [0, 1, 2, 3, 7, rows - 1]
    _, grad, size = O.distillation(np64(z[some]), y.numpy()[some], ids.numpy()[some], teacher.numpy()[some], 2.0, 0.5)
    f = 0.5 / (rows - 1)
    x, args = z.to(DEV), (y.to(DEV), ids.to(DEV), teacher.to(DEV))
    kw = dict(temperature=2.0, weight=0.5)
    loss, plain = distillation_loss_and_grad(x, *args, **kw)
    for scale in (2.0 ** 14, torch.full((1,), 2.0 ** 14, device=DEV), 3.0):
        f_s = f * float(scale)
        same_loss, g = distillation_loss_and_grad(x, *args, grad_scale=scale, **kw)
        assert abs(float(same_loss) - float(loss)) <= 2 * (n_add(V) + 400) * 20 * U * abs(float(loss))
        check_grad(g[some], grad * f_s, size * f_s, TYPES[dtype], V)
        assert bool((g[3] == 0).all())
    if dtype == "fp16":
        lost = (np.abs(grad * f) < 2.0 ** -25) & (np.abs(grad * f) * 2.0 ** 14 > 2.0 ** -20)
        scaled = distillation_loss_and_grad(x, *args, grad_scale=2.0 ** 14, **kw)[1]
        assert lost.any() and (np64(plain[some])[lost] == 0).all() and (np64(scaled[some])[lost] != 0).all()
    scale = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        distillation_loss_and_grad(x, *args, grad_scale=scale, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = distillation_loss_and_grad(x, *args, grad_scale=scale, **kw)
    for k in (1.0, 64.0, 2.0 ** 14):
        scale.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        want = distillation_loss_and_grad(x, *args, grad_scale=k, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("V", [1, 2, 300, 10007, 140001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_without_a_term_are_zero_whatever_they_hold(dtype, V):
    """alpha 1 and no kept entry (no ids, or teacher logits of -inf): loss and gradient are 0, also of a row that has no softmax."""
    from speech_to_text_amd import distillation_loss, distillation_loss_and_grad
    z = randn((10, V), TYPES[dtype], V)
    z[0], z[5] = -np.inf, -np.inf
    z[1, V // 2] = z[6, V // 2] = np.nan
    z[2, V - 1] = z[7, V - 1] = np.inf
    z[3] = torch.finfo(TYPES[dtype]).min
    y = torch.randint(0, V, (10,), generator=torch.Generator().manual_seed(V)).to(DEV)
    ids = torch.full((10, 3), -1, device=DEV)
    ids[4:9] = 0
    t = torch.full((10, 3), -np.inf, device=DEV)
    ids[9], t[9] = 0, 0.0                         # a sound row with a term
    x = z.to(DEV).requires_grad_()
    for tau in (1.0, 2.0):
        each = distillation_loss(x, y, ids, t, temperature=tau, alpha=1.0, reduction="none")
        d, = torch.autograd.grad(each, x, torch.ones(10, device=DEV))
        s, = torch.autograd.grad(distillation_loss(x, y, ids, t, temperature=tau, alpha=1.0, reduction="sum"), x)
        total, m = distillation_loss_and_grad(x, y, ids, t, temperature=tau, alpha=1.0, reduction="sum")
        assert bool((each[:9] == 0).all()) and bool(total == each[9])
        for g in (d, s, m):
            assert bool((g[:9] == 0).all()) and not bool(g[9].isnan().any()) and (V == 1 or bool((g[9] != 0).any()))
