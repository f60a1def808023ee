"""The client-step operators against their definitions in float64.

Tolerances are error bounds, not observations.  u = eps / 2 is a type's unit roundoff;
an output of type T is rounded once (u_T |value|).  A float32 sum of n terms is off by
at most n u_32 sum |terms|, whatever its order; a matrix instruction may chop where it
adds, so products count 2 u_32 per term.  exp and log cost a few u_32 of their value,
and exp turns an absolute error of its argument into a relative one.
"""
import math

import numpy as np
import pytest
import torch

from federated_amd import client_ops as ops

pytestmark = pytest.mark.gpu

U32 = torch.finfo(torch.float32).eps / 2
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
COUNTS = [5, 0, 1, 130, 17]  # an empty client, single rows, tiles that end inside


def unit(dtype):
  return torch.finfo(dtype).eps / 2


def tiny(dtype):  # half the spacing of the subnormals
  return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def rand(rng, shape, dtype, scale=1.0, gpu="cuda"):
  return (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)) * scale).to(gpu).to(dtype)


def flat_params(rng, clients, sizes, dtype, scale, shared=False, pad=3):
  """Views of `sizes` in flat rows [clients, P] (P odd), as a client's parameters lie."""
  total = sum(int(np.prod(s)) for s in sizes) + pad
  total += 1 - total % 2
  rows = rand(rng, (1 if shared else clients, total), dtype, scale).expand(clients, total)
  views, at = [], 1  # an odd first offset: no 16-byte alignment
  for s in sizes:
    n = int(np.prod(s))
    views.append(rows[:, at:at + n].unflatten(1, tuple(s)) if len(s) > 1 else rows[:, at:at + n])
    at += n
  return views


def spans(counts):
  ends = np.cumsum(counts)
  return [(int(e - c), int(e)) for e, c in zip(ends, counts)]


def check(got, want, tol, what):
  got = got.detach().double().cpu()
  want, tol = want.double().cpu(), torch.as_tensor(tol).double().cpu()
  assert got.shape == want.shape, what
  bad = ~((got - want).abs() <= tol)
  assert not bad.any(), "%s: %d of %d off, worst %.3g against %.3g" % (
      what, int(bad.sum()), bad.numel(), float((got - want).abs().max()),
      float(torch.broadcast_to(tol, got.shape)[(got - want).abs() == (got - want).abs().max()].max()))


# --- layer norm ------------------------------------------------------------------


def norm_reference(x, w, b, counts, eps, dy=None, residual=None):
  x = x.double().cpu()
  n, d = x.shape
  mu = x.mean(1)
  s = 1.0 / torch.sqrt(((x - mu[:, None]) ** 2).mean(1) + eps)
  xh = (x - mu[:, None]) * s[:, None]
  client = torch.from_numpy(np.repeat(np.arange(len(counts)), counts))
  g = torch.ones(n, d, dtype=torch.float64) if w is None else w.double().cpu()[client]
  y = xh * g + (0 if b is None else b.double().cpu()[client])
  out = dict(y=y, mean=mu, rstd=s, xh=xh, g=g)
  if dy is not None:
    dy = dy.double().cpu()
    a = dy * g
    dx = s[:, None] * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    out["dx"] = dx if residual is None else dx + residual.double().cpu()
    out["dw"] = torch.stack([(dy * xh)[lo:hi].sum(0) for lo, hi in spans(counts)])
    out["db"] = torch.stack([dy[lo:hi].sum(0) for lo, hi in spans(counts)])
  return out


def norm_tolerances(ref, x, b, dim, dtype, counts=None, dy=None, residual=None):
  x = x.double().cpu()
  # a thread adds at most dim / 64 + 16 terms, and the threads join in 8 steps
  depth = dim / 64 + 24
  s = ref["rstd"]
  e_mean = depth * U32 * x.abs().mean(1) + U32 * ref["mean"].abs()
  # xh = (x - mu) s: the mean's error, a subtraction, and s (relative error: half the
  # variance's, which is depth + 2 roundings plus the mean's error to first order, and
  # four roundings of division, root, sum, product)
  rel_s = (depth + 8) * U32 + s * e_mean
  e_xh = s[:, None] * (e_mean[:, None] + U32 * (x - ref["mean"][:, None]).abs()) + ref["xh"].abs() * (
      rel_s[:, None] + 2 * U32)
  bias = 0 if b is None else float(b.abs().max())
  tol = dict(mean=e_mean, rstd=s * rel_s,
             y=ref["g"].abs() * e_xh + (unit(dtype) + 3 * U32) * (ref["y"].abs() + bias * 2 * U32) + tiny(dtype) +
             2 * U32 * ((ref["xh"] * ref["g"]).abs() + bias))
  if dy is not None:
    dy = dy.double().cpu()
    a = (dy * ref["g"]).abs()
    res = 0 if residual is None else residual.double().cpu().abs()
    xh = ref["xh"].abs()
    # a, its mean and xh mean(a xh) each with their own roundings
    e_m0 = (depth + 2) * U32 * a.mean(1, keepdim=True)
    e_m1 = (depth + 3) * U32 * (a * xh).mean(1, keepdim=True) + (a * e_xh).mean(1, keepdim=True)
    m0, m1 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    inner = a + m0 + xh * m1
    e_dx = s[:, None] * (e_m0 + xh * e_m1 + e_xh * m1 + 5 * U32 * inner) + rel_s[:, None] * s[:, None] * inner
    tol["dx"] = e_dx + unit(dtype) * ref["dx"].abs() + 2 * U32 * (res + ref["dx"].abs()) + tiny(dtype)
    tol["dw"] = torch.stack([((hi - lo + 4) * U32 * (dy.abs() * xh)[lo:hi] + (dy.abs() * e_xh)[lo:hi]).sum(0)
                             for lo, hi in spans(counts)])
    tol["db"] = torch.stack([((hi - lo + 4) * U32 * dy.abs()[lo:hi]).sum(0) for lo, hi in spans(counts)])
  return tol


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [1, 7, 96, 511, 670, 1024, 1027, 2048, 4096, 5000, 8193, 17000])
def test_layer_norm_forward_and_backward(gpu, dtype, dim):
  rng = np.random.default_rng(dim)
  counts = COUNTS if dim < 4096 else [3, 0, 70]
  n = sum(counts)
  batch = ops.ClientBatch(counts)
  x = rand(rng, (n, dim), dtype) + rand(rng, (n, 1), dtype)
  w, b = flat_params(rng, len(counts), [(dim,), (dim,)], dtype, 0.5)
  dy, res = rand(rng, (n, dim), dtype, 0.3), rand(rng, (n, dim), dtype)
  y, mean, rstd = ops.layer_norm(x, w, b, batch)
  rows = torch.full((len(counts), 2 * dim + 1), 7.0, device=gpu)
  dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, batch, residual=res, dweight=rows[:, 1:dim + 1],
                                       dbias=rows[:, dim + 1:])
  ref = norm_reference(x, w, b, counts, 1e-5, dy, res)
  tol = norm_tolerances(ref, x, b, dim, dtype, counts, dy, res)
  for name, got in dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db).items():
    check(got, ref[name], tol[name], name)
  assert (rows[:, 0] == 7.0).all()  # the row's other parameters are not touched
  assert (dw[1] == 0).all() and (db[1] == 0).all()  # the client without rows


@pytest.mark.parametrize("shared", [False, True], ids=["own", "shared"])
def test_layer_norm_options(gpu, shared):
  """Row strides, one weight for all clients, no weight or bias, accumulation, rows behind."""
  rng = np.random.default_rng(3)
  dim, counts = 130, [4, 9]
  n = sum(counts)
  batch = ops.ClientBatch(counts)
  wide = rand(rng, (n + 5, dim + 7), torch.bfloat16)
  wide[n:] = math.nan
  x = wide[:, 3:3 + dim]
  w, b = flat_params(rng, 2, [(dim,), (dim,)], torch.bfloat16, 0.5, shared=shared)
  out = torch.full((n + 5, dim + 1), 5.0, dtype=torch.bfloat16, device=gpu)
  y, mean, rstd = ops.layer_norm(x, w, b, batch, out=out[:, :dim])
  ref = norm_reference(x[:n], w, b, counts, 1e-5)
  check(y[:n], ref["y"], norm_tolerances(ref, x[:n], b, dim, torch.bfloat16)["y"], "y")
  assert (out[n:] == 5.0).all() and (out[:, dim] == 5.0).all()
  y2, _, _ = ops.layer_norm(x, None, None, batch)
  ref2 = norm_reference(x[:n], None, None, counts, 1e-5)
  check(y2[:n], ref2["y"], norm_tolerances(ref2, x[:n], None, dim, torch.bfloat16)["y"], "bare")
  assert (y2[n:] == 0).all()
  dy = rand(rng, (n, dim), torch.bfloat16)
  _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, batch)
  dw2, db2 = dw.clone(), db.clone()
  ops.layer_norm_backward(dy, x, mean, rstd, w, batch, dweight=dw2, dbias=db2, accumulate=True)
  check(dw2, 2 * dw, 4 * n * U32 * dw.abs().double().cpu().max() + 1e-30, "accumulated")
  check(db2, 2 * db, 4 * n * U32 * db.abs().double().cpu().max() + 1e-30, "accumulated bias")


def test_layer_norm_constant_rows_and_nan(gpu):
  """A constant row's variance is zero (y = bias); a NaN stays in its row and client."""
  batch = ops.ClientBatch([2, 2])
  x = torch.full((4, 64), 3.0, device=gpu)
  x[3, 5] = math.nan
  w = torch.ones(2, 64, device=gpu)
  b = torch.full((2, 64), 0.5, device=gpu)
  y, mean, rstd = ops.layer_norm(x, w, b, batch)
  assert (y[:3] == 0.5).all() and y[3].isnan().all()
  _, dw, _ = ops.layer_norm_backward(torch.ones_like(x), x, mean, rstd, w, batch)
  assert (dw[0] == 0).all() and dw[1].isnan().all()


# --- linear ----------------------------------------------------------------------

ACTS = {
    None: (lambda z: z, lambda z: torch.ones_like(z)),
    "relu": (lambda z: z.clamp(min=0), lambda z: (z > 0).double()),
    "gelu": (lambda z: 0.5 * z * torch.special.erfc(-z / math.sqrt(2)),
             lambda z: 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
    "silu": (lambda z: z * torch.sigmoid(z),
             lambda z: torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))),
}


def linear_reference(x, w, counts):
  """(z, bound of its float32 sum) per row."""
  x, w = x.double().cpu(), w.double().cpu()
  z, mag = [], []
  for c, (lo, hi) in enumerate(spans(counts)):
    z.append(x[lo:hi] @ w[c].t())
    mag.append(x[lo:hi].abs() @ w[c].abs().t())
  return torch.cat(z), torch.cat(mag) * (2 * x.shape[1] * U32)


def check_linear(gpu, rng, counts, k, m, dtype, act, shared=False, scale=None, behind=0):
  n = sum(counts)
  batch = ops.ClientBatch(counts)
  x = rand(rng, (n + behind, k), dtype)
  dz = rand(rng, (n + behind, m), dtype, 0.5)
  if behind:
    x[n:], dz[n:] = math.nan, math.nan
  w, b = flat_params(rng, len(counts), [(m, k), (m,)], dtype, scale or 1 / math.sqrt(k), shared=shared)
  res, before = rand(rng, (n, m), dtype), rand(rng, (n, k), dtype)
  below = rand(rng, (n, k), dtype)
  client = torch.from_numpy(np.repeat(np.arange(len(counts)), counts))
  f, slope = ACTS[act]
  u = unit(dtype)

  y, z = ops.linear(x, w, b, batch, activation=act, residual=res if behind == 0 else None, preactivation=True)
  zr, ez = linear_reference(x[:n], w, counts)
  zr = zr + b.double().cpu()[client]
  ez = ez + 2 * U32 * zr.abs()
  check(z[:n], zr, ez + u * (zr.abs() + ez) + tiny(dtype), "z")
  yr = f(zr) + (res.double().cpu() if behind == 0 else 0)
  # the activations' slopes stay below 1.13; their own evaluation a few roundings of z
  ey = 1.13 * ez + 16 * U32 * zr.abs() + 2 * U32 * (yr.abs() + 4)
  check(y[:n], yr, ey + u * (yr.abs() + ey) + tiny(dtype), "y")
  if behind:
    assert (y[n:] == 0).all() and (z[n:] == 0).all()

  dx = ops.linear_backward_input(dz, w, batch, preactivation=before if act else None, activation=act,
                                 residual=below if behind == 0 else None)
  wt = w.double().cpu().transpose(1, 2)
  gr, eg = linear_reference(dz[:n], wt, counts)
  sl = slope(before.double().cpu()) if act else torch.ones(n, k, dtype=torch.float64)
  want = gr * sl + (below.double().cpu() if behind == 0 else 0)
  e = eg * sl.abs() + 16 * U32 * gr.abs() * (1 + before.double().cpu().abs()) + 2 * U32 * want.abs()
  check(dx[:n], want, e + u * (want.abs() + e) + tiny(dtype), "dx")

  rows = torch.full((len(counts), m * k + m + 2), 3.0, device=gpu)
  dw, db = ops.linear_backward_weight(dz, x, batch, dweight=rows[:, 1:1 + m * k].unflatten(1, (m, k)),
                                      dbias=rows[:, 1 + m * k:1 + m * k + m])
  for c, (lo, hi) in enumerate(spans(counts)):
    d, xx = dz[lo:hi].double().cpu(), x[lo:hi].double().cpu()
    check(dw[c], d.t() @ xx, 2 * max(1, hi - lo) * U32 * (d.abs().t() @ xx.abs()), "dw of client %d" % c)
    check(db[c], d.sum(0), 2 * max(1, hi - lo) * U32 * d.abs().sum(0), "db of client %d" % c)
  assert (rows[:, 0] == 3.0).all() and (rows[:, -1] == 3.0).all()
  return rows


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k,m", [(1, 1), (5, 3), (64, 128), (96, 131), (130, 64), (257, 300), (670, 96), (1024, 17)])
def test_linear_sizes(gpu, dtype, k, m):
  rng = np.random.default_rng(k * 1000 + m)
  check_linear(gpu, rng, COUNTS, k, m, dtype, [None, "relu", "gelu", "silu"][(k + m) % 4])


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_activations(gpu, dtype, act):
  check_linear(gpu, np.random.default_rng(11), [33, 2], 40, 72, dtype, act, scale=0.7)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts", [[1], [1] * 40, [0, 0, 3], [16, 15, 17], [129], [300, 1], [700]])
def test_linear_row_counts(gpu, dtype, counts):
  check_linear(gpu, np.random.default_rng(sum(counts)), counts, 136, 200, dtype, "silu")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_long_contractions(gpu, dtype):
  """Few rows over a long axis, and many rows into a small weight (splits, where taken)."""
  check_linear(gpu, np.random.default_rng(1), [2, 1], 4100, 36, dtype, "gelu")
  check_linear(gpu, np.random.default_rng(2), [1], 72, 4099, dtype, None)
  check_linear(gpu, np.random.default_rng(3), [5000, 3], 24, 40, dtype, "relu")


@pytest.mark.parametrize("rows,splits", [(32, 1), (32, 5), (128, 1), (128, 3), (256, 1), (256, 2), (128, 64), (32, 2)])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_every_plan(gpu, monkeypatch, dtype, rows, splits):
  """Each tile height and split of the contraction, whatever the sizes would choose: odd
  sizes (16-bit rows at odd addresses), sizes at multiples of 4 bytes, whole tiles."""
  monkeypatch.setattr(ops, "_plan", lambda tiles, steps, longest, size, aligned: (
      128 if rows == 256 and (size == 4 or not aligned) else rows, splits))
  # odd rows as they lie, or copied to whole vectors first
  monkeypatch.setattr(ops, "_estimate", lambda tiles, steps, longest, size, aligned: (
      1e9 if aligned == (splits == 1) else 1.0, rows, splits))
  rng = np.random.default_rng(rows + splits)
  check_linear(gpu, rng, [40, 0, 1, 300], 131, 77, dtype, "gelu")
  check_linear(gpu, rng, [40, 0, 1, 300], 131, 77, dtype, "relu", shared=True, behind=3)
  check_linear(gpu, rng, [257, 3], 134, 260, dtype, None)
  check_linear(gpu, rng, [256, 128, 31], 256, 256, dtype, "silu", shared=True)
  check_linear(gpu, rng, [5], 4, 2, dtype, "relu")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_shared_weight_and_rows_behind(gpu, dtype):
  rng = np.random.default_rng(21)
  check_linear(gpu, rng, [20, 0, 45], 150, 70, dtype, "gelu", shared=True)
  check_linear(gpu, rng, [20, 0, 45], 150, 70, dtype, None, behind=9)


def test_linear_strides_and_accumulation(gpu):
  rng = np.random.default_rng(5)
  counts, k, m = [7, 140], 48, 56
  n = sum(counts)
  batch = ops.ClientBatch(counts)
  xw, wide = rand(rng, (n, k + 5), torch.bfloat16), rand(rng, (2, m + 1, k + 9), torch.bfloat16, 0.2)
  x, w = xw[:, 2:2 + k], wide[:, 1:, 3:3 + k]
  out = torch.full((n, m + 3), 9.0, dtype=torch.bfloat16, device=gpu)
  y = ops.linear(x, w, None, batch, out=out[:, 1:1 + m])
  assert torch.equal(y, ops.linear(x.contiguous(), w.contiguous(), None, batch))
  assert (out[:, 0] == 9.0).all() and (out[:, m + 1:] == 9.0).all()
  dz = rand(rng, (n, m), torch.bfloat16)
  dw, db = ops.linear_backward_weight(dz, x, batch)
  dw2, db2 = dw.clone(), db.clone()
  ops.linear_backward_weight(dz, x, batch, dweight=dw2, dbias=db2, accumulate=True)
  assert torch.equal(dw2, 2 * dw) and torch.equal(db2, 2 * db)
  dw3, none = ops.linear_backward_weight(dz, x, batch, bias=False)
  assert none is None and torch.equal(dw3, dw)


def test_linear_nan_and_infinity_stay_in_their_rows(gpu):
  batch = ops.ClientBatch([3, 3])
  x = torch.ones(6, 40, device=gpu)
  x[1, 3], x[4, 0] = math.nan, math.inf
  w = torch.ones(2, 50, 40, device=gpu)
  y = ops.linear(x, w, None, batch, activation="relu")
  assert y[1].isnan().all() and (y[4] == math.inf).all()
  assert (y[[0, 2, 3, 5]] == 40).all()
  dw, db = ops.linear_backward_weight(torch.ones(6, 50, device=gpu), x, batch)
  assert dw[0, :, 3].isnan().all() and (dw[0, :, :3] == 3).all() and (dw[1, :, 0] == math.inf).all()
  assert (db == 3).all()


# --- top logits --------------------------------------------------------------------


def top_reference(logits, k, temperature=1.0):
  a = logits.double().cpu()
  key = torch.where(a.isnan(), -math.inf, a)
  # NaN below every number, -inf included: two stable passes
  order = torch.sort(torch.where(a.isnan(), 1, 0), dim=1, stable=True).indices
  by = torch.sort(torch.gather(key, 1, order), dim=1, descending=True, stable=True).indices
  return torch.gather(order, 1, by)[:, :k], torch.logsumexp(a / temperature, 1)


def check_top(logits, k, temperature=1.0):
  index, values, lse = ops.top_logits(logits, k, temperature)
  want, want_lse = top_reference(logits, k, temperature)
  assert torch.equal(index.long().cpu(), want)
  got = torch.gather(logits, 1, index.long())
  assert torch.equal(values.nan_to_num(nan=7e4), got.nan_to_num(nan=7e4))
  finite = want_lse.isfinite()
  assert torch.equal(lse.cpu()[~finite].double().nan_to_num(nan=5.0), want_lse[~finite].nan_to_num(nan=5.0))
  a = logits.double().cpu()[finite]
  if a.numel():
    # the sum: vocab / 1024 + 16 + 20 additions of terms whose exponents are off by two
    # roundings of at most the row's span; then the maximum's product and the log
    span = torch.where(a.isinf(), 0.0, a / temperature).abs().amax(1)
    tol = (a.shape[1] / 1024 + 48 + 4 * span) * 2 * U32
    check(lse[finite.to(lse.device)], want_lse[finite], tol, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab,k", [(1, 1), (7, 7), (100, 3), (1000, 64), (1025, 1024), (10004, 10), (10004, 1000),
                                     (40000, 128), (131072, 64)])
def test_top_logits_sizes(gpu, dtype, vocab, k):
  rng = np.random.default_rng(vocab + k)
  check_top(rand(rng, (5, vocab), dtype, 3.0), k, 1.0 if k % 2 else 1.7)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_top_logits_ties_infinities_nan(gpu, dtype):
  """Whole rows of ties (more than are ranked at once), signed zeros, -inf, NaN, +inf."""
  rng = np.random.default_rng(4)
  v = 9001
  x = rand(rng, (12, v), dtype)
  x[0] = 1.0
  x[1] = -math.inf
  x[2] = math.nan
  x[3, 100:] = -math.inf
  x[4] = 0.0
  x[4, ::2] = -0.0
  x[5] = torch.round(x[5].float()).to(dtype)
  x[6, 17] = math.nan
  x[7, 50], x[7, 4000] = math.inf, math.inf
  x[8] = -math.inf
  x[8, 8999] = 2.0
  x[9] = torch.arange(v, device=gpu).flip(0).to(dtype) / 64
  x[10, :5000] = math.nan
  x[11] = (torch.arange(v, device=gpu) % 2).to(dtype)
  for k in (1, 33, 700):
    check_top(x, k)


def test_top_logits_strides_and_no_rows(gpu):
  rng = np.random.default_rng(9)
  wide = rand(rng, (6, 3000), torch.bfloat16)
  check_top(wide[::2, 5:2505], 20)
  index, values, lse = ops.top_logits(wide[:0], 4)
  assert index.shape == (0, 4) and values.shape == (0, 4) and lse.shape == (0,)


# --- distillation --------------------------------------------------------------------


def distill_reference(logits, index, values, counts, tau, teacher_lse=None, weights=None, dloss=None):
  """(loss, gradient, bound of each) in float64, row by row."""
  n = sum(counts)
  s = logits[:n].double().cpu() / tau
  v = s.shape[1]
  loss = torch.zeros(len(counts), dtype=torch.float64)
  e_loss = torch.zeros(len(counts), dtype=torch.float64)
  grad, e_grad = torch.zeros_like(s), torch.zeros_like(s)
  for c, (lo, hi) in enumerate(spans(counts)):
    for r in range(lo, hi):
      w = 1.0 / (hi - lo) if weights is None else float(weights[r])
      entries = [(int(j), float(t) / tau) for j, t in zip(index[r].cpu(), values[r].double().cpu())
                 if 0 <= int(j) < v and float(t) != -math.inf]
      if not entries or w == 0:
        continue
      t = torch.tensor([t for _, t in entries], dtype=torch.float64)
      j = torch.tensor([j for j, _ in entries])
      L = torch.logsumexp(t, 0) if teacher_lse is None else float(teacher_lse[r])
      p = torch.exp(t - L)
      lse = torch.logsumexp(s[r], 0)
      q = torch.exp(s[r] - lse)
      term = p * (torch.log(p) - (s[r][j] - lse))
      loss[c] += w * tau * tau * term.sum()
      pr = torch.zeros(v, dtype=torch.float64).index_add(0, j, p)
      scale = w * tau * (1.0 if dloss is None else float(dloss[c]))
      grad[r] = scale * (p.sum() * q - pr)
      # errors of exponents: the arguments' roundings (a few u of their size), the
      # log-sum-exp's own sum (vocab / 256 + 32 additions)
      size = float(s[r][s[r].isfinite()].abs().max() + t.abs().max() + lse.abs() + abs(float(L)))
      d = (6 * size + v / 256 + 2 * len(t) + 48) * 2 * U32
      mag = (p * (torch.log(p).abs() + (s[r][j] - lse).abs())).sum() + 2 * p.sum()
      e_loss[c] += w * tau * tau * float(mag) * (2 * d + (hi - lo + 8) * U32)
      e_grad[r] = abs(scale) * (p.sum() * q + pr) * (2 * d + 8 * U32)
  return loss, grad, e_loss, e_grad


def teacher_rows(rng, n, v, k, pad=0.25, gpu="cuda"):
  index = torch.stack([torch.from_numpy(rng.permutation(v)[:k] if k <= v else rng.integers(0, v, k)) for _ in range(n)])
  values = torch.from_numpy(np.sort(rng.standard_normal((n, k)) * 3)[:, ::-1].copy()).float()
  if pad:
    index[torch.from_numpy(rng.random((n, k)) < pad)] = -1
  return index.int().to(gpu), values.to(gpu)


def check_distill(logits, index, values, counts, tau=1.0, **kw):
  batch = ops.ClientBatch(counts)
  dtype, n = logits.dtype, sum(counts)
  weights, teacher_lse = kw.get("row_weights"), kw.get("teacher_lse")
  loss, grad, el, eg = distill_reference(logits, index, values, counts, tau, teacher_lse, weights)
  el, eg = el + 1e-30, eg + unit(dtype) * (grad.abs() + eg) + tiny(dtype)
  got, lse = ops.distillation(logits, index, values, batch, temperature=tau, **kw)
  check(got, loss, el, "loss")
  fused, dfused = ops.distillation_with_gradient(logits, index, values, batch, temperature=tau, **kw)
  check(fused, loss, el, "fused loss")
  check(dfused[:n], grad, eg, "fused gradient")
  dback = ops.distillation_backward(logits, lse, index, values, batch, temperature=tau, **kw)
  check(dback[:n], grad, eg, "gradient")
  dloss = torch.linspace(-1.0, 2.0, len(counts), device=logits.device)
  _, grad2, _, eg2 = distill_reference(logits, index, values, counts, tau, teacher_lse, weights, dloss)
  check(ops.distillation_backward(logits, lse, index, values, batch, temperature=tau, dloss=dloss, **kw)[:n], grad2,
        eg2 + unit(dtype) * (grad2.abs() + eg2) + tiny(dtype), "scaled gradient")
  copy = logits.clone()
  _, inplace = ops.distillation_with_gradient(copy, index, values, batch, temperature=tau, out=copy, **kw)
  assert torch.equal(inplace[:n], dfused[:n])
  copy = logits.clone()
  assert torch.equal(ops.distillation_backward(copy, lse, index, values, batch, temperature=tau, out=copy, **kw)[:n],
                     dback[:n])
  return dfused


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab,k", [(1, 1), (5, 5), (50, 8), (1000, 32), (10004, 64), (33333, 1)])
def test_distillation_sizes(gpu, dtype, vocab, k):
  rng = np.random.default_rng(vocab * 7 + k)
  counts = [3, 0, 4, 1]
  logits = rand(rng, (8, vocab), dtype, 2.0)
  index, values = teacher_rows(rng, 8, vocab, k)
  check_distill(logits, index, values, counts, tau=2.0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distillation_options(gpu, dtype):
  """The teacher's own lse, row weights (one of them zero over NaN logits), -inf values."""
  rng = np.random.default_rng(31)
  counts, v, k = [2, 5], 700, 16
  logits = rand(rng, (7, v), dtype, 2.0)
  index, values = teacher_rows(rng, 7, v, k)
  values[1, 3:] = -math.inf
  lse = torch.logsumexp(values / 1.5, 1) + 0.3
  check_distill(logits, index, values, counts, tau=1.5, teacher_lse=lse)
  weights = torch.tensor([0.5, 0.0, 1.0, 2.0, 0.0, 1.0, 0.25], device=gpu)
  logits[1] = math.nan
  grad = check_distill(logits, index, values, counts, tau=0.7, row_weights=weights)
  assert (grad[1] == 0).all() and (grad[4] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distillation_empty_rows_repeats_and_masks(gpu, dtype):
  """Rows of nothing but padding (over NaN logits), an index that comes twice, indices
  outside the vocabulary, student logits of -inf."""
  rng = np.random.default_rng(8)
  counts, v, k = [4, 1, 3], 300, 8
  logits = rand(rng, (8, v), dtype, 2.0)
  index, values = teacher_rows(rng, 8, v, k, pad=0)
  index[0] = -1
  logits[0] = math.nan
  index[4] = v  # the second client has nothing
  index[1, 2], index[1, 6] = index[1, 0], index[1, 0]
  index[2, :4] = torch.tensor([v, -7, 2**31 - 1, -2**31])
  mask = torch.ones(v, dtype=torch.bool, device=gpu)
  mask[index[3].long()] = False
  logits[3] = torch.where(mask, -math.inf, logits[3])
  grad = check_distill(logits, index, values, counts)
  assert (grad[0] == 0).all() and (grad[4] == 0).all()
  # an index repeated: the same as one entry of the summed probability
  batch = ops.ClientBatch([1])
  one = torch.tensor([[5, 5]], dtype=torch.int32, device=gpu)
  l2, _ = ops.distillation_with_gradient(logits[5:6], one, torch.zeros(1, 2, device=gpu), batch)
  g1 = ops.distillation_with_gradient(logits[5:6], one[:, :1].contiguous(), torch.zeros(1, 1, device=gpu), batch)
  assert abs(float(l2) - (float(g1[0]) - math.log(2))) < 1e-5


def test_distillation_student_without_distribution(gpu):
  """All of a row's logits -inf: an infinite loss, and the teacher's side of the gradient."""
  batch = ops.ClientBatch([1])
  logits = torch.full((1, 40), -math.inf, device=gpu)
  index = torch.tensor([[3, 9]], dtype=torch.int32, device=gpu)
  loss, grad = ops.distillation_with_gradient(logits, index, torch.zeros(1, 2, device=gpu), batch)
  assert float(loss) == math.inf
  want = torch.zeros(1, 40)
  want[0, [3, 9]] = -0.5
  check(grad, want, 4 * U32, "gradient")


def test_distillation_gradient_by_differences(gpu):
  """Central differences of the float32 loss: step h = 2^-6 leaves h^2 / 6 of a third
  derivative below 2 w tau^2 / tau^3, and 2 u |loss| / h from the loss's own rounding."""
  rng = np.random.default_rng(77)
  v, tau, h = 24, 1.5, 2.0**-6
  batch = ops.ClientBatch([1, 1])
  logits = rand(rng, (2, v), torch.float32)
  index, values = teacher_rows(rng, 2, v, 4, pad=0)
  loss, grad = ops.distillation_with_gradient(logits, index, values, batch, temperature=tau)
  for j in range(v):
    up, down = logits.clone(), logits.clone()
    up[:, j] += h
    down[:, j] -= h
    a = ops.distillation(up, index, values, batch, temperature=tau)[0].double()
    b = ops.distillation(down, index, values, batch, temperature=tau)[0].double()
    tol = 2 / tau * h * h / 6 + (64 * U32 * (loss.double().abs() + 10)) / h
    check((a - b) / (2 * h), grad[:, j], tol.cpu(), "column %d" % j)


# --- together ------------------------------------------------------------------------


class Step:
  """One client step of a residual block and a head under a teacher's top logits: the
  operators as they are used, gradients in the clients' flat rows."""

  def __init__(self, rng, counts, dtype, d=40, hidden=88, v=121, shared=False, gpu="cuda"):
    self.counts, self.dtype = counts, dtype
    self.sizes = [(d,), (d,), (hidden, d), (hidden,), (d, hidden), (d,), (v, d), (v,)]
    self.P = sum(int(np.prod(s)) for s in self.sizes)
    c = len(counts)
    rows = rand(rng, (1 if shared else c, self.P), dtype, 0.2).expand(c, self.P)
    self.params = self.views(rows)
    self.update = torch.zeros(c, self.P, device=gpu)
    self.grads = self.views(self.update)
    n = sum(counts)
    self.batch = ops.ClientBatch(counts)
    self.x = rand(rng, (n, d), dtype)
    teacher = rand(rng, (n, v), torch.float32, 3.0)
    self.index, self.values, self.lse = ops.top_logits(teacher, 12, temperature=2.0)

  def views(self, rows):
    out, at = [], 0
    for s in self.sizes:
      k = int(np.prod(s))
      out.append(rows[:, at:at + k].unflatten(1, s) if len(s) > 1 else rows[:, at:at + k])
      at += k
    return out

  def run(self):
    g, b, w1, b1, w2, b2, w3, b3 = self.params
    dg, db, dw1, db1, dw2, db2, dw3, db3 = self.grads
    batch = self.batch
    h, mean, rstd = ops.layer_norm(self.x, g, b, batch)
    a, z = ops.linear(h, w1, b1, batch, activation="gelu", preactivation=True)
    y = ops.linear(a, w2, b2, batch, residual=self.x)
    logits = ops.linear(y, w3, b3, batch)
    loss, dlogits = ops.distillation_with_gradient(logits, self.index, self.values, batch, temperature=2.0,
                                                   teacher_lse=self.lse, out=logits)
    ops.linear_backward_weight(dlogits, y, batch, dweight=dw3, dbias=db3)
    dy = ops.linear_backward_input(dlogits, w3, batch)
    ops.linear_backward_weight(dy, a, batch, dweight=dw2, dbias=db2)
    dz = ops.linear_backward_input(dy, w2, batch, preactivation=z, activation="gelu")
    ops.linear_backward_weight(dz, h, batch, dweight=dw1, dbias=db1)
    dh = ops.linear_backward_input(dz, w1, batch)
    dx, _, _ = ops.layer_norm_backward(dh, self.x, mean, rstd, g, batch, residual=dy, dweight=dg, dbias=db)
    return loss, dx

  def autograd(self):
    """The same step in float64 by torch's own differentiation, client by client."""
    params = [p.double().cpu().clone().requires_grad_() for p in self.params]
    x = self.x.double().cpu().requires_grad_()
    losses = []
    for c, (lo, hi) in enumerate(spans(self.counts)):
      if lo == hi:
        losses.append(torch.zeros((), dtype=torch.float64))
        continue
      g, b, w1, b1, w2, b2, w3, b3 = [p[c] for p in params]
      xc = x[lo:hi]
      hc = torch.nn.functional.layer_norm(xc, (xc.shape[1],), g, b)
      y = torch.nn.functional.gelu(hc @ w1.t() + b1) @ w2.t() + b2 + xc
      logq = torch.log_softmax((y @ w3.t() + b3) / 2.0, 1)
      p = torch.exp(self.values[lo:hi].double().cpu() / 2.0 - self.lse[lo:hi].double().cpu()[:, None])
      losses.append(4.0 * (p * (torch.log(p) - torch.gather(logq, 1, self.index[lo:hi].long().cpu()))).sum(1).mean())
    loss = torch.stack(losses)
    grads = torch.autograd.grad(loss.sum(), params + [x])
    return loss, grads[-1], grads[:-1]


@pytest.mark.parametrize("shared", [False, True], ids=["own", "shared"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_step_gradients(gpu, dtype, shared):
  """The whole step against float64 autograd.  Every stored activation and gradient is
  rounded to the type once; a parameter's gradient passes at most 10 such roundings,
  each relative to its own tensor, so 10 u (plus float32's sums) of the gradient's
  norm, four times for the products of perturbed factors, bounds its error's norm."""
  step = Step(np.random.default_rng(6), [12, 0, 33, 1], dtype, shared=shared)
  loss, dx = step.run()
  want_loss, want_dx, want = step.autograd()
  bound = 4 * (10 * unit(dtype) + 400 * U32)
  for got, ref in [(loss, want_loss), (dx, want_dx)] + list(zip(step.grads, want)):
    ref = ref.double()
    err = (got.double().cpu() - ref).norm()
    assert float(err) <= bound * float(ref.norm()), (got.shape, float(err), float(ref.norm()))
  assert (step.update[1] == 0).all()


def test_step_feeds_the_codec(gpu):
  """The step's rows go through the default aggregator as they lie, bit for bit the
  oracle's round."""
  from federated_amd.aggregators import quantize_encode  # pylint: disable=g-import-not-at-top
  from oracle import aggregators as oagg  # pylint: disable=g-import-not-at-top
  step = Step(np.random.default_rng(16), [9, 4, 20], torch.bfloat16)
  step.run()
  step.update.mul_(50.0)
  seeds = np.array([[1, 2], [3, 4], [5, 6]], np.int64)
  process = quantize_encode.QuantizeEncodeFactory(0.05, rounding_type="stochastic").create((np.float32, (step.P,)))
  out = process.next(process.initialize(), step.update, seeds=seeds)
  want, meas, _ = oagg.quantize_encode_next([r.cpu().numpy() for r in step.update], 0.05, "stochastic", seeds=seeds)
  assert np.array_equal(out.result.cpu().numpy(), want)
  assert out.measurements["avg_bitrate"] == meas["avg_bitrate"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step_twice_is_bitwise_equal_and_graph_replays(gpu, dtype):
  """Two eager runs agree bit for bit; a captured step replays with new inputs in
  place, eager work between the replays; two graphs share nothing."""
  step = Step(np.random.default_rng(26), [40, 3, 0, 77], dtype)
  other = Step(np.random.default_rng(27), [15, 60], dtype)

  def eager(s):
    loss, dx = s.run()
    torch.cuda.synchronize()
    return [t.clone() for t in (loss, dx, s.update)]

  a, b = eager(step), eager(step)
  assert all(torch.equal(p, q) for p, q in zip(a, b))
  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  graphs = []
  with torch.cuda.stream(stream):
    for s in (step, other):
      s.run()
    torch.cuda.synchronize()
    for s in (step, other):
      g = torch.cuda.CUDAGraph()
      with torch.cuda.graph(g, stream=stream):
        out = s.run()
      graphs.append((g, s, out))
  torch.cuda.synchronize()
  rng = np.random.default_rng(5)
  for _ in range(4):
    for g, s, out in graphs:
      s.x.copy_(rand(rng, tuple(s.x.shape), dtype))
      want = eager(s)
      s.update.fill_(-1.0)
      g.replay()
      graphs[1 - [h[0] for h in graphs].index(g)][0].replay()  # the other graph right behind it
      torch.cuda.synchronize()
      assert all(torch.equal(p, q) for p, q in zip((out[0], out[1], s.update), want))


def test_step_on_another_stream(gpu):
  step = Step(np.random.default_rng(36), [25, 31], torch.bfloat16)
  loss, dx = step.run()
  want = [t.clone() for t in (loss, dx, step.update)]
  step.update.zero_()
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    loss, dx = step.run()
  s.synchronize()
  assert all(torch.equal(p, q) for p, q in zip((loss, dx, step.update), want))


def test_batches_without_rows(gpu):
  batch = ops.ClientBatch([0, 0])
  x = torch.empty(0, 8, device=gpu)
  w = torch.ones(2, 5, 8, device=gpu)
  y, _, _ = ops.layer_norm(x, None, None, batch)
  assert y.shape == (0, 8) and ops.linear(x, w, None, batch).shape == (0, 5)
  dw, db = ops.linear_backward_weight(torch.empty(0, 5, device=gpu), x, batch)
  assert (dw == 0).all() and (db == 0).all() and dw.shape == (2, 5, 8)
  assert ops.linear_backward_input(torch.empty(0, 5, device=gpu), w, batch).shape == (0, 8)
  idx = torch.empty(0, 3, dtype=torch.int32, device=gpu)
  loss, grad = ops.distillation_with_gradient(x, idx, torch.empty(0, 3, device=gpu), batch)
  assert (loss == 0).all() and grad.shape == (0, 8)
  st = torch.empty(0, device=gpu)
  _, dg, dbt = ops.layer_norm_backward(x, x, st, st, None, batch)
  assert (dg == 0).all() and (dbt == 0).all()


# --- refusals ------------------------------------------------------------------------


def test_batch_refusals(gpu):
  for bad in ([], [[1, 2]], [1.5], [-1, 2], [1 << 31]):
    with pytest.raises(ValueError):
      ops.ClientBatch(bad)
  with pytest.raises(ValueError):
    ops.ClientBatch([1], device="cpu")


def test_operator_refusals(gpu):
  batch = ops.ClientBatch([3, 2])
  x = torch.zeros(5, 8, device=gpu)
  w, b = torch.zeros(2, 6, 8, device=gpu), torch.zeros(2, 6, device=gpu)
  dz = torch.zeros(5, 6, device=gpu)
  idx = torch.zeros(5, 2, dtype=torch.int32, device=gpu)
  val = torch.zeros(5, 2, device=gpu)
  one = torch.zeros(1, device=gpu)
  st = torch.zeros(5, device=gpu)
  calls = [
      lambda: ops.layer_norm(x[:4], None, None, batch),  # too few rows
      lambda: ops.layer_norm(x.cpu(), None, None, batch),
      lambda: ops.layer_norm(x.double(), None, None, batch),
      lambda: ops.layer_norm(x.t().contiguous().t(), None, None, batch),
      lambda: ops.layer_norm(x[None], None, None, batch),
      lambda: ops.layer_norm(x, torch.zeros(2, 7, device=gpu), None, batch),
      lambda: ops.layer_norm(x, torch.zeros(3, 8, device=gpu), None, batch),
      lambda: ops.layer_norm(x, torch.zeros(2, 8, device=gpu).half(), None, batch),
      lambda: ops.layer_norm(x, None, None, batch, out=one.expand(5, 8)),
      lambda: ops.layer_norm_backward(x, x, st[:4], st, None, batch),
      lambda: ops.layer_norm_backward(x.half(), x, st, st, None, batch),
      lambda: ops.layer_norm_backward(x, x, st, st, None, batch, accumulate=True),
      lambda: ops.layer_norm_backward(x, x, st, st, None, batch, dweight=torch.zeros(8, device=gpu).expand(2, 8)),
      lambda: ops.linear(x, w, b, batch, activation="tanh"),
      lambda: ops.linear(x, w[:, :, :7], b, batch),
      lambda: ops.linear(x, w[:1], b, batch),
      lambda: ops.linear(x, w.half(), b, batch),
      lambda: ops.linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), b, batch),
      lambda: ops.linear(x, w, b[:, :5], batch),
      lambda: ops.linear(x, w, b, batch, residual=x),
      lambda: ops.linear(x, w, b, batch, out=torch.zeros(5, 7, device=gpu)),
      lambda: ops.linear_backward_input(dz, w, batch, activation="relu"),
      lambda: ops.linear_backward_input(dz, w, batch, preactivation=x),
      lambda: ops.linear_backward_input(x, w, batch),
      lambda: ops.linear_backward_weight(dz, x.half(), batch),
      lambda: ops.linear_backward_weight(dz, x, batch, dweight=w.half()),
      lambda: ops.linear_backward_weight(dz, x, batch, dweight=w[:1].expand(2, 6, 8)),
      lambda: ops.linear_backward_weight(dz, x, batch, accumulate=True),
      lambda: ops.linear_backward_weight(dz, x, batch, bias=False, dbias=b),
      lambda: ops.top_logits(x, 0),
      lambda: ops.top_logits(x, 9),
      lambda: ops.top_logits(torch.zeros(1, 2000, device=gpu), 1025),
      lambda: ops.top_logits(x, 2, temperature=0.0),
      lambda: ops.top_logits(x.cpu(), 2),
      lambda: ops.top_logits(x.int(), 2),
      lambda: ops.distillation(x, idx.long(), val, batch),
      lambda: ops.distillation(x, idx[:4], val, batch),
      lambda: ops.distillation(x, idx, val[:, :1], batch),
      lambda: ops.distillation(x, idx, val, batch, temperature=float("inf")),
      lambda: ops.distillation(x, idx, val, batch, teacher_lse=st[:3]),
      lambda: ops.distillation(x, idx, val, batch, row_weights=st.double()),
      lambda: ops.distillation(x, idx.cpu(), val, batch),
      lambda: ops.distillation(x, idx.repeat(1, 600), val.repeat(1, 600), batch),
      lambda: ops.distillation_backward(x, st[:2], idx, val, batch),
      lambda: ops.distillation_backward(x, st, idx, val, batch, dloss=one),
      lambda: ops.distillation_with_gradient(x, idx, val, batch, out=dz),
  ]
  for i, call in enumerate(calls):
    with pytest.raises(ValueError):
      call()
      pytest.fail("call %d was not refused" % i)


# --- limits: launch shapes, lowest values, wide strides, many clients, shared memory --------


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [1021, 1029, 2043, 4093, 5115, 10237, 16381, 20477, 32765, 65531, 65541])
def test_distillation_every_launch_shape(gpu, dtype, vocab):
  rng = np.random.default_rng(vocab)
  logits = rand(rng, (3, vocab), dtype, 2.0)
  index, values = teacher_rows(rng, 3, vocab, 5)
  check_distill(logits, index, values, [2, 1], tau=1.5)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab,k", [(4096, 32), (4097, 32), (2048, 33), (2049, 33), (513, 200), (32768, 128), (32769, 128),
                                     (32768, 129), (32771, 5), (70001, 1024)])
def test_top_logits_every_launch_shape(gpu, dtype, vocab, k):
  check_top(rand(np.random.default_rng(vocab + k), (3, vocab), dtype, 2.0), k, 1.3)


@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [96, 3001, 70001])
def test_rows_of_the_lowest_value(gpu, dtype, tau, vocab):
  """A mask of the type's lowest value over a whole row leaves a uniform softmax, over most
  of it one over the rest; a teacher whose values are all the lowest is uniform too.  A
  gradient is w tau (q - p): q by an exponential, a sum of vocab / 64 + 24 terms and a
  division, p by an exponential of a logarithm of 4."""
  low = torch.finfo(dtype).min
  logits = torch.full((3, vocab), low, dtype=dtype, device=gpu)
  logits[1, 7:11] = 0.0
  batch = ops.ClientBatch([2, 1])
  index = torch.tensor([[1, 8, 60, 95]] * 3, dtype=torch.int32, device=gpu)
  values = torch.zeros(3, 4, device=gpu)
  values[2] = torch.finfo(torch.float32).min
  q = torch.full((3, vocab), 1.0 / vocab, dtype=torch.float64)
  q[1] = 0.0
  q[1, 7:11] = 0.25
  grad = q.clone()
  grad[:, index[0].long().cpu()] -= 0.25
  w = torch.tensor([0.5, 0.5, 1.0], dtype=torch.float64)[:, None]
  grad = grad * w * tau
  tol = ((vocab / 64 + 24) * U32 * (q + 0.25) + 16 * U32) * tau + unit(dtype) * grad.abs() + tiny(dtype)
  loss, got = ops.distillation_with_gradient(logits, index, values, batch, temperature=tau)
  check(got, grad, tol, "gradient")
  loss2, lse = ops.distillation(logits, index, values, batch, temperature=tau)
  check(ops.distillation_backward(logits, lse, index, values, batch, temperature=tau), grad, tol, "gradient alone")
  assert torch.equal(loss, loss2)
  row = math.log(vocab / 4)  # of rows 0 and 2: p log(p / q)
  e = (vocab / 64 + 64) * U32 * tau * tau * (row + 2)
  check(loss[1:], torch.tensor([tau * tau * row]), e, "loss")
  top, _, top_lse = ops.top_logits(logits, 4, tau)
  assert top[0].tolist() == [0, 1, 2, 3] and top[1].tolist() == [7, 8, 9, 10]
  assert abs(float(top_lse[1]) - math.log(4)) < 8 * U32


@pytest.mark.parametrize("vocab", [301, 40001])
def test_distillation_far_from_zero(gpu, vocab):
  """Logits around 3000: a saved lse holds q to 3000 u only, the softmax itself to the
  roundings of the differences (below 16) and of the sum (vocab / 64 + 24 terms)."""
  rng = np.random.default_rng(9)
  batch = ops.ClientBatch([2, 1])
  logits = rand(rng, (3, vocab), torch.float32) + 3000.0
  index, values = teacher_rows(rng, 3, vocab, 4, pad=0)
  weights = torch.tensor([0.5, 0.5, 1.0], dtype=torch.float64)
  q, p = torch.softmax(logits.double().cpu(), 1), torch.softmax(values.double().cpu(), 1)
  want = weights[:, None] * q.scatter_add(1, index.long().cpu(), -p)
  tol = (2 * 16 + vocab / 64 + 24 + 16) * 2 * U32 * (q + want.abs() + p.sum(1, keepdim=True) * (want < 0))
  _, lse = ops.distillation(logits, index, values, batch)
  check(ops.distillation_with_gradient(logits, index, values, batch)[1], want, tol, "gradient")
  check(ops.distillation_backward(logits, lse, index, values, batch), want, tol, "gradient alone")


def far_rows(rows, width, stride, dtype, rng, scale=1.0):
  """[rows, width] at a row stride such that the last row lies past 2^31 elements."""
  assert (rows - 1) * stride > 2**31
  t = torch.empty((rows - 1) * stride + width, dtype=dtype, device="cuda").as_strided((rows, width), (stride, 1))
  t.copy_(rand(rng, (rows, width), dtype, scale))
  return t


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_offsets_past_32_bits(gpu, dtype, odd):
  rng = np.random.default_rng(odd)
  stride, u = 2**30 + 2 + odd, unit(dtype)
  x = far_rows(4, 300, stride, dtype, rng)
  check_top(x, 5)
  index, values = teacher_rows(rng, 4, 300, 5)
  batch = ops.ClientBatch([1, 3])
  loss, grad, el, eg = distill_reference(x, index, values, [1, 3], 1.0)
  far = torch.empty_strided((4, 300), (stride, 1), dtype=dtype, device=gpu)
  got, lse = ops.distillation(x, index, values, batch)
  check(got, loss, el, "loss")
  eg = eg + u * (grad.abs() + eg) + tiny(dtype)
  check(ops.distillation_with_gradient(x, index, values, batch, out=far)[1], grad, eg, "gradient")
  check(ops.distillation_backward(x, lse, index, values, batch, out=far), grad, eg, "gradient alone")
  del far
  y, mean, rstd = ops.layer_norm(x, None, None, batch)
  ref = norm_reference(x, None, None, [1, 3], 1e-5)
  check(y, ref["y"], norm_tolerances(ref, x, None, 300, dtype)["y"], "norm")
  dx, _, _ = ops.layer_norm_backward(x, x, mean, rstd, None, batch)
  near = ops.layer_norm_backward(x.contiguous(), x.contiguous(), mean, rstd, None, batch)[0]
  assert torch.equal(dx, near)
  # clients' weights that far apart, activations too, and gradients written there
  many = ops.ClientBatch([1, 0, 2, 1])
  flat = far_rows(4, 70 * 300, stride, dtype, rng, 1 / math.sqrt(300))
  w = flat.unflatten(1, (70, 300))
  wide = torch.empty(3 * stride + 70, dtype=dtype, device=gpu).as_strided((4, 70), (stride, 1))
  ops.linear(x, w, None, many, out=wide)
  want, e = linear_reference(x, w, [1, 0, 2, 1])
  check(wide, want, e + u * (want.abs() + e) + tiny(dtype), "linear")
  back = ops.linear_backward_input(wide, w, many)
  want, e = linear_reference(wide, w.double().cpu().transpose(1, 2), [1, 0, 2, 1])
  check(back, want, e + u * (want.abs() + e) + tiny(dtype), "input gradient")
  del flat, w
  rows = torch.empty(3 * stride + 70 * 301, device=gpu).as_strided((4, 70 * 301), (stride, 1))
  dw, db = ops.linear_backward_weight(wide, x, many, dweight=rows[:, :70 * 300].unflatten(1, (70, 300)),
                                      dbias=rows[:, 70 * 300:])
  for c, (lo, hi) in enumerate(spans([1, 0, 2, 1])):
    d, xx = wide[lo:hi].double().cpu(), x[lo:hi].double().cpu()
    check(dw[c], d.t() @ xx, 2 * max(1, hi - lo) * U32 * (d.abs().t() @ xx.abs()), "dw")
    check(db[c], d.sum(0), 2 * max(1, hi - lo) * U32 * d.abs().sum(0), "db")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k,m", [(1, 3), (3, 1), (7, 5), (40, 33)])
def test_linear_rows_that_overlap(gpu, dtype, k, m):
  """One row of activations for all (stride 0), and windows one element apart."""
  rng = np.random.default_rng(k)
  counts = [200, 0, 70]
  batch = ops.ClientBatch(counts)
  w = rand(rng, (3, m, k), dtype, 1 / math.sqrt(k))
  for x, dz in [(rand(rng, (1, k), dtype).expand(270, k), rand(rng, (1, m), dtype).expand(270, m)),
                (rand(rng, (269 + k,), dtype).as_strided((270, k), (1, 1)),
                 rand(rng, (269 + m,), dtype).as_strided((270, m), (1, 1)))]:
    want, e = linear_reference(x, w, counts)
    check(ops.linear(x, w, None, batch), want, e + unit(dtype) * (want.abs() + e) + tiny(dtype), "y")
    dw, db = ops.linear_backward_weight(dz, x, batch)
    for c, (lo, hi) in enumerate(spans(counts)):
      d, xx = dz[lo:hi].double().cpu(), x[lo:hi].double().cpu()
      check(dw[c], d.t() @ xx, 2 * max(1, hi - lo) * U32 * (d.abs().t() @ xx.abs()), "dw")
      check(db[c], d.sum(0), 2 * max(1, hi - lo) * U32 * d.abs().sum(0), "db")


@pytest.mark.parametrize("rows,splits", [(32, 5), (128, 3), (256, 2)])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_odd_widths_with_rows_behind(gpu, monkeypatch, dtype, rows, splits):
  plan = (1.0, 128 if rows == 256 and dtype == torch.float32 else rows, splits)
  monkeypatch.setattr(ops, "_estimate", lambda *a: plan if a[4] else (9.0, min(plan[1], 128), splits))
  check_linear(gpu, np.random.default_rng(rows), [70, 0, 129], 257, 131, dtype, "gelu", behind=5)
  check_linear(gpu, np.random.default_rng(splits), [70, 0, 129], 130, 262, dtype, None, shared=True, behind=300)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_clients(gpu, dtype):
  """More clients than a grid's second axis holds; every other one without rows."""
  rng = np.random.default_rng(3)
  n, k, m, u = 70001, 5, 3, unit(dtype)
  counts = np.arange(n) % 2
  rows = int(counts.sum())
  batch = ops.ClientBatch(counts)
  x, dz = rand(rng, (rows, k), dtype), rand(rng, (rows, m), dtype)
  flat = rand(rng, (n, m * k), dtype)
  w = flat.unflatten(1, (m, k))
  mine = w[1::2].double()
  y = ops.linear(x, w, None, batch)
  want = (mine * x.double()[:, None]).sum(2)
  e = 2 * k * U32 * (mine * x.double()[:, None]).abs().sum(2)
  check(y, want, (e + u * (want.abs() + e) + tiny(dtype)).cpu(), "y")
  dx = ops.linear_backward_input(dz, w, batch)
  want = (mine * dz.double()[:, :, None]).sum(1)
  e = 2 * m * U32 * (mine * dz.double()[:, :, None]).abs().sum(1)
  check(dx, want, (e + u * (want.abs() + e) + tiny(dtype)).cpu(), "dx")
  dw, db = ops.linear_backward_weight(dz, x, batch)
  outer = dz.double()[:, :, None] * x.double()[:, None]
  check(dw[1::2], outer, (2 * U32 * outer.abs()).cpu(), "dw")
  assert (dw[::2] == 0).all() and (db[::2] == 0).all() and torch.equal(db[1::2], dz.float())
  _, mean, rstd = ops.layer_norm(x, None, None, batch)
  _, gw, gb = ops.layer_norm_backward(dx, x, mean, rstd, None, batch)
  assert (gw[::2] == 0).all() and torch.equal(gb[1::2], dx.float())
  index = torch.zeros(rows, 1, dtype=torch.int32, device=gpu)
  loss, _ = ops.distillation_with_gradient(x, index, torch.zeros(rows, 1, device=gpu), batch)
  want = torch.logsumexp(x.double(), 1) - x.double()[:, 0]
  check(loss[1::2], want, 64 * U32 * (1 + x.double().abs().amax(1)).cpu(), "loss")
  assert (loss[::2] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_outputs_beside_and_over_their_inputs(gpu, dtype):
  """Columns of one buffer as inputs and outputs, an output over the residual; an output
  over anything else is refused before it is written."""
  rng = np.random.default_rng(5)
  counts = [30, 3]
  batch = ops.ClientBatch(counts)
  buf = rand(rng, (33, 160), dtype)
  x, out, res = buf[:, :64], buf[:, 64:128], buf[:, 128:]
  w = rand(rng, (2, 64, 64), dtype, 0.1)
  want = ops.linear(x.clone(), w, None, batch)
  assert torch.equal(ops.linear(x, w, None, batch, out=out), want)
  down = rand(rng, (2, 32, 64), dtype, 0.1)
  want = ops.linear(x.clone(), down, None, batch, residual=res.clone())
  assert torch.equal(ops.linear(x, down, None, batch, residual=res, out=res), want)
  y, mean, rstd = ops.layer_norm(x, None, None, batch)
  want = ops.layer_norm_backward(y, x, mean, rstd, None, batch, residual=out.clone())[0]
  assert torch.equal(ops.layer_norm_backward(y, x, mean, rstd, None, batch, residual=out, out=out)[0], want)
  before, w0 = buf.clone(), w.clone()
  index, values = torch.zeros(33, 2, dtype=torch.int32, device=gpu), torch.zeros(33, 2, device=gpu)
  grads = torch.zeros(2, 64 * 65, device=gpu)
  calls = [
      lambda: ops.linear(x, w, None, batch, out=x),
      lambda: ops.linear(x, w, None, batch, out=buf[:, 32:96]),
      lambda: ops.linear(x, w, None, batch, residual=buf[:, 65:129], out=out),
      lambda: ops.linear(x, w, None, batch, out=w.view(-1)[:33 * 64].view(33, 64)),
      lambda: ops.linear_backward_input(x, w, batch, out=x),
      lambda: ops.layer_norm(x, None, None, batch, out=x),
      lambda: ops.layer_norm_backward(y, x, mean, rstd, None, batch, out=y),
      lambda: ops.layer_norm_backward(y, x, mean, rstd, None, batch, out=x),
      lambda: ops.layer_norm_backward(y, x, mean, rstd, None, batch, dweight=grads[:, :64], dbias=grads[:, 1:65]),
      lambda: ops.linear_backward_weight(x, x, batch, dweight=grads[:, :4096].unflatten(1, (64, 64)),
                                         dbias=grads[:, 4095:4159]),
      lambda: ops.distillation_with_gradient(x, index, values, batch, out=buf[:, 1:65]),
      lambda: ops.layer_norm(x, None, None, batch, eps=-1e-5),
      lambda: ops.top_logits(x, 2, temperature=1e-16),
      lambda: ops.top_logits(x, 2, temperature=1e16),
  ]
  for i, call in enumerate(calls):
    with pytest.raises(ValueError):
      call()
      pytest.fail("call %d was not refused" % i)
  assert torch.equal(buf, before) and torch.equal(w, w0)


def test_two_streams_at_once_and_a_batch_that_ends(gpu):
  """The same weights on two streams at a time, with a batch each that is dropped while its
  kernels may still run."""
  rng = np.random.default_rng(6)
  counts = [700, 0, 300]
  x, dz = rand(rng, (1000, 520), torch.bfloat16), rand(rng, (1000, 515), torch.bfloat16)
  w = rand(rng, (3, 515, 520), torch.bfloat16, 0.05)

  def run():
    batch = ops.ClientBatch(counts)
    y = ops.linear(x, w, None, batch, activation="gelu")
    return [y, ops.linear_backward_input(dz, w, batch), *ops.linear_backward_weight(dz, x, batch)]

  want = run()
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  batches, outs = [ops.ClientBatch(counts) for _ in streams], []
  for s, batch in zip(streams, batches):
    with torch.cuda.stream(s):
      y = ops.linear(x, w, None, batch, activation="gelu")
      outs.append([y, ops.linear_backward_input(dz, w, batch), *ops.linear_backward_weight(dz, x, batch)])
  del batches, batch
  filler = [torch.full((1 << 16,), 7, dtype=torch.int32, device=gpu) for _ in range(64)]
  for s in streams:
    s.synchronize()
  for out in outs:
    for a, b in zip(out, want):
      assert torch.equal(a, b)
  del filler


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [2, 3, 4, 255, 258, 510, 515, 766, 771, 1022, 1030, 1537, 2046, 2051, 2500, 4095, 4101,
                                 6001, 7999, 8195, 12003, 16381, 16390])
def test_layer_norm_every_launch_shape(gpu, dtype, dim):
  """Widths on both sides of every shape's limit, none of them whole vectors; tiles that end
  inside a block's row groups; parameters at odd elements; NaN behind the batch and its rows."""
  rng = np.random.default_rng(dim)
  counts = [3, 0, 37]
  batch = ops.ClientBatch(counts)
  buf = torch.full((42, dim + 3), math.nan, dtype=dtype, device=gpu)
  buf[:40, 1:1 + dim] = rand(rng, (40, dim), dtype) + 0.5
  x = buf[:, 1:1 + dim]
  dy, res = rand(rng, (40, dim), dtype), rand(rng, (40, dim), dtype)
  w, b = flat_params(rng, 3, [(dim,), (dim,)], dtype, 1.0)
  out = torch.full((42, dim + 3), 9.0, dtype=dtype, device=gpu)
  y, mean, rstd = ops.layer_norm(x, w, b, batch, out=out[:, 1:1 + dim])
  ref = norm_reference(x[:40], w, b, counts, 1e-5, dy, res)
  tol = norm_tolerances(ref, x[:40], b, dim, dtype, counts, dy, res)
  check(y[:40], ref["y"], tol["y"], "y")
  check(mean[:40], ref["mean"], tol["mean"], "mean")
  check(rstd[:40], ref["rstd"], tol["rstd"], "rstd")
  rows = torch.full((3, 2 * dim + 3), 3.0, device=gpu)
  dx = torch.full((42, dim + 3), 9.0, dtype=dtype, device=gpu)
  _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, batch, residual=res, dweight=rows[:, 1:1 + dim],
                                      dbias=rows[:, 2 + dim:2 + 2 * dim], out=dx[:, 1:1 + dim])
  check(dx[:40, 1:1 + dim], ref["dx"], tol["dx"], "dx")
  check(dw, ref["dw"], tol["dw"], "dw")
  check(db, ref["db"], tol["db"], "db")
  for t in (out, dx):
    assert (t[:, 0] == 9.0).all() and (t[:, 1 + dim:] == 9.0).all() and (t[40:] == 9.0).all()
  assert (rows[:, 0] == 3.0).all() and (rows[:, 1 + dim] == 3.0).all() and (rows[:, -1] == 3.0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k,m", [(1, 1), (3, 70), (17, 300), (64, 256), (65, 257), (131, 77), (256, 64), (515, 130)])
@pytest.mark.parametrize("counts", [[1], [8, 0, 3], [16, 1, 0, 9], [7, 40, 0, 33]], ids=str)
def test_weight_gradient_of_few_rows(gpu, monkeypatch, dtype, k, m, counts):
  """The kernel for few rows at every shape, also where it takes a client's rows in turns;
  rows behind the batch NaN, accumulation, no bias, overlapping client rows left alone."""
  monkeypatch.setattr(ops, "_few_rows", lambda *a: True)
  rng = np.random.default_rng(k + m)
  n = sum(counts)
  batch = ops.ClientBatch(counts)
  wide = rand(rng, (n + 2, k + m + 1), dtype)
  wide[n:] = math.nan
  x, dz = wide[:, :k], wide[:, k + 1:]
  rows = torch.full((len(counts), m * k + m + 2), 3.0, device=gpu)
  dw, db = ops.linear_backward_weight(dz, x, batch, dweight=rows[:, 1:1 + m * k].unflatten(1, (m, k)),
                                      dbias=rows[:, 1 + m * k:1 + m * k + m])
  for c, (lo, hi) in enumerate(spans(counts)):
    d, xx = dz[lo:hi].double().cpu(), x[lo:hi].double().cpu()
    check(dw[c], d.t() @ xx, 2 * max(1, hi - lo) * U32 * (d.abs().t() @ xx.abs()), "dw of client %d" % c)
    check(db[c], d.sum(0), 2 * max(1, hi - lo) * U32 * d.abs().sum(0), "db of client %d" % c)
  assert (rows[:, 0] == 3.0).all() and (rows[:, -1] == 3.0).all()
  alone, none = ops.linear_backward_weight(dz, x, batch, bias=False)
  assert none is None and torch.equal(alone, dw)
  two = rows.clone()
  ops.linear_backward_weight(dz, x, batch, dweight=two[:, 1:1 + m * k].unflatten(1, (m, k)),
                             dbias=two[:, 1 + m * k:1 + m * k + m], accumulate=True)
  for c, (lo, hi) in enumerate(spans(counts)):
    tol = 2 * (hi - lo + 2) * U32 * (dz[lo:hi].double().abs().t() @ x[lo:hi].double().abs()).cpu() * 2
    check(two[c, 1:1 + m * k].view(m, k), 2 * dw[c].double(), tol + U32 * dw[c].double().abs().cpu() * 2, "twice")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k,m", [(64, 640), (640, 64), (96, 1000), (1000, 96), (128, 300), (300, 128), (31, 515), (515, 31),
                                 (20, 257), (257, 20), (41, 129), (130, 2), (2, 130)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_walking_along_the_columns(gpu, monkeypatch, dtype, k, m, act):
  """Short contractions by blocks that walk: one step and two, whole, in whole vectors and
  not, columns that end inside a tile and a vector, operands copied and as they lie."""
  size = torch.finfo(dtype).bits // 8
  seen = []

  def walks(batch, columns, a, weight):
    ok = size == 2 and a.shape[1] <= 128 and not (ops._odd(a) or ops._odd(weight))
    seen.append(ok)
    return ok

  monkeypatch.setattr(ops, "_walks", walks)
  monkeypatch.setattr(ops, "_estimate", lambda *a: (1.0 if a[4] else 1e9, 32, 1))
  rng = np.random.default_rng(k + m)
  check_linear(gpu, rng, [129, 0, 40], k, m, dtype, act)
  check_linear(gpu, rng, [300, 1], k, m, dtype, act, shared=True, behind=3)
  assert any(seen) == (size == 2)


def test_linear_walks_by_its_own_rule(gpu):
  check_linear(gpu, np.random.default_rng(1), [700] * 8, 96, 5004, torch.bfloat16, None)
  check_linear(gpu, np.random.default_rng(2), [128] * 40, 5002, 64, torch.bfloat16, "relu", shared=True)
  batch = ops.ClientBatch([700] * 8)
  x, w = torch.zeros(5600, 96, device=gpu, dtype=torch.bfloat16), torch.zeros(8, 5004, 96, device=gpu, dtype=torch.bfloat16)
  assert ops._walks(batch, 5004, x, w) and not ops._walks(batch, 5004, x, w[:, :, 1:])


def test_graph_of_every_path(gpu):
  """Walking blocks, few rows, split contractions, copied odd rows, wide norms and streamed
  rows in one captured graph: every replay, on new inputs and with eager work between, gives
  the eager calls' bits."""
  rng = np.random.default_rng(12)
  many, few, one, odd = [ops.ClientBatch(c) for c in ([700] * 8, [8, 0, 3, 5], [1], [900, 0, 773])]
  bf, h = torch.bfloat16, torch.float16
  inputs = dict(
      x1=rand(rng, (5600, 96), bf), w1=rand(rng, (8, 5004, 96), bf, 0.1),
      x2=rand(rng, (16, 130), torch.float32), d2=rand(rng, (16, 70), torch.float32),
      x3=rand(rng, (1, 4096), bf), w3=rand(rng, (1, 512, 4096), bf, 0.02),
      x4=rand(rng, (1673, 1021), h), w4=rand(rng, (3, 515, 1021), h, 0.03), d4=rand(rng, (1673, 515), h),
      x5=rand(rng, (16, 9001), bf), d5=rand(rng, (16, 9001), bf),
      s6=rand(rng, (16, 70001), bf), t6=rand(rng, (16, 70001), bf))

  def run(i):
    out = [ops.linear(i["x1"], i["w1"], None, many)]
    out += ops.linear_backward_weight(i["d2"], i["x2"], few)
    out += ops.linear(i["x3"], i["w3"], None, one, activation="silu", preactivation=True)
    out += [ops.linear(i["x4"], i["w4"], None, odd), ops.linear_backward_input(i["d4"], i["w4"], odd)]
    out += ops.linear_backward_weight(i["d4"], i["x4"], odd)
    y, mean, rstd = ops.layer_norm(i["x5"], None, None, few)
    out += [y, mean, rstd, *ops.layer_norm_backward(i["d5"], i["x5"], mean, rstd, None, few)]
    index, values, lse = ops.top_logits(i["t6"], 300, 2.0)
    out += [index, values, lse]
    out += ops.distillation_with_gradient(i["s6"], index, values, few, temperature=2.0, teacher_lse=lse)
    return out

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    run(inputs)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = run(inputs)
  for _ in range(4):
    for t in inputs.values():
      t.copy_(rand(rng, tuple(t.shape), t.dtype, float(t.float().std())))
    want = [t.clone() for t in run(inputs)]
    graph.replay()
    torch.cuda.synchronize()
    for n, (a, b) in enumerate(zip(captured, want)):
      assert torch.equal(a, b), n


@pytest.mark.parametrize("vocab,k", [(8192, 201), (8193, 200), (8193, 201), (8193, 700), (8193, 701), (2049, 1024), (32769, 701),
                                     (5000, 600)])
def test_top_logits_many_of_a_row(gpu, vocab, k):
  """On both sides of the limits by k, on rows with few distinct values too: many ties."""
  rng = np.random.default_rng(vocab + k)
  x = rand(rng, (4, vocab), torch.bfloat16, 2.0)
  x[2] = torch.round(x[2].float()).to(x.dtype)
  x[3] = (torch.arange(vocab, device=gpu) % 700).to(x.dtype)
  check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("behind", [0, 3])
def test_distillation_without_rows(gpu, dtype, behind):
  """Every form on a batch without rows, over logits of none and over rows behind the batch."""
  batch = ops.ClientBatch([0, 0])
  logits = torch.full((behind, 8), 2.0, dtype=dtype, device=gpu)
  idx = torch.zeros(behind, 3, dtype=torch.int32, device=gpu)
  val = torch.zeros(behind, 3, device=gpu)
  loss, lse = ops.distillation(logits, idx, val, batch)
  assert (loss == 0).all() and loss.shape == (2,) and lse.shape == (behind,)
  grad = ops.distillation_backward(logits, lse, idx, val, batch)
  assert grad.shape == (behind, 8) and grad.dtype == dtype and (grad == 0).all()
  grad = ops.distillation_backward(logits, lse, idx, val, batch, dloss=torch.ones(2, device=gpu), out=logits)
  assert (grad == 2.0).all()
  loss, grad = ops.distillation_with_gradient(logits, idx, val, batch)
  assert (loss == 0).all() and grad.shape == (behind, 8)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [40, 3001, 70001])
def test_distillation_gradient_of_rows_the_loss_left_out(gpu, dtype, vocab):
  """A saved log-sum-exp serves a gradient by other weights and another teacher: rows that
  the loss did not look at (no weight, nothing but padding) are summed by the gradient."""
  rng = np.random.default_rng(vocab)
  counts = [3, 2]
  batch = ops.ClientBatch(counts)
  logits = rand(rng, (5, vocab), dtype, 2.0) + 3.0
  index, values = teacher_rows(rng, 5, vocab, 6, pad=0)
  bare = index.clone()
  bare[1] = -1
  weights = torch.tensor([1.0, 0.5, 0.0, 0.0, 2.0], device=gpu)
  _, lse = ops.distillation(logits, bare, values, batch, row_weights=weights)
  _, grad, _, eg = distill_reference(logits, index, values, counts, 1.0)
  got = ops.distillation_backward(logits, lse, index, values, batch)
  check(got, grad, eg + unit(dtype) * (grad.abs() + eg) + tiny(dtype), "gradient")
  assert lse.isnan().tolist() == [False, True, True, True, False]


# A launch has fewer than 2^32 threads, so a row or client each past these counts takes another.
MOST = {64: (2**32 - 1) // 64, 256: (2**32 - 1) // 256}


def around(n, at):
  """Rows to look at: both ends and both sides of a launch's last."""
  return torch.tensor(sorted({0, 1, 777, at - 2, at - 1, at, at + 1, n - 2, n - 1}), device="cuda")


def test_top_logits_of_more_rows_than_a_launch(gpu):
  """16.8 million rows of 40, k 33: blocks of 256 threads."""
  n, v, k = MOST[256] + 300, 40, 33
  gen = torch.Generator(device=gpu).manual_seed(3)
  x = torch.empty(n, v, dtype=torch.bfloat16, device=gpu).normal_(0.0, 2.0, generator=gen)
  index, values, lse = ops.top_logits(x, k)
  rows = around(n, MOST[256])
  want, want_lse = top_reference(x[rows], k)
  assert torch.equal(index[rows].long().cpu(), want)
  assert torch.equal(values[rows], torch.gather(x[rows], 1, index[rows].long()))
  check(lse[rows], want_lse, (v / 1024 + 48 + 4 * 16) * 2 * U32, "lse")
  # every row: falling values at the places they are said to be at
  for lo in range(0, n, 1 << 22):
    i, val = index[lo:lo + (1 << 22)], values[lo:lo + (1 << 22)]
    assert bool((val[:, 1:] <= val[:, :-1]).all()) and bool((i >= 0).all()) and bool((i < v).all())
    assert torch.equal(torch.gather(x[lo:lo + (1 << 22)], 1, i.long()), val)
    assert bool(lse[lo:lo + (1 << 22)].isfinite().all())


def test_distillation_of_more_rows_than_a_launch(gpu):
  """67 million rows of 8: blocks of one wave; loss alone, gradient alone, both."""
  n, v = MOST[64] + 500, 8
  gen = torch.Generator(device=gpu).manual_seed(4)
  x = torch.empty(n, v, dtype=torch.float16, device=gpu).normal_(0.0, 2.0, generator=gen)
  index = torch.randint(0, v, (n, 1), generator=gen, device=gpu, dtype=torch.int32)
  values = torch.zeros(n, 1, device=gpu)
  lse_t = torch.empty(n, device=gpu).uniform_(0.1, 1.0, generator=gen)
  weights = torch.ones(n, device=gpu)
  counts = [MOST[64] - 1, 400, 101]
  batch = ops.ClientBatch(counts)
  loss, grad = ops.distillation_with_gradient(x, index, values, batch, teacher_lse=lse_t, row_weights=weights)
  loss2, lse = ops.distillation(x, index, values, batch, teacher_lse=lse_t, row_weights=weights)
  assert torch.equal(loss, loss2)
  back = ops.distillation_backward(x, lse, index, values, batch, teacher_lse=lse_t, row_weights=weights)
  rows = around(n, MOST[64])
  want, g, el, eg = distill_reference(x[rows], index[rows], values[rows], [len(rows)], 1.0, lse_t[rows], weights[rows])
  eg = eg + unit(torch.float16) * (g.abs() + eg) + tiny(torch.float16)
  check(grad[rows], g, eg, "gradient")
  check(back[rows], g, eg, "gradient alone")
  # every row: p (log p - log q) summed over the last two clients, in float64
  for c, (lo, hi) in list(enumerate(spans(counts)))[1:]:
    logp = -lse_t[lo:hi].double()
    logq = torch.log_softmax(x[lo:hi].double(), 1).gather(1, index[lo:hi].long())[:, 0]
    term = logp.exp() * (logp - logq)
    tol = float((logp.exp() * (logp.abs() + logq.abs() + 2)).sum()) * (2 * (6 * 32 + 52) * 2 + hi - lo + 8) * U32
    check(loss[c], term.sum(), tol, "loss")
  assert bool(lse.isfinite().all()) and bool(grad.isfinite().all())


def test_more_clients_than_a_launch(gpu):
  """16.8 million clients of one row: the losses' join and the norm's tiles."""
  n, d = MOST[256] + 300, 4
  gen = torch.Generator(device=gpu).manual_seed(5)
  batch = ops.ClientBatch(np.ones(n, np.int64))
  x = torch.empty(n, d, device=gpu).normal_(0.0, 1.0, generator=gen)
  index = torch.randint(0, d, (n, 1), generator=gen, device=gpu, dtype=torch.int32)
  loss, lse = ops.distillation(x, index, torch.zeros(n, 1, device=gpu), batch)
  want = torch.logsumexp(x.double(), 1)
  size = 1 + x.double().abs().amax(1)
  assert bool(((lse.double() - want).abs() <= 64 * U32 * size).all())
  want = want - x.double().gather(1, index.long())[:, 0]
  assert bool(((loss.double() - want).abs() <= 64 * U32 * size).all())
  y, mean, rstd = ops.layer_norm(x, None, None, batch)
  rows = around(n, MOST[256])
  ref = norm_reference(x[rows], None, None, [len(rows)], 1e-5)
  tol = norm_tolerances(ref, x[rows], None, d, torch.float32)
  for name, got in dict(y=y, mean=mean, rstd=rstd).items():
    check(got[rows], ref[name], tol[name], name)
  mu = x.double().mean(1)
  assert bool(((mean.double() - mu).abs() <= 32 * U32 * x.double().abs().amax(1)).all())


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
def test_gelu_of_every_value(gpu, dtype):
  """All values from -13.5 to 13.5 of a 16-bit type, through products by one: relative to each
  value, in the negative tail too.  The distribution function's relative error stays
  below (1 + z^2) 2^-19, and what is below 16 least normal float32 may vanish."""
  z = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(dtype)
  z = z[z.isfinite() & (z.abs() <= 13.5)]
  n = z.numel()
  batch, one = ops.ClientBatch([n]), torch.ones(1, 1, 1, dtype=dtype, device=gpu)
  x = z.to(gpu)[:, None]
  f, slope = ACTS["gelu"]
  z64 = z.double()
  e = (1 + z64 * z64) * 2.0**-19
  least = 16 * 2.0**-126 + tiny(dtype)
  want = f(z64)
  check(ops.linear(x, one, None, batch, activation="gelu")[:, 0], want, (unit(dtype) + e) * want.abs() + least, "gelu")
  want = slope(z64)
  parts = 0.5 * torch.special.erfc(-z64 / math.sqrt(2)) + z64.abs() * torch.exp(-z64 * z64 / 2) / math.sqrt(2 * math.pi)
  got = ops.linear_backward_input(torch.ones_like(x), one, batch, preactivation=x, activation="gelu")[:, 0]
  check(got, want, unit(dtype) * want.abs() + (1 + unit(dtype)) * e * parts + least, "slope")


def test_gelu_of_float32_in_its_tail(gpu):
  """Relative to each value from -13.5 to 13.5.  The argument z / sqrt 2 carries 1.3 roundings
  (its product and its constant), which erfc takes z^2 + 1 times; erfc and exp are good to 4
  units, and two products follow: (12 + 2 z^2) u."""
  z = torch.linspace(-13.5, 13.5, 400001, dtype=torch.float64).float()
  batch, one = ops.ClientBatch([z.numel()]), torch.ones(1, 1, 1, device=gpu)
  x = z.to(gpu)[:, None]
  f, slope = ACTS["gelu"]
  z64 = z.double()
  e = (12 + 2 * z64 * z64) * U32
  least = 16 * 2.0**-126
  want = f(z64)
  check(ops.linear(x, one, None, batch, activation="gelu")[:, 0], want, e * want.abs() + least, "gelu")
  parts = 0.5 * torch.special.erfc(-z64 / math.sqrt(2)) + z64.abs() * torch.exp(-z64 * z64 / 2) / math.sqrt(2 * math.pi)
  got = ops.linear_backward_input(torch.ones_like(x), one, batch, preactivation=x, activation="gelu")[:, 0]
  check(got, slope(z64), e * parts + least, "slope")


def check_added(rng, counts, k, m, dtype):
  """Gradients added to what is there, and outputs over their residuals: as without, plus one
  addition (a split's parts are added to the old value one by one)."""
  n, c = sum(counts), len(counts)
  batch = ops.ClientBatch(counts)
  x, dz = rand(rng, (n, k), dtype), rand(rng, (n, m), dtype, 0.5)
  w, b = flat_params(rng, c, [(m, k), (m,)], dtype, 1 / math.sqrt(k))
  old = rand(rng, (c, m * k + m + 2), torch.float32)
  rows = old.clone()
  ops.linear_backward_weight(dz, x, batch, dweight=rows[:, 1:1 + m * k].unflatten(1, (m, k)),
                             dbias=rows[:, 1 + m * k:1 + m * k + m], accumulate=True)
  assert torch.equal(rows[:, 0], old[:, 0]) and torch.equal(rows[:, -1], old[:, -1])
  for i, (lo, hi) in enumerate(spans(counts)):
    d, xx = dz[lo:hi].double().cpu(), x[lo:hi].double().cpu()
    o, r = old[i, 1:1 + m * k].view(m, k).double().cpu(), rows[i, 1:1 + m * k].view(m, k)
    mag = d.abs().t() @ xx.abs()
    check(r, o + d.t() @ xx, (2 * max(1, hi - lo) + 70) * U32 * mag + 70 * U32 * o.abs(), "dw of client %d" % i)
    o, r = old[i, 1 + m * k:1 + m * k + m].double().cpu(), rows[i, 1 + m * k:1 + m * k + m]
    mag = d.abs().sum(0)
    check(r, o + d.sum(0), (2 * max(1, hi - lo) + 70) * U32 * mag + 70 * U32 * o.abs(), "db of client %d" % i)
  res, below = rand(rng, (n, m), dtype), rand(rng, (n, k), dtype)
  before = rand(rng, (n, k), dtype)
  want = ops.linear(x, w, b, batch, activation="silu", residual=res.clone())
  assert torch.equal(ops.linear(x, w, b, batch, activation="silu", residual=res, out=res), want)
  want = ops.linear_backward_input(dz, w, batch, preactivation=before, activation="relu", residual=below.clone())
  assert torch.equal(ops.linear_backward_input(dz, w, batch, preactivation=before, activation="relu", residual=below,
                                               out=below), want)


@pytest.mark.parametrize("rows,splits", [(32, 1), (32, 5), (128, 1), (128, 3), (256, 1), (256, 2), (128, 64)])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_every_plan_adds(gpu, monkeypatch, dtype, rows, splits):
  monkeypatch.setattr(ops, "_few_rows", lambda *a: False)
  monkeypatch.setattr(ops, "_plan", lambda tiles, steps, longest, size, aligned: (
      128 if rows == 256 and (size == 4 or not aligned) else rows, splits))
  monkeypatch.setattr(ops, "_estimate", lambda tiles, steps, longest, size, aligned: (
      1e9 if aligned == (splits == 1) else 1.0, rows, splits))
  rng = np.random.default_rng(rows + splits)
  check_added(rng, [40, 0, 1, 300], 131, 77, dtype)
  check_added(rng, [257, 3], 134, 260, dtype)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("k,m", [(96, 1000), (41, 129), (128, 64)])
def test_linear_walking_adds(gpu, monkeypatch, dtype, k, m):
  monkeypatch.setattr(ops, "_walks", lambda batch, columns, a, weight: a.shape[1] <= 128 and not (
      ops._odd(a) or ops._odd(weight)))
  monkeypatch.setattr(ops, "_estimate", lambda *a: (1.0 if a[4] else 1e9, 32, 1))
  check_added(np.random.default_rng(k + m), [129, 0, 40], k, m, dtype)


@pytest.mark.parametrize("vocab,k", [(3000, 5), (10004, 64), (10004, 300), (40000, 128)])
def test_top_logits_of_float16_rows_far_from_zero(gpu, vocab, k):
  """Rows around 1000: a value's last three bits lie below the bits the bound is found by."""
  x = rand(np.random.default_rng(vocab + k), (5, vocab), torch.float16) + 1000.0
  check_top(x, k, 2.0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset", [30.0, 60.0, 200.0, -250.0, 500.0, 1000.0])
@pytest.mark.parametrize("tau", [1.0, 0.5])
def test_distillation_gradient_alone_at_an_offset(gpu, dtype, offset, tau):
  """A saved log-sum-exp carries four roundings of its size into q, 2^-22 |lse| relative: as
  far as 64 for a float32 gradient (1.5e-5), 256 for 16-bit ones (6e-5, an eighth of
  float16's half step); beyond, the softmax's own roundings alone."""
  rng = np.random.default_rng(int(abs(offset) + 10 * tau))
  vocab, n = 501, 40
  batch = ops.ClientBatch([n])
  logits = rand(rng, (n, vocab), dtype) + offset
  index, values = teacher_rows(rng, n, vocab, 4, pad=0)
  s = logits.double().cpu() / tau
  q, p = torch.softmax(s, 1), torch.softmax(values.double().cpu() / tau, 1)
  want = (q.scatter_add(1, index.long().cpu(), -p)) * tau / n
  _, lse = ops.distillation(logits, index, values, batch, temperature=tau)
  far = float(torch.logsumexp(s, 1).abs().max()) > (64.0 if dtype == torch.float32 else 256.0)
  saved = 0.0 if far else 2.0**-22 * torch.logsumexp(s, 1).abs()[:, None]
  both = (q + p.sum(1, keepdim=True) * (want < 0)) * tau / n
  tol = (2 * 16 / tau + vocab / 64 + 24 + 16) * 2 * U32 * both + 2 * saved * q * tau / n
  tol = tol + unit(dtype) * (want.abs() + tol) + tiny(dtype)
  got = ops.distillation_backward(logits, lse, index, values, batch, temperature=tau)
  check(got, want, tol, "gradient")
