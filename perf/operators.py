"""The client's local step: what its operators are measured on.

The four operators of ``federated_amd.client_ops`` (layer norm, linear, top logits,
distillation), each over a round's clients: a ragged batch of rows, client c's
weights and gradients inside its own flat parameter row.  ``run`` computes one pass
either in plain torch operations (``own`` false) or with the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
  return [
      # A handful of clients' single examples through a small embedding's norm: a
      # call that is all latency (evaluation while a round is being sampled).
      dict(name="norm-smallest", op="layer_norm", clients=4, rows=7, dim=96, dtype="float32", shared=False,
           backward=False, spread=1),
      # A simulated round's local step: 256 clients with some hundred rows each, of
      # the word-prediction model's recurrent width, every client its own weights.
      dict(name="norm-round", op="layer_norm", clients=256, rows=81920, dim=670, dtype="bfloat16", shared=False,
           backward=True, spread=2),
      # Few large clients (silos) with a wide model's activations.
      dict(name="norm-silos", op="layer_norm", clients=6, rows=65541, dim=4096, dtype="bfloat16", shared=False,
           backward=True, spread=3),
      # One row through one wide projection: a client answering token by token; the
      # weight's bytes are everything.
      dict(name="linear-token", op="linear", clients=1, rows=1, inner=4096, outer=14336, dtype="bfloat16",
           activation="silu", residual=False, shared=False, phase="forward", spread=4),
      # The first local step's evaluation of a round: a few rows for each of 256
      # clients through the word-prediction model's dense layer, in float32.
      dict(name="linear-few-rows", op="linear", clients=256, rows=1500, inner=670, outer=96, dtype="float32",
           activation="relu", residual=False, shared=False, phase="forward", spread=5),
      # The same model's output head in a local step of 64 clients: forward and both
      # gradients, no activation, an odd vocabulary, every client its own head.
      dict(name="linear-head-step", op="linear", clients=64, rows=20480, inner=96, outer=10004, dtype="bfloat16",
           activation="none", residual=False, shared=False, phase="train", spread=6),
      # A step of a wide feed-forward projection, silos of thousands of rows.
      dict(name="linear-silos-step", op="linear", clients=8, rows=16384, inner=4096, outer=8192, dtype="bfloat16",
           activation="gelu", residual=True, shared=False, phase="train", spread=7),
      # Sizes that are a multiple of nothing, with one weight broadcast to all clients
      # (a round's first step), float16.
      dict(name="linear-odd-step", op="linear", clients=33, rows=9001, inner=1021, outer=2050, dtype="float16",
           activation="silu", residual=True, shared=True, phase="train", spread=8),
      # The server ranks a few evaluation rows' logits.
      dict(name="top-few", op="top_logits", rows=3, vocab=10004, top=10, dtype="float32", spread=9),
      # A teacher's message for a silo's batch: 64 of a large vocabulary's logits.
      dict(name="top-message", op="top_logits", rows=4096, vocab=131072, top=64, dtype="bfloat16", spread=10),
      # A round's distillation step over the word-prediction vocabulary, a fifth of
      # the teacher's entries padding.
      dict(name="distill-round", op="distillation", clients=256, rows=20480, vocab=10004, top=32, dtype="float32",
           temperature=2.0, tail=False, padding=0.2, phase="train", spread=11),
      # The same over a large vocabulary, with the tail's mass known.
      dict(name="distill-silos", op="distillation", clients=4, rows=8197, vocab=131072, top=64, dtype="bfloat16",
           temperature=1.5, tail=True, padding=0.0, phase="train", spread=12),
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["layer_norm", "linear", "linear", "top_logits", "distillation"])
  dtype = rng.choice(["float32", "bfloat16", "float16"])
  spread = rng.randrange(1, 1 << 20)
  clients = _log_int(rng, 1, 512)
  if op == "layer_norm":
    dim = _log_int(rng, 17, 8192)
    rows = _log_int(rng, 1, min(131072, (1 << 28) // dim))
    return dict(op=op, clients=clients, rows=rows, dim=dim, dtype=dtype, shared=rng.random() < 0.3,
                backward=rng.random() < 0.7, spread=spread)
  if op == "linear":
    inner, outer = _log_int(rng, 16, 8192), _log_int(rng, 16, 16384)
    clients = min(clients, max(1, (1 << 27) // (inner * outer)))
    rows = _log_int(rng, 1, min(32768, max(1, (1 << 38) // (inner * outer))))
    return dict(op=op, clients=clients, rows=rows, inner=inner, outer=outer, dtype=dtype,
                activation=rng.choice(["none", "relu", "gelu", "silu"]), residual=rng.random() < 0.5,
                shared=rng.random() < 0.3, phase=rng.choice(["forward", "train"]), spread=spread)
  vocab = _log_int(rng, 300, 160000)
  rows = _log_int(rng, 1, min(32768, (1 << 28) // vocab))
  top = _log_int(rng, 1, 128)
  if op == "top_logits":
    return dict(op=op, rows=rows, vocab=vocab, top=top, dtype=dtype, spread=spread)
  return dict(op=op, clients=clients, rows=rows, vocab=vocab, top=top, dtype=dtype,
              temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), tail=rng.random() < 0.5,
              padding=rng.choice([0.0, 0.2]), phase=rng.choice(["loss", "train"]), spread=spread)


def client_counts(case):
  """Rows of each client: an uneven split of the case's rows (part of the case, so
  that its work is known); some clients have none when rows are few."""
  rng = np.random.default_rng(case["spread"])
  share = rng.exponential(size=case["clients"]) + 0.3
  cuts = np.floor(np.cumsum(share) / share.sum() * case["rows"]).astype(np.int64)
  cuts[-1] = case["rows"]
  return np.diff(cuts, prepend=0)


def _normal(gen, shape, scale, dtype):
  return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen).to(dtype)


def prepare(case, seed):
  gen = torch.Generator(device="cuda").manual_seed(int(seed))
  dtype = DTYPES[case["dtype"]]
  st = dict(case)
  n = case["rows"]
  if case["op"] != "top_logits":
    counts = client_counts(case)
    st["counts"] = counts
    if own:
      from federated_amd import client_ops  # pylint: disable=g-import-not-at-top
      st["batch"] = client_ops.ClientBatch(counts, device="cuda")
    else:
      # row -> client and row -> place in a [clients, longest] padding
      client = np.repeat(np.arange(counts.size), counts)
      start = np.cumsum(counts) - counts
      st["client"] = torch.from_numpy(client).cuda()
      st["longest"] = int(max(1, counts.max()))
      st["place"] = torch.from_numpy(client * st["longest"] + np.arange(n) - start[client]).cuda()
      st["count"] = torch.from_numpy(counts).cuda()
  copies = 1 if case.get("shared") else case.get("clients", 1)
  if case["op"] == "layer_norm":
    d = case["dim"]
    st["x"] = _normal(gen, (n, d), 1.0, dtype) + _normal(gen, (n, 1), 0.5, dtype)
    # the client's flat parameter row: weight, then bias
    params = _normal(gen, (copies, 2 * d), 0.2, dtype)
    params[:, :d] += 1.0
    params = params.expand(case["clients"], 2 * d)
    st["weight"], st["bias"] = params[:, :d], params[:, d:]
    if case["backward"]:
      st["dy"] = _normal(gen, (n, d), 0.1, dtype)
      grads = torch.empty(case["clients"], 2 * d, device="cuda")
      st["dweight"], st["dbias"] = grads[:, :d], grads[:, d:]
  elif case["op"] == "linear":
    k, m = case["inner"], case["outer"]
    st["x"] = _normal(gen, (n, k), 1.0, dtype)
    params = _normal(gen, (copies, m * k + m), 1.0 / math.sqrt(k), dtype)
    params = params.expand(case["clients"], m * k + m)
    st["weight"], st["bias"] = params[:, :m * k].unflatten(1, (m, k)), params[:, m * k:]
    st["residual"] = _normal(gen, (n, m), 1.0, dtype) if case["residual"] else None
    if case["phase"] == "train":
      # the gradient at this product's pre-activation, and the pre-activation the
      # input came from
      st["dz"] = _normal(gen, (n, m), 0.1, dtype)
      st["before"] = _normal(gen, (n, k), 1.0, dtype) if case["activation"] != "none" else None
      grads = torch.empty(case["clients"], m * k + m, device="cuda")
      st["dweight"], st["dbias"] = grads[:, :m * k].unflatten(1, (m, k)), grads[:, m * k:]
  elif case["op"] == "top_logits":
    st["logits"] = _normal(gen, (n, case["vocab"]), 3.0, dtype)
  else:
    v, t = case["vocab"], min(case["top"], case["vocab"])
    st["top"] = t
    first = torch.randint(0, v, (n, 1), generator=gen, device="cuda")
    step = torch.randint(1, max(2, v // t), (n, 1), generator=gen, device="cuda")
    index = (first + step * torch.arange(t, device="cuda")) % v
    gap = torch.empty(n, t, device="cuda").exponential_(4.0, generator=gen)
    values = 8.0 - torch.cumsum(gap, 1)
    st["logits"] = _normal(gen, (n, v), 2.0, dtype)
    st["logits"].scatter_add_(1, index, (0.6 * values).to(dtype))
    st["values"] = values
    if case["padding"]:
      # rows of fewer than t entries, some of none
      keep = torch.empty(n, 1, device="cuda").uniform_(0.0, 1.0 / (1.0 - case["padding"]), generator=gen)
      keep = torch.clamp(torch.floor(keep * (t + 1)), max=t)
      index = torch.where(torch.arange(t, device="cuda") < keep, index, -1)
    st["index"] = index.to(torch.int32)
    st["teacher_lse"] = None
    if case["tail"]:
      rest = torch.empty(n, device="cuda").uniform_(0.05, 0.7, generator=gen)
      st["teacher_lse"] = torch.logsumexp(values / case["temperature"], 1) + rest
  return st


def work(case):
  size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
  n = case["rows"]
  if case["op"] == "top_logits":
    t = min(case["top"], case["vocab"])
    return dict(bytes=n * (case["vocab"] * size + t * (4 + size) + 4), flops=3 * n * case["vocab"])
  c = case["clients"]
  if case["op"] == "layer_norm":
    d = case["dim"]
    sets = 1 if case["shared"] else c
    if case["backward"]:
      return dict(bytes=n * d * 4 * size + n * 8 + sets * 2 * d * size + c * 2 * d * 4, flops=20 * n * d)
    return dict(bytes=n * d * 2 * size + n * 8 + sets * 2 * d * size, flops=8 * n * d)
  if case["op"] == "linear":
    k, m = case["inner"], case["outer"]
    # only clients that have rows need their weights
    sets = 1 if case["shared"] else int((client_counts(case) > 0).sum())
    moved = n * k * size + n * m * size * (3 if case["activation"] != "none" and case["phase"] == "train" else
                                           1) + sets * (m * k + m) * size
    if case["activation"] != "none" and case["phase"] == "train":
      moved -= n * m * size  # y and z written; the input's pre-activation is counted below
    if case["residual"]:
      moved += n * m * size
    flops = 2 * n * m * k
    if case["phase"] == "train":
      moved += n * m * size + n * k * size * (2 if case["activation"] != "none" else 1) + c * (m * k + m) * 4
      flops *= 3
    return dict(bytes=moved, flops=flops)
  t = min(case["top"], case["vocab"])
  moved = n * case["vocab"] * size + n * t * 8 + n * 4 + c * 4
  if case["phase"] == "train":
    moved += n * case["vocab"] * size
  return dict(bytes=moved, flops=6 * n * case["vocab"])


def run(state):
  if own:
    return _own_run(state)
  return _PLAIN[state["op"]](state)


# --- the framework's operators ------------------------------------------------


def _own_run(st):
  from federated_amd import client_ops as ops  # pylint: disable=g-import-not-at-top
  if st["op"] == "layer_norm":
    y, mean, rstd = ops.layer_norm(st["x"], st["weight"], st["bias"], st["batch"])
    if not st["backward"]:
      return y, mean, rstd
    dx, dw, db = ops.layer_norm_backward(st["dy"], st["x"], mean, rstd, st["weight"], st["batch"],
                                         dweight=st["dweight"], dbias=st["dbias"])
    return y, mean, rstd, dx, dw, db
  if st["op"] == "linear":
    act = None if st["activation"] == "none" else st["activation"]
    if st["phase"] == "forward":
      return ops.linear(st["x"], st["weight"], st["bias"], st["batch"], activation=act, residual=st["residual"])
    keep = act is not None
    out = ops.linear(st["x"], st["weight"], st["bias"], st["batch"], activation=act, residual=st["residual"],
                     preactivation=keep)
    dx = ops.linear_backward_input(st["dz"], st["weight"], st["batch"], preactivation=st["before"], activation=act)
    dw, db = ops.linear_backward_weight(st["dz"], st["x"], st["batch"], dweight=st["dweight"], dbias=st["dbias"])
    return (*out, dx, dw, db) if keep else (out, dx, dw, db)
  if st["op"] == "top_logits":
    return ops.top_logits(st["logits"], min(st["top"], st["vocab"]))
  if st["phase"] == "loss":
    return ops.distillation(st["logits"], st["index"], st["values"], st["batch"], temperature=st["temperature"],
                            teacher_lse=st["teacher_lse"])[0]
  return ops.distillation_with_gradient(st["logits"], st["index"], st["values"], st["batch"],
                                        temperature=st["temperature"], teacher_lse=st["teacher_lse"])


# --- the same in plain torch operations, float32 --------------------------------


def _pad(st, rows):
  out = rows.new_zeros(len(st["counts"]) * st["longest"], rows.shape[1])
  return out.index_copy_(0, st["place"], rows).unflatten(0, (-1, st["longest"]))


def _plain_layer_norm(st):
  x = st["x"].float()
  shared = st["weight"].stride(0) == 0
  weight = st["weight"][0].float() if shared else st["weight"].float()[st["client"]]
  bias = st["bias"][0].float() if shared else st["bias"].float()[st["client"]]
  mean = x.mean(1, keepdim=True)
  centred = x - mean
  rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
  hat = centred * rstd
  y = (hat * weight + bias).to(st["x"].dtype)
  if not st["backward"]:
    return y, mean[:, 0], rstd[:, 0]
  dy = st["dy"].float()
  a = dy * weight
  dx = rstd * (a - a.mean(1, keepdim=True) - hat * (a * hat).mean(1, keepdim=True))
  dw, db = _pad(st, dy * hat).sum(1), _pad(st, dy).sum(1)
  return y, mean[:, 0], rstd[:, 0], dx.to(st["x"].dtype), dw, db


def _act(name, z):
  if name == "relu":
    return torch.clamp(z, min=0)
  if name == "gelu":
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
  if name == "silu":
    return z / (1 + torch.exp(-z))
  return z


def _act_slope(name, z):
  if name == "relu":
    return (z > 0).to(z.dtype)
  if name == "gelu":
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
  if name == "silu":
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))
  return torch.ones_like(z)


def _plain_linear(st):
  dtype, shared = st["x"].dtype, st["weight"].stride(0) == 0
  if shared:
    z = st["x"].float() @ st["weight"][0].float().t() + st["bias"][0].float()
  else:
    weight = st["weight"].float()
    z = torch.bmm(_pad(st, st["x"].float()), weight.transpose(1, 2)) + st["bias"].float()[:, None]
    z = z.flatten(0, 1)[st["place"]]
  y = _act(st["activation"], z)
  if st["residual"] is not None:
    y = y + st["residual"].float()
  if st["phase"] == "forward":
    return y.to(dtype)
  dz = st["dz"].float()
  dzp = _pad(st, dz)
  if shared:
    dx = dz @ st["weight"][0].float()
  else:
    dx = torch.bmm(dzp, weight).flatten(0, 1)[st["place"]]
  if st["before"] is not None:
    dx = dx * _act_slope(st["activation"], st["before"].float())
  dw = torch.bmm(dzp.transpose(1, 2), _pad(st, st["x"].float()))
  db = dzp.sum(1)
  if st["activation"] == "none":
    return y.to(dtype), dx.to(dtype), dw, db
  return y.to(dtype), z.to(dtype), dx.to(dtype), dw, db


def _plain_top_logits(st):
  logits, t = st["logits"], min(st["top"], st["vocab"])
  # an integer per logit that orders like it, the index below it: ties to the lowest
  bits = (logits.float() + 0.0).view(torch.int32)
  rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
  key = rank * (1 << 32) + (st["vocab"] - torch.arange(st["vocab"], device=logits.device))
  index = st["vocab"] - (torch.topk(key, t, dim=1).values & 0xFFFFFFFF)
  wide = logits.float()
  top = wide.max(1, keepdim=True).values
  lse = top[:, 0] + torch.log(torch.exp(wide - top).sum(1))
  return index.to(torch.int32), torch.gather(logits, 1, index), lse


def _plain_distillation(st):
  tau = st["temperature"]
  s = st["logits"].float() / tau
  there = st["index"] >= 0
  index = torch.clamp(st["index"], min=0).long()
  t = torch.where(there, st["values"] / tau, -math.inf)
  if st["teacher_lse"] is None:
    top = torch.clamp(t.max(1, keepdim=True).values, min=-1e30)
    total = torch.exp(t - top).sum(1, keepdim=True)
    logp = t - top - torch.log(torch.clamp(total, min=1e-30))
  else:
    logp = t - st["teacher_lse"][:, None]
  p = torch.exp(logp)
  high = s.max(1, keepdim=True).values
  lse = high + torch.log(torch.exp(s - high).sum(1, keepdim=True))
  logq = torch.gather(s, 1, index) - lse
  row = tau * tau * (p * torch.where(there, logp - logq, 0.0)).nan_to_num(nan=0.0).sum(1)
  weight = 1.0 / st["count"].float()[st["client"]]
  loss = _pad(st, (weight * row)[:, None]).sum((1, 2))
  if st["phase"] == "loss":
    return loss
  grad = p.sum(1, keepdim=True) * torch.exp(s - lse)
  grad.scatter_add_(1, index, -p)
  return loss, (grad * (tau * weight)[:, None]).to(st["logits"].dtype)


_PLAIN = {"layer_norm": _plain_layer_norm, "linear": _plain_linear, "top_logits": _plain_top_logits,
          "distillation": _plain_distillation}


# --- the definitions in float64, client by client, row block by row block --------


def exact(case, seed):
  if case["op"] == "linear" and case["rows"] * case["inner"] * case["outer"] > 2e12:
    return None
  st = prepare(case, seed)
  if case["op"] == "top_logits":
    return _exact_top_logits(st)
  ends = np.cumsum(st["counts"])
  spans = [(int(e - c), int(e)) for e, c in zip(ends, st["counts"])]
  return {"layer_norm": _exact_layer_norm, "linear": _exact_linear,
          "distillation": _exact_distillation}[case["op"]](st, spans)


def _exact_layer_norm(st, spans):
  n, d = st["x"].shape
  wide = dict(dtype=torch.float64, device="cuda")
  y, mean, rstd, dx = torch.empty(n, d, **wide), torch.empty(n, **wide), torch.empty(n, **wide), None
  if st["backward"]:
    dx = torch.empty(n, d, **wide)
    dw, db = torch.zeros(len(spans), d, **wide), torch.zeros(len(spans), d, **wide)
  for c, (lo, hi) in enumerate(spans):
    if lo == hi:
      continue
    x, g, b = st["x"][lo:hi].double(), st["weight"][c].double(), st["bias"][c].double()
    mu = x.sum(1) / d
    var = ((x - mu[:, None]) ** 2).sum(1) / d
    s = (var + 1e-5) ** -0.5
    hat = (x - mu[:, None]) * s[:, None]
    y[lo:hi], mean[lo:hi], rstd[lo:hi] = g * hat + b, mu, s
    if st["backward"]:
      dy = st["dy"][lo:hi].double()
      dhat = dy * g
      along = (dhat * hat).sum(1, keepdim=True) / d
      dx[lo:hi] = (dhat - dhat.sum(1, keepdim=True) / d - hat * along) * s[:, None]
      dw[c], db[c] = (dy * hat).sum(0), dy.sum(0)
  return (y, mean, rstd, dx, dw, db) if st["backward"] else (y, mean, rstd)


def _exact_linear(st, spans):
  n = st["x"].shape[0]
  c_all, m, k = st["weight"].shape
  wide = dict(dtype=torch.float64, device="cuda")
  y, z, train = torch.empty(n, m, **wide), torch.empty(n, m, **wide), st["phase"] == "train"
  if train:
    dx, dw, db = torch.empty(n, k, **wide), torch.zeros(c_all, m, k, **wide), torch.zeros(c_all, m, **wide)
  for c, (lo, hi) in enumerate(spans):
    if lo == hi:
      continue
    w = st["weight"][c].double()
    x = st["x"][lo:hi].double()
    z[lo:hi] = x @ w.t() + st["bias"][c].double()
    u = z[lo:hi]
    if st["activation"] == "relu":
      y[lo:hi] = torch.where(u > 0, u, 0.0)
    elif st["activation"] == "gelu":
      y[lo:hi] = u * 0.5 * torch.special.erfc(-u / math.sqrt(2.0))
    elif st["activation"] == "silu":
      y[lo:hi] = u * torch.sigmoid(u)
    else:
      y[lo:hi] = u
    if st["residual"] is not None:
      y[lo:hi] += st["residual"][lo:hi].double()
    if train:
      dz = st["dz"][lo:hi].double()
      g = dz @ w
      if st["before"] is not None:
        u = st["before"][lo:hi].double()
        if st["activation"] == "relu":
          g = torch.where(u > 0, g, 0.0)
        elif st["activation"] == "gelu":
          g = g * (0.5 * torch.special.erfc(-u / math.sqrt(2.0)) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi))
        else:
          sig = torch.sigmoid(u)
          g = g * (sig + u * sig * (1 - sig))
      dx[lo:hi], dw[c], db[c] = g, dz.t() @ x, dz.sum(0)
  if not train:
    return y
  return (y, dx, dw, db) if st["activation"] == "none" else (y, z, dx, dw, db)


def _exact_top_logits(st):
  n, v = st["logits"].shape
  t = min(st["top"], v)
  index = torch.empty(n, t, dtype=torch.int32, device="cuda")
  values = torch.empty(n, t, dtype=torch.float64, device="cuda")
  lse = torch.empty(n, dtype=torch.float64, device="cuda")
  block = max(1, (1 << 26) // v)
  for lo in range(0, n, block):
    wide = st["logits"][lo:lo + block].double()
    order = torch.sort(wide, dim=1, descending=True, stable=True)
    index[lo:lo + block], values[lo:lo + block] = order.indices[:, :t].int(), order.values[:, :t]
    lse[lo:lo + block] = torch.logsumexp(wide, 1)
  return index, values, lse


def _exact_distillation(st, spans):
  tau = float(st["temperature"])
  n, v = st["logits"].shape
  loss = torch.zeros(len(spans), dtype=torch.float64, device="cuda")
  grad = torch.empty(n, v, dtype=torch.float64, device="cuda") if st["phase"] == "train" else None
  block = max(1, (1 << 26) // v)
  for c, (begin, end) in enumerate(spans):
    for lo in range(begin, end, block):
      hi = min(end, lo + block)
      logq = torch.log_softmax(st["logits"][lo:hi].double() / tau, 1)
      index = st["index"][lo:hi].long()
      there = (index >= 0).double()
      index = torch.clamp(index, min=0)
      if st["teacher_lse"] is None:
        p = there * torch.exp((st["values"][lo:hi].double() - 8.0) / tau)
        p = p / torch.clamp(p.sum(1, keepdim=True), min=1e-300)
      else:
        p = there * torch.exp(st["values"][lo:hi].double() / tau - st["teacher_lse"][lo:hi].double()[:, None])
      rows = torch.special.xlogy(p, p) - p * torch.gather(logq, 1, index)
      loss[c] += tau * tau * rows.sum() / (end - begin)
      if grad is not None:
        g = p.sum(1, keepdim=True) * torch.exp(logq)
        g.scatter_add_(1, index, -p)
        grad[lo:hi] = g * (tau / (end - begin))
  return loss if grad is None else (loss, grad)
