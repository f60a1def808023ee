"""Operators of the clients' local step, batched over a round's clients.

What a round's codec reads -- one float32 row of P elements per client -- is made by
every sampled client's local step (trainer.py:286-291 hands the model's deltas to the
aggregator).  These operators run that step's products, norms and losses for all of
a round's clients in one launch each:

  - a ``ClientBatch`` says which rows of an activation tensor are whose (any number
    per client, none included);
  - weights are [clients, ...] tensors with any client stride: views into the
    clients' flat parameter rows ([clients, P], one row per client), or one weight
    broadcast to all clients (``expand``, stride 0: a round's first step);
  - weight gradients are float32 and can be written straight into views of the
    [clients, P] rows that ``codec.quantize_encode`` and the aggregators take.

Activations and weights are float32, bfloat16 or float16, of one type per call;
sums, statistics and gradients of weights are held in float32.  All calls are
asynchronous on the current stream of the tensors' device, allocate what they return
(unless given ``out``) and keep nothing.  Rows behind the batch's last are not read;
in a given output they are left as they were, in an allocated one they are zero.  A
given output shares no memory with the call's other tensors (rows side by side in one
buffer are apart), but may be ``residual`` itself.  A batch whose calls were captured
into a graph has to live as long as the graph.

Forward and backward are separate calls with explicit gradients: a broadcast weight
still gets one gradient per client, which is what the codec encodes.  The calls are no
part of torch's autograd: an input's ``requires_grad`` is not looked at, and outputs carry
no graph.
"""
import ctypes
import functools
import math
import operator

import numpy as np
import torch

from federated_amd import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}
_TILES = (16, 32, 128, 256)
MAX_TOP = 1024  # FC_MAX_TOP
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-15, 1e15  # FC_MIN_TEMPERATURE, FC_MAX_TEMPERATURE


class ClientBatch:
  """Which rows belong to which client: ``counts[c]`` rows for client c, in order.

  Built once per round from the clients' row counts (host integers); holds the
  offsets and the row-tile tables the kernels read on ``device``.
  """

  def __init__(self, counts, device=None):
    _lib.require_gpu()
    counts = np.ascontiguousarray(np.asarray(counts))
    if counts.ndim != 1 or counts.size == 0:
      raise ValueError("counts must be a non-empty list of row counts")
    if not np.issubdtype(counts.dtype, np.integer):
      raise ValueError("row counts must be integers, got %s" % counts.dtype)
    counts = counts.astype(np.int64)
    if counts.min() < 0:
      raise ValueError("row counts must not be negative")
    # each first: a sum of any may wrap
    if int(counts.max()) >= (1 << 31) - 1024 or int(counts.sum()) >= (1 << 31) - 1024:
      raise ValueError("a batch holds fewer than 2^31 - 1024 rows")
    self.device = torch.device("cuda" if device is None else device)
    if self.device.type != "cuda":
      raise ValueError("a ClientBatch lives on the GPU, got %s" % self.device)
    if self.device.index is None:
      self.device = torch.device("cuda", torch.cuda.current_device())
    self.counts = counts
    self.num_clients = int(counts.size)
    self.num_rows = int(counts.sum())
    self.longest = int(counts.max())
    ends = np.cumsum(counts)
    # one host buffer, one copy: offsets, row -> client, a table entry per client, tiles
    parts = [np.concatenate([[0], ends]).astype(np.int32),
             np.repeat(np.arange(counts.size, dtype=np.int32), counts),
             np.stack([np.arange(counts.size), ends - counts, counts, np.zeros_like(counts)], 1).astype(np.int32)]
    for rows in _TILES:
      parts.extend(self._tile_table(rows))
    starts, at = [], 0
    for p in parts:
      starts.append(at)
      at += (p.size + 3) // 4 * 4  # 16-byte aligned
    host = np.zeros(at, np.int32)
    for p, s in zip(parts, starts):
      host[s:s + p.size] = p.reshape(-1)
    dev = torch.from_numpy(host).to(self.device)
    self._buffer, self._streams = dev, {torch.cuda.current_stream(self.device).cuda_stream}
    views = [dev[s:s + p.size] for p, s in zip(parts, starts)]
    self.offsets, self.row_client, self._clients = views[:3]
    self._tiles = {rows: (views[3 + 2 * i], views[4 + 2 * i], parts[3 + 2 * i].shape[0])
                   for i, rows in enumerate(_TILES)}
    self.tile_counts = tuple(self._tiles[rows][2] for rows in _TILE_COSTS)

  def _used_on(self, stream):
    """The tables are read on another stream than they were made on (a raw handle, the current one)."""
    self._buffer.record_stream(torch.cuda.current_stream(self.device))
    self._streams.add(stream)

  def _tile_table(self, rows):
    lib = _lib.load()
    counts = self.counts.ctypes.data_as(ctypes.c_void_p)
    n = int(lib.fc_client_tiles(counts, self.num_clients, rows, None, None))
    if n < 0:
      _lib.check(n)
    tiles = np.zeros((n, 4), np.int32)
    first = np.zeros(self.num_clients + 1, np.int32)
    lib.fc_client_tiles(counts, self.num_clients, rows, tiles.ctypes.data_as(ctypes.c_void_p),
                        first.ctypes.data_as(ctypes.c_void_p))
    return tiles, first


# --- argument checks -------------------------------------------------------------


def _activations(name, t, batch, width=None, like=None):
  if not isinstance(t, torch.Tensor) or t.dim() != 2:
    raise ValueError("%s must be a [rows, width] tensor" % name)
  if t.dtype not in _DTYPES:
    raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
  if like is not None and t.dtype != like.dtype:
    raise ValueError("%s is %s, expected %s" % (name, t.dtype, like.dtype))
  if t.device != batch.device:
    raise ValueError("%s is on %s, the batch on %s" % (name, t.device, batch.device))
  if t.shape[0] < batch.num_rows:
    raise ValueError("%s has %d rows, the batch %d" % (name, t.shape[0], batch.num_rows))
  if t.shape[1] == 0 or (width is not None and t.shape[1] != width):
    raise ValueError("%s has width %d%s" % (name, t.shape[1], "" if width is None else ", expected %d" % width))
  _rows_ok(name, t)
  return t


def _rows_ok(name, t):
  if t.shape[-1] > 1 and t.stride(-1) != 1:
    raise ValueError("%s must be contiguous along its last axis" % name)


def _distinct(name, t):
  """An output whose elements must not overlap."""
  need = 1
  for size, stride in sorted(zip(t.shape, t.stride()), key=lambda p: p[1]):
    if size > 1:
      if stride < need:
        raise ValueError("%s has overlapping elements" % name)
      need = stride * (size - 1) + need
  return t


def _params(name, t, batch, shape, dtype):
  if not isinstance(t, torch.Tensor) or tuple(t.shape) != (batch.num_clients,) + shape:
    raise ValueError("%s must be a %s tensor, got %s" % (
        name, [batch.num_clients] + list(shape), list(t.shape) if isinstance(t, torch.Tensor) else type(t)))
  if t.dtype != dtype:
    raise ValueError("%s is %s, expected %s" % (name, t.dtype, dtype))
  if t.device != batch.device:
    raise ValueError("%s is on %s, the batch on %s" % (name, t.device, batch.device))
  _rows_ok(name, t)
  return t


def _grad_out(name, t, batch, shape, *others):
  if t is None:
    return torch.empty((batch.num_clients,) + shape, dtype=torch.float32, device=batch.device)
  _distinct(name, _params(name, t, batch, shape, torch.float32))
  _apart(name, t, None, *others)
  return t


def _out(name, out, like, batch, width, itself=None, *others):
  if out is not None:
    _distinct(name, _activations(name, out, batch, width, like))
    _apart(name, out, itself, *others)
    return out
  out = torch.empty((like.shape[0], width), dtype=like.dtype, device=like.device)
  if like.shape[0] > batch.num_rows:
    out[batch.num_rows:].zero_()
  return out


def _extent(t):
  """(first byte, bytes of an outermost entry, bytes between those, entries)."""
  size = t.element_size()
  inner = 1
  for n, stride in zip(t.shape[1:], t.stride()[1:]):
    inner += (n - 1) * stride
  return t.data_ptr(), inner * size, t.stride(0) * size, t.shape[0]


def _apart(name, out, itself, *others):
  """A given output that must not share memory with the call's other tensors.

  Rows side by side in a wider buffer are apart; ``itself`` may be ``out``.
  """
  if itself is not None and itself.data_ptr() == out.data_ptr() and itself.stride() == out.stride():
    itself = None
  start, inner, outer, n = _extent(out)
  end = start + (n - 1) * outer + inner
  storage = out.untyped_storage().data_ptr()
  for t in (itself,) + others:
    # the two cheap tests end nearly all pairs
    if t is None or t.data_ptr() >= end or t.untyped_storage().data_ptr() != storage or not n or not t.shape[0]:
      continue
    start2, inner2, outer2, n2 = _extent(t)
    if start2 + (n2 - 1) * outer2 + inner2 <= start:
      continue
    if outer == outer2 > 0 and (start2 - start) % outer >= inner and (start - start2) % outer >= inner2:
      continue
    raise ValueError("%s shares memory with another tensor of the call (%s)" % (name, list(t.shape)))


def _vector(name, t, rows, device):
  if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.dtype != torch.float32 or t.shape[0] < rows:
    raise ValueError("%s must be a float32 vector of at least %d" % (name, rows))
  if t.device != device:
    raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
  if t.shape[0] > 1 and t.stride(0) != 1:
    raise ValueError("%s must be contiguous" % name)
  return t


def _stats(rows, batch):
  t = torch.empty(rows, dtype=torch.float32, device=batch.device)
  if rows > batch.num_rows:
    t[batch.num_rows:].zero_()
  return t


def _ptr(t):
  return None if t is None else t.data_ptr()


def _ld(t):
  return 0 if t is None else t.stride(0)


def _call(where, name, *args):
  """A C entry point on the current stream of `where`: a batch, or a device."""
  batch = where if isinstance(where, ClientBatch) else None
  device = batch.device if batch else where
  index = device.index
  # the raw handle: torch.cuda.current_stream(device) makes a Stream object, at 2 us a
  # sixth of a small call
  stream = torch._C._cuda_getCurrentRawStream(index)  # pylint: disable=protected-access
  if batch and stream not in batch._streams:  # pylint: disable=protected-access
    batch._used_on(stream)  # pylint: disable=protected-access
  fn = getattr(_lib.load(), name)
  if index == torch.cuda.current_device():
    rc = fn(*args, stream)
  else:
    with torch.cuda.device(device):
      rc = fn(*args, stream)
  if rc:
    _lib.check(rc)


# --- layer norm ------------------------------------------------------------------


def layer_norm(x, weight, bias, batch, eps=1e-5, out=None):
  """y = (x - mean) rstd weight_c + bias_c over the last axis, client by client.

  ``weight`` / ``bias``: [clients, dim] of x's type, or None.  Returns (y, mean,
  rstd), the statistics as float32 [rows] for the backward pass.
  """
  _activations("x", x, batch)
  dim = x.shape[1]
  for name, t in (("weight", weight), ("bias", bias)):
    if t is not None:
      _params(name, t, batch, (dim,), x.dtype)
  if not 0.0 <= float(eps) < float("inf"):
    raise ValueError("eps must not be negative, got %r" % (eps,))
  out = _out("out", out, x, batch, dim, None, x, weight, bias)
  mean, rstd = _stats(x.shape[0], batch), _stats(x.shape[0], batch)
  tiles, _, ntiles = batch._tiles[16]  # pylint: disable=protected-access
  _call(batch, "fc_layer_norm", _ptr(x), x.stride(0), _DTYPES[x.dtype], _ptr(tiles), ntiles, dim,
        _ptr(weight), _ld(weight), _ptr(bias), _ld(bias), float(eps), _ptr(out), out.stride(0), _ptr(mean),
        _ptr(rstd))
  return out, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight, batch, residual=None, dweight=None, dbias=None,
                        accumulate=False, out=None):
  """Gradients of ``layer_norm``: (dx, dweight, dbias).

  ``residual``: a gradient added to dx (the branch around the norm).  ``dweight`` /
  ``dbias``: float32 [clients, dim] outputs (views of the clients' rows), allocated
  when None; ``accumulate`` adds to the given ones.  A client without rows gets zeros.
  """
  _activations("x", x, batch)
  dim = x.shape[1]
  _activations("dy", dy, batch, dim, x)
  _vector("mean", mean, batch.num_rows, batch.device)
  _vector("rstd", rstd, batch.num_rows, batch.device)
  if weight is not None:
    _params("weight", weight, batch, (dim,), x.dtype)
  if residual is not None:
    _activations("residual", residual, batch, dim, x)
  if accumulate and (dweight is None or dbias is None):
    raise ValueError("accumulate needs dweight and dbias to add to")
  dbias = _grad_out("dbias", dbias, batch, (dim,), dy, x, mean, rstd, weight, residual)
  dweight = _grad_out("dweight", dweight, batch, (dim,), dbias, dy, x, mean, rstd, weight, residual)
  out = _out("out", out, x, batch, dim, residual, dweight, dbias, dy, x, mean, rstd, weight)
  tiles, first, ntiles = batch._tiles[32]  # pylint: disable=protected-access
  part = torch.empty(ntiles * 2 * dim, dtype=torch.float32, device=batch.device)
  _call(batch, "fc_layer_norm_backward", _ptr(dy), dy.stride(0), _ptr(x), x.stride(0), _DTYPES[x.dtype],
        _ptr(mean), _ptr(rstd), _ptr(tiles), ntiles, _ptr(first), batch.num_clients, dim, _ptr(weight), _ld(weight),
        _ptr(residual), _ld(residual), _ptr(out), out.stride(0), _ptr(dweight), dweight.stride(0), _ptr(dbias),
        dbias.stride(0), int(bool(accumulate)), _ptr(part))
  return out, dweight, dbias


# --- linear ----------------------------------------------------------------------


def _activation(activation):
  if activation not in _ACTIVATIONS:
    raise ValueError("activation must be None, 'relu', 'gelu' or 'silu', got %r" % (activation,))
  return _ACTIVATIONS[activation]


def _weight(weight, batch, dtype, inner=None, outer=None):
  if not isinstance(weight, torch.Tensor) or weight.dim() != 3:
    raise ValueError("weight must be a [clients, out_features, in_features] tensor")
  m, k = weight.shape[1:]
  if m == 0 or k == 0 or (inner is not None and k != inner) or (outer is not None and m != outer):
    raise ValueError("weight is [clients, %d, %d], expected [clients, %s, %s]" % (
        m, k, "out" if outer is None else outer, "in" if inner is None else inner))
  _params("weight", weight, batch, (m, k), dtype)
  return m, k


# How long a product takes with tiles of `rows` rows, from one card's measurements (us):
# a CU's time for one 128-byte k-step of one tile in 16-bit types (1.03 us for two 128 x
# 128 tiles side by side, 1.8 for one of 256 x 256, 1.2 for four of 32 x 128) and in
# float32 (the matrix unit's time), a tile's start and end, and how many a CU holds.  A
# k-step takes 0.9 however little it computes, from the wait for memory.
_TILE_COSTS = {32: (0.3, 0.53, 5.0, 4), 128: (0.52, 2.08, 9.0, 2), 256: (1.8, 0.0, 12.0, 1)}
_STEP_LATENCY = 0.9
# a further launch (the parts' join; a copy costs two, with its allocation), on the host: what
# counts in small calls
_LAUNCH = 8.0
_CUS = 256
_WALK = -1  # FC_WALK


@functools.lru_cache(maxsize=4096)
def _estimate(tiles, steps, longest, size, aligned):
  """(us, tile rows, splits of the contraction) of a product, by the lowest estimate.

  ``tiles``: output tiles for each of _TILE_COSTS' heights; ``steps`` / ``longest``: the
  mean and the largest number of k-steps of a tile.  Splitting pays where there are
  fewer tiles than the chip holds: 1 x 4096 by 14336 x 4096 (bfloat16) takes 56 us whole
  and 29 in four parts; where the tiles fill it, it only costs (64 clients, 20480 rows, 96
  to 10004: 287 us whole, 1057 in two).
  """
  best = None
  for (rows, (step16, step32, ends, resident)), count in zip(_TILE_COSTS.items(), tiles):
    if rows == 256 and (size == 4 or not aligned):
      continue  # the kernel's limits
    step = step32 if size == 4 else step16
    splits = 1
    while splits <= 16 and (splits == 1 or 2 * splits <= longest):
      blocks = max(1, count * splits)
      rounds, rest = divmod(blocks, _CUS * resident)
      each = max(_STEP_LATENCY * longest, resident * step * steps) / splits + ends
      if rounds >= 4:  # workgroups no longer start and end together
        t = blocks / (_CUS * resident) * each
      else:
        t = rounds * each
        if rest:
          t += max(_STEP_LATENCY * longest, -(-rest // _CUS) * step * steps) / splits + ends
      if splits > 1:  # the parts' write and read, and the joining launch
        t += _LAUNCH + 3 * blocks * rows * max(128, rows) * 4 / 4e6
      if best is None or t < best[0]:
        best = (t, rows, splits)
      splits *= 2
  return best


def _plan(tiles, steps, longest, size, aligned):
  return _estimate(tiles, steps, longest, size, aligned)[1:]


def _odd(t):
  """Whether some row of a 16-bit operand starts at an odd element (of a 4-byte word).

  Or the rows are too far apart for 32-bit offsets inside a tile.
  """
  return t.data_ptr() & 3 or (t.stride(0) | t.stride(-2)) & 1 or t.stride(-2) >= 1 << 22


def _matrices(t, rows):
  """(how many, rows of each) an operand holds: [rows, width], or [clients, out, in]."""
  if t.dim() == 2:
    return 1, rows
  return (1 if t.stride(0) == 0 else t.shape[0]), t.shape[1]


def _packs(t, rows):
  """Whether one launch copies the operand: below 2^24 blocks of 256 vectors."""
  clients, per = _matrices(t, rows)
  return clients * -(-per * ((t.shape[-1] + 7) // 8) // 256) < 1 << 24


def _packed(t, rows):
  """``t``'s rows ([rows, width], or [clients, out, in]) at a stride of whole vectors."""
  width = t.shape[-1]
  stride = (width + 7) // 8 * 8
  clients, per = _matrices(t, rows)
  if t.dim() == 2:
    client_stride = 0
    out = torch.empty((rows, stride), dtype=t.dtype, device=t.device)
  else:
    client_stride = t.stride(0)
    out = torch.empty((clients, per, stride), dtype=t.dtype, device=t.device)
  _call(t.device, "fc_pack_rows", _ptr(t), client_stride, t.stride(-2), _DTYPES[t.dtype], clients, per, width, _ptr(out),
        stride)
  return out.expand(t.shape[0], per, stride) if t.dim() == 3 else out


def _operands(a, b, rows, tiles, steps, longest):
  """A product's operands as it reads them: (a, b, tile rows, splits).

  Rows of a 16-bit operand at odd elements go through registers, at about 2.2 times a
  step's cost (two thirds of the load rate, and the wait is in the step); copied to
  whole vectors first they do not.  Copying pays where a row is read by many tiles: 33
  clients, 9001 rows in all, 1021 to 2050 (float16): 120 + 196 + 183 us as they are,
  against 100 + 90 + 148 with the copies.
  """
  size = a.element_size()
  odd = (_odd(a), _odd(b)) if size == 2 else (0, 0)
  if (odd[0] or odd[1]) and rows and all(_packs(t, rows) for o, t in zip(odd, (a, b)) if o):
    copies = sum(2 * _LAUNCH + math.prod(_matrices(t, rows)) * t.shape[-1] * 4 / 4e6 for o, t in zip(odd, (a, b)) if o)
    if _estimate(tiles, steps, longest, 2, True)[0] + copies < 2.2 * _estimate(tiles, steps, longest, 2, False)[0]:
      if odd[0]:
        a = _packed(a, rows)
      if odd[1]:
        b = _packed(b, rows)
      odd = (0, 0)
  height, splits = _plan(tiles, steps, longest, size, not (odd[0] or odd[1]))
  return a, b, height, splits


def _workspace(blocks, rows, splits, device):
  if splits in (1, _WALK):
    return None
  need = int(_lib.load().fc_linear_workspace_bytes(blocks, rows, splits))
  return torch.empty(need, dtype=torch.uint8, device=device)


def _walks(batch, columns, a, weight):
  """Whether blocks that walk along the columns make the product faster.

  A short contraction of 16-bit types, row tiles that are not mostly empty, and tiles for
  every place on the chip: 64 clients of 320 rows, 96 to 10004: 204 us against 287 in the
  best tiles, 96 to 1000: 24 against 34; of 20 rows, 96 to 10004: 46 against 33.
  """
  n = batch.tile_counts[1]
  return (a.element_size() == 2 and a.shape[1] <= 128 and batch.num_rows >= 48 * n and n * -(-columns // 128) >= 512 and
          not (_odd(a) or _odd(weight)))


def _row_product(batch, columns, a, weight):
  """_operands for an output of the activations' rows by `columns`; and the row tiles."""
  n32, n128, n256 = batch.tile_counts
  narrow, wide = -(-columns // 128), -(-columns // 256)
  steps = -(-a.shape[1] * a.element_size() // 128)
  a, weight, rows, splits = _operands(a, weight, batch.num_rows, (n32 * narrow, n128 * narrow, n256 * wide), steps, steps)
  if _walks(batch, columns, a, weight):
    rows, splits = 128, _WALK
  tiles, _, ntiles = batch._tiles[rows]  # pylint: disable=protected-access
  ws = _workspace(ntiles * (wide if rows == 256 else narrow), rows, splits, batch.device)
  return a, weight, (_ptr(tiles), ntiles, rows), (splits, _ptr(ws), 0 if ws is None else ws.numel()), ws


def linear(x, weight, bias, batch, activation=None, residual=None, preactivation=False, out=None):
  """y = activation(x weight_c^T + bias_c) + residual, client by client.

  ``weight``: [clients, out_features, in_features]; ``bias``: [clients, out_features]
  or None, both of x's type.  ``activation``: None, "relu", "gelu" (the exact one) or
  "silu".  With ``preactivation`` returns (y, z), z the value under the activation
  (rounded to x's type), which the backward pass of the next operator down reads.
  """
  _activations("x", x, batch)
  act = _activation(activation)
  m, k = _weight(weight, batch, x.dtype, inner=x.shape[1])
  if bias is not None:
    _params("bias", bias, batch, (m,), x.dtype)
  if residual is not None:
    _activations("residual", residual, batch, m, x)
  out = _out("out", out, x, batch, m, residual, x, weight, bias)
  z = _out("z", None, x, batch, m) if preactivation else None
  x, weight, tiles, last, _ws = _row_product(batch, m, x, weight)
  _call(batch, "fc_linear", _ptr(x), x.stride(0), _DTYPES[x.dtype], *tiles, batch.num_clients, k, m,
        _ptr(weight), weight.stride(0), weight.stride(1), _ptr(bias), _ld(bias), act, _ptr(residual), _ld(residual),
        _ptr(z), _ld(z), _ptr(out), out.stride(0), *last)
  return (out, z) if preactivation else out


def linear_backward_input(dz, weight, batch, preactivation=None, activation=None, residual=None, out=None):
  """dx = (dz weight_c) * activation'(preactivation) + residual, client by client.

  ``dz``: the gradient at this product's pre-activation.  ``preactivation`` /
  ``activation``: of the operator below, so that dx is the gradient at ITS
  pre-activation.
  """
  act = _activation(activation)
  _activations("dz", dz, batch)
  m, k = _weight(weight, batch, dz.dtype, outer=dz.shape[1])
  if (act != 0) != (preactivation is not None):
    raise ValueError("activation and preactivation go together")
  if preactivation is not None:
    _activations("preactivation", preactivation, batch, k, dz)
  if residual is not None:
    _activations("residual", residual, batch, k, dz)
  out = _out("out", out, dz, batch, k, residual, dz, weight, preactivation)
  dz, weight, tiles, last, _ws = _row_product(batch, k, dz, weight)
  _call(batch, "fc_linear_backward_input", _ptr(dz), dz.stride(0), _DTYPES[dz.dtype], *tiles,
        batch.num_clients, k, m, _ptr(weight), weight.stride(0), weight.stride(1), act, _ptr(preactivation),
        _ld(preactivation), _ptr(residual), _ld(residual), _ptr(out), out.stride(0), *last)
  return out


def _few_rows(batch, columns, dtype):
  """Whether the weight gradient written for few rows is the faster one.

  Up to 8 rows always (60 clients of 8 rows, 1604 x 1105: 113 us against 175 in float32, 114
  against 130 in bfloat16); up to 16 where a matrix tile does worse, in float32 (16 rows:
  157 against 179; bfloat16 143 against 133) and of at most 64 columns (103 clients of 16
  rows, 10354 x 43, bfloat16: 99 against 135).
  """
  return batch.longest <= (16 if dtype == torch.float32 or columns <= 64 else 8)


def linear_backward_weight(dz, x, batch, dweight=None, dbias=None, bias=True, accumulate=False):
  """(dweight, dbias): dweight_c = sum over client c's rows of dz x^T, dbias_c of dz.

  float32 [clients, out_features, in_features] and [clients, out_features]: given
  (views of the clients' rows; ``accumulate`` adds to them) or allocated.  ``bias``
  False leaves dbias out (None).  A client without rows gets zeros.
  """
  _activations("x", x, batch)
  _activations("dz", dz, batch, None, x)
  m, k = dz.shape[1], x.shape[1]
  if not bias and dbias is not None:
    raise ValueError("dbias given with bias=False")
  if accumulate and (dweight is None or (bias and dbias is None)):
    raise ValueError("accumulate needs dweight and dbias to add to")
  if bias:
    dbias = _grad_out("dbias", dbias, batch, (m,), dz, x)
  dweight = _grad_out("dweight", dweight, batch, (m, k), dz, x, dbias)
  if _few_rows(batch, k, x.dtype):
    _call(batch, "fc_linear_backward_weight_few", _ptr(dz), dz.stride(0), _ptr(x), x.stride(0), _DTYPES[x.dtype],
          _ptr(batch._clients), batch.num_clients, batch.longest, k, m, _ptr(dweight), dweight.stride(0),  # pylint: disable=protected-access
          dweight.stride(1), _ptr(dbias), _ld(dbias), int(bool(accumulate)))
    return dweight, dbias
  tiles = tuple(batch.num_clients * -(-m // h) * -(-k // max(128, h)) for h in _TILE_COSTS)
  per = 128 // x.element_size()
  dz, x, rows, splits = _operands(dz, x, batch.num_rows, tiles, -(-batch.num_rows // (per * batch.num_clients)),
                                  -(-batch.longest // per))
  ws = _workspace(batch.num_clients * -(-m // rows) * -(-k // max(128, rows)), rows, splits, batch.device)
  _call(batch, "fc_linear_backward_weight", _ptr(dz), dz.stride(0), _ptr(x), x.stride(0), _DTYPES[x.dtype],
        _ptr(batch._clients), batch.num_clients, k, m, _ptr(dweight), dweight.stride(0), dweight.stride(1),  # pylint: disable=protected-access
        _ptr(dbias), _ld(dbias), int(bool(accumulate)), rows, splits, _ptr(ws), 0 if ws is None else ws.numel())
  return dweight, dbias


# --- top logits and distillation ---------------------------------------------------


def top_logits(logits, k, temperature=1.0):
  """The k largest logits of every row: (indices int32, values, lse).

  The message of a teacher: ``indices`` [rows, k] in falling order of value (ties to
  the lowest index; NaN below every number), ``values`` [rows, k] of the logits' type,
  ``lse`` float32 [rows] = log sum exp(logits / temperature) over the whole row.
  """
  if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or not logits.is_cuda:
    raise ValueError("logits must be a [rows, vocabulary] tensor on the GPU")
  if logits.dtype not in _DTYPES:
    raise ValueError("logits must be float32, bfloat16 or float16, got %s" % logits.dtype)
  _rows_ok("logits", logits)
  rows, vocab = logits.shape
  k = operator.index(k)
  if not 1 <= k <= min(vocab, MAX_TOP):
    raise ValueError("k must be in [1, %d], got %d" % (min(vocab, MAX_TOP), k))
  _temperature(temperature)
  index = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
  values = torch.empty((rows, k), dtype=logits.dtype, device=logits.device)
  lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
  _call(logits.device, "fc_top_logits", _ptr(logits), logits.stride(0), _DTYPES[logits.dtype], rows, vocab, k,
        float(temperature), _ptr(index), _ptr(values), _ptr(lse))
  return index, values, lse


def _temperature(t):
  if not MIN_TEMPERATURE <= float(t) <= MAX_TEMPERATURE:
    raise ValueError("temperature must be in [%g, %g], got %r" % (MIN_TEMPERATURE, MAX_TEMPERATURE, t))


def _teacher(logits, indices, values, batch, temperature, teacher_lse, row_weights):
  _activations("logits", logits, batch)
  _temperature(temperature)
  n = batch.num_rows
  for name, t, dtype in (("indices", indices, torch.int32), ("values", values, None)):
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.shape[0] < n or t.shape[1] != indices.shape[1]:
      raise ValueError("%s must be a [rows, k] tensor of at least %d rows" % (name, n))
    if t.device != batch.device:
      raise ValueError("%s is on %s, the batch on %s" % (name, t.device, batch.device))
    if dtype is not None and t.dtype != dtype:
      raise ValueError("%s is %s, expected %s" % (name, t.dtype, dtype))
  if not 1 <= indices.shape[1] <= MAX_TOP:
    raise ValueError("k must be in [1, %d], got %d" % (MAX_TOP, indices.shape[1]))
  if values.dtype not in _DTYPES:
    raise ValueError("values must be float32, bfloat16 or float16, got %s" % values.dtype)
  for name, t in (("teacher_lse", teacher_lse), ("row_weights", row_weights)):
    if t is not None:
      _vector(name, t, n, batch.device)
  return indices.contiguous(), values.float().contiguous()


def _distill(logits, indices, values, batch, temperature, teacher_lse, row_weights, lse, grad, want_loss, dloss):
  loss = torch.empty(batch.num_clients, dtype=torch.float32, device=batch.device) if want_loss else None
  row_loss = torch.empty(batch.num_rows, dtype=torch.float32, device=batch.device) if want_loss else None
  _call(batch, "fc_distill", _ptr(logits), logits.stride(0), _DTYPES[logits.dtype], batch.num_rows,
        logits.shape[1], _ptr(indices), _ptr(values), indices.shape[1], _ptr(batch.row_client), _ptr(batch.offsets),
        batch.num_clients, float(temperature), _ptr(teacher_lse), _ptr(row_weights), _ptr(dloss), _ptr(row_loss),
        _ptr(lse), _ptr(loss), _ptr(grad), _ld(grad))
  return loss


def distillation(logits, indices, values, batch, temperature=1.0, teacher_lse=None, row_weights=None):
  """Distillation loss of every client from a teacher's top logits: (loss, lse).

    p_k = exp(values_k / T - L),  q = softmax(logits / T)
    loss_c = sum over the client's rows of  w_r T^2 sum_k p_k (log p_k - log q[indices_k])

  ``indices`` / ``values``: [rows, k] as ``top_logits`` gives them; an index outside the
  vocabulary (-1) or a value of -inf is padding, and a row of nothing but padding has
  no loss and no gradient.  An index that comes twice counts twice.  L is
  ``teacher_lse`` (float32 [rows], at this temperature: p then sums to less than one,
  the rest of the teacher's mass is left out) or, when None, makes p sum to one.
  ``row_weights``: float32 [rows]; None: 1 / (the client's rows), the mean.  A row of
  weight 0 is not looked at.  ``lse`` (float32 [rows], of the logits at this temperature; NaN
  where a row was not looked at) is for ``distillation_backward``, whose teacher and
  weights may be others.
  """
  indices, values = _teacher(logits, indices, values, batch, temperature, teacher_lse, row_weights)
  lse = _stats(logits.shape[0], batch)
  loss = _distill(logits, indices, values, batch, temperature, teacher_lse, row_weights, lse, None, True, None)
  return loss, lse


def distillation_backward(logits, lse, indices, values, batch, temperature=1.0, teacher_lse=None, row_weights=None,
                          dloss=None, out=None):
  """Gradient of ``distillation`` by the logits; ``dloss``: float32 [clients] or None (ones).

  ``out`` may be ``logits`` itself.
  """
  indices, values = _teacher(logits, indices, values, batch, temperature, teacher_lse, row_weights)
  _vector("lse", lse, batch.num_rows, batch.device)
  if dloss is not None:
    _vector("dloss", dloss, batch.num_clients, batch.device)
  out = _out("out", out, logits, batch, logits.shape[1], logits, indices, values, lse, teacher_lse, row_weights, dloss)
  _distill(logits, indices, values, batch, temperature, teacher_lse, row_weights, lse, out, False, dloss)
  return out


def distillation_with_gradient(logits, indices, values, batch, temperature=1.0, teacher_lse=None, row_weights=None,
                               out=None):
  """(loss, gradient by the logits) of ``distillation`` in one pass over the logits.

  ``out`` may be ``logits`` itself.
  """
  indices, values = _teacher(logits, indices, values, batch, temperature, teacher_lse, row_weights)
  out = _out("out", out, logits, batch, logits.shape[1], logits, indices, values, teacher_lse, row_weights)
  loss = _distill(logits, indices, values, batch, temperature, teacher_lse, row_weights, None, out, True, None)
  return loss, out
