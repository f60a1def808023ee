"""The client-step operators' C entry points without a GPU: refusals come before any
device work, and the host-side row-tile table."""
import ctypes

import numpy as np
import pytest

from federated_amd import _lib

NULL = None


def _buf():
  return ctypes.addressof(ctypes.create_string_buffer(64))


def refused(rc, word):
  assert rc != 0 and word in _lib.load().fc_last_error(), (rc, _lib.load().fc_last_error())


def test_client_tiles_cover_every_row_once():
  lib = _lib.load()
  for counts, height in [([5], 16), ([0, 16, 0, 17, 1], 16), ([0, 0], 64), ([130, 128, 127], 128), ([1] * 300, 64)]:
    c = np.asarray(counts, np.int64)
    p = c.ctypes.data_as(ctypes.c_void_p)
    n = lib.fc_client_tiles(p, c.size, height, None, None)
    assert n == sum(-(-k // height) for k in counts)
    tiles, first = np.full((n, 4), -1, np.int32), np.full(c.size + 1, -1, np.int32)
    assert lib.fc_client_tiles(p, c.size, height, tiles.ctypes.data_as(ctypes.c_void_p),
                               first.ctypes.data_as(ctypes.c_void_p)) == n
    seen = []
    start = np.cumsum(c) - c
    for k in range(c.size):
      rows = [r for t in tiles[first[k]:first[k + 1]] for r in range(t[1], t[1] + t[2])]
      assert all(t[0] == k and 0 < t[2] <= height for t in tiles[first[k]:first[k + 1]])
      assert rows == list(range(start[k], start[k] + c[k]))
      seen += rows
    assert seen == list(range(c.sum())) and first[-1] == n


def test_client_tiles_refusals():
  lib = _lib.load()
  c = np.array([3, -1], np.int64)
  p = c.ctypes.data_as(ctypes.c_void_p)
  assert lib.fc_client_tiles(p, 2, 16, None, None) == -1 and b"negative" in lib.fc_last_error()
  assert lib.fc_client_tiles(None, 2, 16, None, None) == -1
  assert lib.fc_client_tiles(p, 0, 16, None, None) == -1
  assert lib.fc_client_tiles(p, 1, 0, None, None) == -1
  c[:] = 1 << 31, 1
  assert lib.fc_client_tiles(p, 2, 1 << 20, None, None) == -1 and b"too many rows" in lib.fc_last_error()


def test_layer_norm_refusals():
  lib, b = _lib.load(), _buf()
  refused(lib.fc_layer_norm(b, 4, 0, b, 1, 0, b, 4, b, 4, 1e-5, b, 4, b, b, None), b"sizes")
  refused(lib.fc_layer_norm(b, 4, 0, b, -1, 4, b, 4, b, 4, 1e-5, b, 4, b, b, None), b"sizes")
  refused(lib.fc_layer_norm(NULL, 4, 0, b, 1, 4, b, 4, b, 4, 1e-5, b, 4, b, b, None), b"null")
  refused(lib.fc_layer_norm(b, 4, 3, b, 1, 4, b, 4, b, 4, 1e-5, b, 4, b, b, None), b"dtype")
  assert lib.fc_layer_norm(b, 4, 0, b, 0, 4, b, 4, b, 4, 1e-5, b, 4, b, b, None) == 0  # no rows: nothing to do
  refused(lib.fc_layer_norm_backward(b, 4, b, 4, 0, b, b, b, 1, NULL, 1, 4, b, 4, NULL, 0, b, 4, b, 4, b, 4, 0, b,
                                     None), b"null")
  refused(lib.fc_layer_norm_backward(b, 4, b, 4, 0, b, b, b, 1, b, 0, 4, b, 4, NULL, 0, b, 4, b, 4, b, 4, 0, b,
                                     None), b"sizes")
  refused(lib.fc_layer_norm_backward(b, 4, b, 4, 0, b, b, b, 1, b, 1, 4, b, 4, NULL, 0, b, 4, b, 4, b, 4, 0, NULL,
                                     None), b"null")


def test_top_logits_and_distillation_refusals():
  lib, b = _lib.load(), _buf()
  for k in (0, 9, 1025):
    refused(lib.fc_top_logits(b, 8, 0, 1, 8 if k < 100 else 5000, k, 1.0, b, b, b, None), b"bad k")
  for t in (0.0, -1.0, float("inf"), float("nan")):
    refused(lib.fc_top_logits(b, 8, 0, 1, 8, 2, t, b, b, b, None), b"temperature")
  refused(lib.fc_top_logits(b, 8, 0, 1, 8, 2, 1.0, NULL, b, b, None), b"null")
  refused(lib.fc_top_logits(b, 8, 7, 1, 8, 2, 1.0, b, b, b, None), b"dtype")

  def distill(rows=1, vocab=8, k=2, clients=1, tau=1.0, dloss=NULL, row_loss=b, lse=b, loss=b, grad=NULL, logits=b,
              dtype=0):
    return lib.fc_distill(logits, 8, dtype, rows, vocab, b, b, k, b, b, clients, tau, NULL, NULL, dloss, row_loss, lse,
                          loss, grad, 8, None)

  refused(distill(k=0), b"bad k")
  refused(distill(k=1025), b"bad k")
  refused(distill(tau=0.0), b"temperature")
  refused(distill(vocab=0), b"sizes")
  refused(distill(clients=0), b"sizes")
  refused(distill(loss=NULL), b"null")  # neither a loss nor a gradient wanted
  refused(distill(loss=NULL, grad=b, lse=NULL), b"null")  # the gradient alone needs the saved lse
  refused(distill(row_loss=NULL), b"null")
  refused(distill(dloss=b), b"dloss")
  refused(distill(logits=NULL), b"null")
  refused(distill(dtype=4), b"dtype")


def test_linear_refusals():
  lib, b = _lib.load(), _buf()

  def forward(dtype=1, ntiles=1, rows=128, clients=1, k=8, m=8, act=0, splits=1, ws=NULL, nbytes=0, x=b, stride=8):
    return lib.fc_linear(x, stride, dtype, b, ntiles, rows, clients, k, m, b, 64, 8, NULL, 0, act, NULL, 0, NULL, 0, b,
                         8, splits, ws, nbytes, None)

  refused(forward(k=0), b"sizes")
  refused(forward(clients=0), b"sizes")
  refused(forward(ntiles=-1), b"sizes")
  refused(forward(act=4), b"activation")
  refused(forward(x=NULL), b"null")
  refused(forward(dtype=9), b"dtype")
  refused(forward(rows=64), b"tile_rows")
  refused(forward(dtype=0, rows=256), b"tile_rows")
  refused(forward(rows=256, stride=9), b"multiples of 4 bytes")
  refused(forward(splits=0), b"splits")
  refused(forward(splits=1025), b"splits")
  refused(forward(splits=2), b"workspace")
  refused(forward(splits=2, ws=b, nbytes=64), b"workspace")
  assert forward(ntiles=0) == 0

  def backward_input(act=0, pre=NULL, dz=b):
    return lib.fc_linear_backward_input(dz, 8, 1, b, 1, 128, 1, 8, 8, b, 64, 8, act, pre, 8, NULL, 0, b, 8, 1, NULL, 0,
                                        None)

  refused(backward_input(act=1), b"pre-activation")
  refused(backward_input(act=7), b"activation")
  refused(backward_input(dz=NULL), b"null")

  def weight(clients=1, m=8, dw=b, splits=1):
    return lib.fc_linear_backward_weight(b, 8, b, 8, 1, b, clients, 8, m, dw, 64, 8, NULL, 0, 0, 128, splits, NULL, 0,
                                         None)

  refused(weight(clients=0), b"sizes")
  refused(weight(m=0), b"sizes")
  refused(weight(dw=NULL), b"null")
  refused(weight(splits=3), b"workspace")


def test_linear_workspace():
  lib = _lib.load()
  assert lib.fc_linear_workspace_bytes(7, 128, 1) == 0
  assert lib.fc_linear_workspace_bytes(7, 32, 3) == 7 * 3 * (32 * 128 + 32) * 4
  assert lib.fc_linear_workspace_bytes(2, 256, 2) == 2 * 2 * (256 * 256 + 256) * 4
  for args in [(1, 64, 1), (1, 128, 0), (-1, 128, 1), (1, 128, 2000)]:
    assert lib.fc_linear_workspace_bytes(*args) == -1


def test_pack_rows_refusals():
  lib, b = _lib.load(), ctypes.create_string_buffer(128)
  at = (ctypes.addressof(b) + 15) // 16 * 16

  def pack(src=at, dst=at, cols=7, stride=8, dtype=1, clients=1, rows=1):
    return lib.fc_pack_rows(src, 0, 7, dtype, clients, rows, cols, dst, stride, None)

  refused(pack(cols=0), b"sizes")
  refused(pack(clients=0), b"sizes")
  refused(pack(stride=6), b"sizes")
  refused(pack(stride=12), b"vectors")
  refused(pack(dst=at + 8), b"vectors")
  refused(pack(src=NULL), b"null")
  refused(pack(dtype=5), b"dtype")
  assert pack(rows=0) == 0


def test_limits_of_scalars_and_sizes():
  lib, b = _lib.load(), _buf()
  for t in (1e-16, 1e16, 1e-40):
    refused(lib.fc_top_logits(b, 8, 0, 1, 8, 2, t, b, b, b, None), b"temperature")
  for eps in (-1e-5, float("nan")):
    refused(lib.fc_layer_norm(b, 4, 0, b, 1, 4, b, 4, b, 4, eps, b, 4, b, b, None), b"eps")
  # the gradients' join: clients x columns in one launch of fewer than 2^32 threads
  refused(lib.fc_layer_norm_backward(b, 4, b, 4, 0, b, b, b, 0, b, 1 << 20, 4096, b, 4, NULL, 0, b, 4, b, 4, b, 4, 0, b,
                                     None), b"sizes")
  refused(lib.fc_linear(b, 8, 1, b, 1, 128, 1, 1 << 31, 8, b, 64, 8, NULL, 0, 0, NULL, 0, NULL, 0, b, 8, 1, NULL, 0,
                        None), b"sizes")
  refused(lib.fc_linear_backward_weight(b, 8, b, 8, 1, b, 1 << 24, 8, 8, b, 64, 8, NULL, 0, 0, 128, 1, NULL, 0, None),
          b"too many tiles")
  refused(lib.fc_pack_rows(b, 8, 8, 1, 1 << 30, 1 << 20, 8, b - b % 16, 8, None), b"too many rows")


def test_memory_that_two_tensors_share():
  import torch
  from federated_amd import client_ops as ops
  buf = torch.zeros(10, 100)
  left, right, mid = buf[:, :50], buf[:, 50:], buf[:, 40:60]
  ops._apart("out", left, None, right)
  ops._apart("out", right, None, left, None)
  ops._apart("out", buf[:5], None, buf[5:])
  ops._apart("out", left, left, right)
  ops._apart("out", buf[3:4, 20:30], None, left[:3], left[4:])
  ops._apart("out", buf[:0], None, buf)
  ops._apart("out", torch.zeros(1, 8).as_strided((1, 8), (0, 1)), None, buf)
  whole = buf[:, :99].unflatten(1, (9, 11))
  ops._apart("dweight", whole, None, buf[:, 99:])
  for out, x in [(left, mid), (mid, left), (right, mid), (buf, right), (left, left), (left[:1], buf), (whole, buf[:, 98:]),
                 (left, buf.view(-1)[:50].expand(10, 50))]:
    with pytest.raises(ValueError):
      ops._apart("out", out, None, x)
  with pytest.raises(ValueError):
    ops._apart("out", left, mid)


def test_weight_gradient_of_few_rows_refusals():
  lib, b = _lib.load(), _buf()

  def few(dz=b, dw=b, clients=1, longest=1, k=8, m=8, dtype=1):
    return lib.fc_linear_backward_weight_few(dz, 8, b, 8, dtype, b, clients, longest, k, m, dw, 64, 8, NULL, 0, 0, None)

  for kw in (dict(clients=0), dict(longest=-1), dict(k=0), dict(m=0), dict(k=1 << 31), dict(m=1 << 31)):
    refused(few(**kw), b"sizes")
  refused(few(dz=NULL), b"null")
  refused(few(dw=NULL), b"null")
  refused(few(dtype=3), b"dtype")
  refused(few(clients=1 << 30, k=1 << 12), b"too many tiles")


def test_walk_refusals():
  lib, b = _lib.load(), _buf()
  b -= b % 16

  def forward(rows=128, k=8, x=b, ldx=8, ldw=8, dtype=1, client=64):
    return lib.fc_linear(x, ldx, dtype, b, 1, rows, 1, k, 8, b, client, ldw, NULL, 0, 0, NULL, 0, NULL, 0, b, 8, -1,
                         NULL, 0, None)

  for kw in (dict(rows=32), dict(rows=256), dict(k=129), dict(k=65, dtype=0), dict(x=b + 2), dict(ldx=9), dict(ldw=9),
             dict(client=65), dict(ldx=1 << 22)):
    refused(forward(**kw), b"FC_WALK")
  refused(lib.fc_linear_backward_weight(b, 8, b, 8, 1, b, 1, 8, 8, b, 64, 8, NULL, 0, 0, 128, -1, NULL, 0, None),
          b"splits")


def test_pack_rows_takes_16_bit_rows_only():
  lib, b = _lib.load(), ctypes.create_string_buffer(128)
  at = (ctypes.addressof(b) + 15) // 16 * 16
  refused(lib.fc_pack_rows(at, 0, 7, 0, 1, 1, 7, at, 8, None), b"dtype")


def test_distillation_without_rows():
  """No rows and no loss wanted: the gradient of an empty tensor may be a null pointer."""
  lib, b = _lib.load(), _buf()

  def distill(rows, lse=NULL, grad=NULL, logits=NULL):
    return lib.fc_distill(logits, 8, 0, rows, 8, b, b, 2, b, b, 1, 1.0, NULL, NULL, NULL, NULL, lse, NULL, grad, 8, None)

  assert distill(0) == 0 and distill(0, lse=b, grad=b, logits=b) == 0
  refused(distill(1, lse=b, logits=b), b"null")
  refused(distill(1, grad=b, logits=b), b"null")
  refused(distill(1, lse=b, grad=b), b"null")


def host_batch(counts):
  """What the argument checks read of a batch, its tensors on the host."""
  import torch
  from federated_amd import client_ops as ops
  batch = object.__new__(ops.ClientBatch)
  batch.device, batch.num_clients, batch.num_rows = torch.device("cpu"), len(counts), sum(counts)
  batch.row_client = batch.offsets = torch.zeros(8, dtype=torch.int32)
  return batch


@pytest.mark.parametrize("over", ["teacher_lse", "row_weights", "dloss", "lse"])
def test_a_gradient_over_the_rows_vectors_is_refused(monkeypatch, over):
  """Blocks read these while others write gradient rows."""
  import torch
  from federated_amd import client_ops as ops
  calls = []
  monkeypatch.setattr(ops, "_call", lambda where, name, *args: calls.append(name))
  batch, buf = host_batch([3, 2]), torch.ones(200)
  logits, out = torch.zeros(5, 8), buf[:40].view(5, 8)
  idx, val = torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2)
  for start in (0, 17, 35):
    vectors = dict(teacher_lse=buf[40:45], row_weights=buf[50:55], dloss=buf[60:62], lse=buf[70:75])
    vectors[over] = buf[start:start + (2 if over == "dloss" else 5)]
    dloss, lse = vectors.pop("dloss"), vectors.pop("lse")
    with pytest.raises(ValueError, match="shares memory"):
      ops.distillation_backward(logits, lse, idx, val, batch, dloss=dloss, out=out, **vectors)
    if over in vectors:
      with pytest.raises(ValueError, match="shares memory"):
        ops.distillation_with_gradient(logits, idx, val, batch, out=out, **vectors)
  assert not calls
  # beside them: taken
  vectors = dict(teacher_lse=buf[40:45], row_weights=buf[50:55])
  assert ops.distillation_backward(logits, buf[70:75], idx, val, batch, dloss=buf[60:62], out=out, **vectors) is out
  assert ops.distillation_with_gradient(logits, idx, val, batch, out=out, **vectors)[1] is out
  assert calls == ["fc_distill"] * 2


def test_inline_assembly_names_the_scalar_register_it_sets():
  """A statement that writes M0 says so: the compiler keeps its own values there."""
  import glob
  import os
  import re
  root = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
  writes = 0
  for path in glob.glob(os.path.join(root, "federated_amd", "csrc", "*")):
    with open(path) as f:
      for statement in re.findall(r"asm volatile\(.*?\);\n", f.read(), re.S):
        code, *rest = statement.split("::")
        if re.search(r"\bs_mov_b32 m0\b", code):
          writes += 1
          assert '"m0"' in "".join(rest), (path, statement)
  assert writes


@pytest.mark.parametrize("counts", [[1 << 62] * 4, [1 << 63, 1 << 63], [(1 << 63) - 1] * 2 + [9], [1 << 30] * 2,
                                    [(1 << 31) - 1024], [1, -1], [-(1 << 62)] * 4, [1 << 64]], ids=str)
def test_row_counts_whose_sum_wraps_are_refused(monkeypatch, counts):
  import torch
  from federated_amd import client_ops as ops
  monkeypatch.setattr(_lib, "require_gpu", lambda: None)
  monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
  with pytest.raises(ValueError):
    ops.ClientBatch(counts)


def test_weight_gradient_refuses_missing_operands():
  """They would be read on the device, by whichever client has rows."""
  lib, b = _lib.load(), _buf()
  for dz, x, clients in [(NULL, b, b), (b, NULL, b), (b, b, NULL)]:
    # the workspace is refused after it, should it be missed: nothing is launched
    refused(lib.fc_linear_backward_weight(dz, 8, x, 8, 1, clients, 1, 8, 8, b, 64, 8, NULL, 0, 0, 128, 3, NULL, 0, None),
            b"null")


@pytest.mark.parametrize("which", ["a", "b", "weight"])
def test_operands_too_large_for_one_copy_are_read_as_they_lie(monkeypatch, which):
  """Rows at odd elements are copied where that pays, but not more of them than the copy's one
  launch takes (2^24 - 1 blocks of 256 vectors)."""
  import torch
  from federated_amd import client_ops as ops
  packed = []
  monkeypatch.setattr(ops, "_packed", lambda t, rows: packed.append(t) or t)
  monkeypatch.setattr(ops, "_estimate", lambda tiles, steps, longest, size, aligned: (1.0 if aligned else 1e9, 128, 1))
  lib, at = _lib.load(), _buf() // 16 * 16 + 16
  half = torch.float16
  for over in (False, True):
    rows = (1 << 32) // 126 + (1000 if over else -10000)  # of 126 vectors; a matrix ends inside a block
    if which == "weight":
      a, n = torch.empty(9, 8, dtype=half, device="meta"), 9
      b = torch.empty(4, rows // 4, 1001, dtype=half, device="meta")
      pack = (b.shape[0], b.shape[1])
    else:
      big, small = torch.empty(rows, 1001, dtype=half, device="meta"), torch.empty(rows, 8, dtype=half, device="meta")
      a, b, n = (big, small, rows) if which == "a" else (small, big, rows)
      pack = (1, rows)
    if over:  # as the copy's entry has it
      refused(lib.fc_pack_rows(at, 0, 1001, 2, pack[0], pack[1], 1001, at, 1008, None), b"too many rows")
    packed.clear()
    out = ops._operands(a, b, n, (1, 1, 1), 1, 1)
    assert bool(packed) != over and out[0] is a and out[1] is b and out[2:] == (128, 1)
